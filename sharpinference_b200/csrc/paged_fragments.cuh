// The tensor-core fragments of attention over the paged 4-bit cache: one warp,
// eight pairs of a row and a query head, two tiles of 16 tokens at a time; and
// the second look at pairs that one token owns.
#pragma once

#include "paged_attention.cuh"

namespace si::dev {

constexpr int kPairs = 8;  // pairs of a row and a head in one pass

// N words from shared memory by the widest loads that N allows.
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&dst)[N], const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = reinterpret_cast<const uint4 *>(p)[i / 4];
            dst[i] = x.x, dst[i + 1] = x.y, dst[i + 2] = x.z, dst[i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 x = reinterpret_cast<const uint2 *>(p)[i / 2];
            dst[i] = x.x, dst[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) dst[i] = reinterpret_cast<const uint32_t *>(p)[i];
    }
}

// A warp copies one tile into its ring. Four lanes t of a fragment read value
// rows 4 t + i together, a multiple of 128 B apart: their 16-byte chunks are
// exchanged (chunk ^ 2 t) so that they lie in different banks.
template <int D>
__device__ __forceinline__ void copy_tile(uint8_t *dst, const uint8_t *src) {
    constexpr int kChunks = tile_bytes(D) / 16, kValues = D / 2;
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int i = 0; i < (kChunks + 31) / 32; ++i) {
        const int c = lane + 32 * i;
        int to = c;
        if (32 * i + 31 >= kValues && 32 * i < 2 * kValues)
            if (c >= kValues && c < 2 * kValues) to = c ^ ((((c - kValues) / (D / 8)) & 3) << 1);
        if (32 * i + 31 < kChunks || c < kChunks)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst + 16 * to)), "l"(src + 16 * c)
                         : "memory");
    }
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// Eight channels of each group of a pair's queries, zeros where the pair is not live.
template <class T, int D>
__device__ __forceinline__ void load_queries(const T *src, bool live, bool vec, float (&qv)[D / 32][8]) {
    const int lt = threadIdx.x & 3;
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
        if (live) {
            load8(src + 32 * j + 8 * lt, qv[j], vec);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) qv[j][e] = 0.0f;
        }
    }
}

// The queries as A fragments, rounded to F16 in rows 0..7 and what that leaves in
// rows 8..15, scaled by a power of two; returns what makes scores of their products.
template <int D>
__device__ __forceinline__ float split_queries(const float (&qv)[D / 32][8], float scale, uint32_t (&q)[D / 16][4]) {
    constexpr int NG = D / 32;
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(qv[j][e]));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    // a power of two brings the largest below 2, into F16's range
    int ex = top > 0.0f && top < INFINITY ? int(__float_as_uint(top) >> 23) - 127 : 0;
    ex = min(max(ex, -100), 126);
    const float down = __uint_as_float(uint32_t(127 - ex) << 23);
#pragma unroll
    for (int j = 0; j < NG; ++j)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const float q0 = qv[j][2 * s] * down, q1 = qv[j][2 * s + 1] * down;
            const __half2 hi = __floats2half2_rn(q0, q1);
            const float2 back = __half22float2(hi);
            q[2 * j + s / 2][2 * (s & 1)] = h2u(hi);
            q[2 * j + s / 2][2 * (s & 1) + 1] = h2u(__floats2half2_rn(q0 - back.x, q1 - back.y));
        }
    return fminf(fmaxf(scale * __uint_as_float(uint32_t(127 + ex) << 23), 1e-30f), 1e30f);
}

// Where a lane's words lie in a staged tile.
template <int D>
struct LanePlaces {
    static constexpr int W = D / 64, NS = D == 192 ? 3 : 1, kRowsHeld = D == 192 ? 4 : D == 128 ? 2 : 1;
    int key, key_scale;
    int value[kRowsHeld][NS];  // row 4 lt + i of the values, its chunks as copy_tile put them; words of one chunk are n = 0
    __device__ __forceinline__ LanePlaces() {
        const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
        key = (4 * (lg >> 1) + (lg & 1)) * (D / 2) + lt * (D / 8);
        key_scale = 16 * D + (4 * (lg >> 1) + (lg & 1)) * (D / 16);
#pragma unroll
        for (int i = 0; i < kRowsHeld; ++i)
#pragma unroll
            for (int n = 0; n < NS; ++n) value[i][n] = 8 * D + (((4 * lt + i) * (D / 2) + 4 * (W * lg + n)) ^ (lt << 5));
    }
    __device__ __forceinline__ int value_row(int i, int n) const {
        if constexpr (D == 64) return value[0][0] ^ (32 * i);
        else if constexpr (D == 128) return value[i & 1][0] + 128 * (i >> 1);
        else if constexpr (D == 192) return value[i][n];
        else return value[0][0] + 128 * i;
    }
};

// Scores of two staged tiles: s[z][i] of pair lg and token 16 z + 4 lt + i.
template <int D>
__device__ __forceinline__ void score_two(const uint8_t *stage, const LanePlaces<D> &at, const uint32_t (&q)[D / 16][4],
                                          float (&s)[2][4]) {
    constexpr int NG = D / 32, TB = tile_bytes(D);
    float c[2][2][4];
#pragma unroll
    for (int zu = 0; zu < 4; ++zu) {
        const uint8_t *p = stage + (zu >> 1) * TB + (zu & 1) * D;
        uint32_t k[NG], ks[NG / 2];
        load_words(k, p + at.key);
        load_words(ks, stage + (zu >> 1) * TB + (zu & 1) * (4 * NG) + at.key_scale);
#pragma unroll
        for (int j = 0; j < NG; ++j) {
            const __half2 both = u2h(ks[j / 2]), offs = __hmul2(both, __float2half2_rn(-24.0f));
            const __half2 sc = j & 1 ? __high2half2(both) : __low2half2(both);
            const __half2 off = j & 1 ? __high2half2(offs) : __low2half2(offs);
            if (j == 0) mma_first(c[zu >> 1][zu & 1], q[0], unpack<0>(k[0], sc, off), unpack<1>(k[0], sc, off));
            else mma(c[zu >> 1][zu & 1], q[2 * j], unpack<0>(k[j], sc, off), unpack<1>(k[j], sc, off));
            mma(c[zu >> 1][zu & 1], q[2 * j + 1], unpack<2>(k[j], sc, off), unpack<3>(k[j], sc, off));
        }
    }
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[z][i] = c[z][i >> 1][i & 1] + c[z][i >> 1][2 + (i & 1)];
}

// Scales of the lane's values: four tokens 4 lt .. of each tile.
template <int D, int NS>
__device__ __forceinline__ void value_scales(const uint8_t *stage, uint2 (&vs)[2][NS]) {
    constexpr int W = D / 64;
    const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
#pragma unroll
    for (int z = 0; z < 2; ++z)
#pragma unroll
        for (int n = 0; n < NS; ++n)
            vs[z][n] =
                *reinterpret_cast<const uint2 *>(stage + z * tile_bytes(D) + 17 * D + (W * lg + n) / 4 * 32 + 8 * lt);
}

// Adds the probabilities times the values of two staged tiles: o[4 w + i] of channels 8 (W lg + w) + 2 i .. + 1 and
// pairs 2 lt, 2 lt + 1.
template <int D, bool kLow, int NS>
__device__ __forceinline__ void add_values(const uint8_t *stage, const LanePlaces<D> &at, const uint2 (&vs)[2][NS],
                                           const uint32_t (&hi)[2][2], const uint32_t (&lo)[2][2],
                                           float (&o)[4 * (D / 64)][4]) {
    constexpr int W = D / 64, TB = tile_bytes(D);
#pragma unroll
    for (int z = 0; z < 2; ++z) {
        uint32_t v[4][W];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (NS == 1) {
                load_words(v[i], stage + z * TB + at.value_row(i, 0));
            } else {
#pragma unroll
                for (int n = 0; n < NS; ++n)
                    v[i][n] = *reinterpret_cast<const uint32_t *>(stage + z * TB + at.value_row(i, n));
            }
        }
#pragma unroll
        for (int w = 0; w < W; ++w) {
            const uint2 sv = vs[z][NS == 3 ? w : 0];
            const __half2 s01 = u2h(sv.x), s23 = u2h(sv.y), minus = __float2half2_rn(-24.0f);
            const __half2 f01 = __hmul2(s01, minus), f23 = __hmul2(s23, minus);
            const uint32_t lo01 = __byte_perm(v[0][w], v[1][w], 0x5410), hi01 = __byte_perm(v[0][w], v[1][w], 0x7632),
                           lo23 = __byte_perm(v[2][w], v[3][w], 0x5410), hi23 = __byte_perm(v[2][w], v[3][w], 0x7632);
            auto step = [&](float (&acc)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                const uint32_t f[4] = {a0, a1, a2, a3};
                mma(acc, f, hi[z][0], hi[z][1]);
                if constexpr (kLow) mma(acc, f, lo[z][0], lo[z][1]);
            };
            step(o[4 * w], unpack<0>(lo01, s01, f01), unpack<0>(hi01, s01, f01), unpack<0>(lo23, s23, f23),
                 unpack<0>(hi23, s23, f23));
            step(o[4 * w + 1], unpack<1>(lo01, s01, f01), unpack<1>(hi01, s01, f01), unpack<1>(lo23, s23, f23),
                 unpack<1>(hi23, s23, f23));
            step(o[4 * w + 2], unpack<2>(lo01, s01, f01), unpack<2>(hi01, s01, f01), unpack<2>(lo23, s23, f23),
                 unpack<2>(hi23, s23, f23));
            step(o[4 * w + 3], unpack<3>(lo01, s01, f01), unpack<3>(hi01, s01, f01), unpack<3>(lo23, s23, f23),
                 unpack<3>(hi23, s23, f23));
        }
    }
}

// ---- pairs that one token owns ---------------------------------------------------------------------------------
// In a row that one token owns the channels in which that token's value is 0 consist of the other tokens' small
// probabilities, which F16 does not hold. Such rows are summed again, a window of 17 binary orders of magnitude at a
// time: within its window every probability keeps 21 bits as two F16 numbers, and the windows' sums are added up from
// the smallest on, in FP32. Seven windows reach 2^-119 of the largest; those that hold no token are left out. It costs a
// walk over the scores and one for every window that holds a token, for eight pairs together; calls whose rows are all
// owned, us against the same call with ordinary scores: 64 streams of up to 4096 tokens 485 / 79, one of 32768 99 / 26,
// three chunks of up to 777 rows 2200 / 126, 16 rows on 32768 tokens 1990 / 57 (213000 with a row to a warp in FP32).
// The sums stay in their accumulators: what truncation takes off them is a small part of 2^-16 of a row.
constexpr int kWindows = 7;
constexpr float kWindowBits = 17.0f, kWindowLift = 14.0f;  // log2 of a window's width, of its largest probability

// A lane's pair (lg) in such a pass; the same in the four lanes of a group.
template <class T>
struct OwnedPair {
    const T *query;
    int position, first;
    bool live;
};

// Walks two tiles of [t_begin, t_end) at a time through a ring of two stages: f(stage, scores), those that a pair does
// not see at -inf.
template <class T, int D, class F>
__device__ __forceinline__ void score_all(const PagedArgs &a, const OwnedPair<T> &p, int stream, int kvh, int t_begin,
                                          int t_end, const uint32_t (&q)[D / 16][4], uint8_t *ring, F &&f) {
    constexpr int TB = tile_bytes(D);
    const LanePlaces<D> at;
    const int lt = threadIdx.x & 3;
    auto fetch = [&](int t, uint8_t *stage) {
        int there = 0;
        for (int z = 0; z < 2; ++z)
            if (t + z < t_end)
                if (const uint8_t *tile = tile_of(a, stream, 16 * (t + z), kvh)) {
                    copy_tile<D>(stage + z * TB, tile);
                    there |= 1 << z;
                }
        copy_commit();
        return there;
    };
    __syncwarp();
    int there = fetch(t_begin, ring), coming = 0;
#pragma unroll 1
    for (int t = t_begin; t < t_end; t += 2, there = coming) {
        const uint8_t *stage = ring + ((t - t_begin) & 2) * TB;
        __syncwarp();  // the other stage's readers are done
        coming = fetch(t + 2, ring + ((t + 2 - t_begin) & 2) * TB);
        copy_wait<1>();
        __syncwarp();
        float s[2][4];
        score_two<D>(stage, at, q, s);
#pragma unroll
        for (int z = 0; z < 2; ++z)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int token = 16 * (t + z) + 4 * lt + i;
                if (!p.live || !((there >> z) & 1) || token < p.first || token > p.position) s[z][i] = -INFINITY;
            }
        f(stage, at, there, t, s);
    }
    copy_wait<0>();
    __syncwarp();
}

// A pair's largest score of these tiles (before its scale) and a bit for each window below it that may hold a token.
struct Windows {
    float most;
    uint32_t held;
    // the same windows counted from a larger score on
    __device__ __forceinline__ uint32_t below(float top, float scale) const {
        if (most == -INFINITY) return 0;
        const float by = (top - most) * scale * (1.0f / kWindowBits);
        if (by == 0.0f) return held;
        if (!(by < float(kWindows))) return 0;
        return (held << int(by) | held << (int(by) + 1)) & ((1u << kWindows) - 1);
    }
};

// (Queries are read by element: ptxas of CUDA 12.9 ends in a fault on a 32-byte load in a function that is called.)
template <class T, int D>
__device__ __noinline__ Windows find_windows(const PagedArgs &a, float scale, const OwnedPair<T> p, int stream,
                                             int kvh, int t_begin, int t_end, uint8_t *ring, float *unscale) {
    uint32_t q[D / 16][4];
    {
        float qv[D / 32][8];
        load_queries<T, D>(p.query, p.live, false, qv);
        *unscale = split_queries<D>(qv, scale, q);
    }
    const float us = *unscale;
    Windows w{-INFINITY, 0};
    score_all<T, D>(a, p, stream, kvh, t_begin, t_end, q, ring,
                    [&](const uint8_t *, const LanePlaces<D> &, int, int, const float(&s)[2][4]) {
                        float top = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i >> 2][i & 3]);
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                        if (top > w.most) {
                            w.held = w.below(top, us);
                            w.most = top;
                        }
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float x = (w.most - s[i >> 2][i & 3]) * us * (1.0f / kWindowBits);
                            // near a border both windows are taken to hold the token
                            if (x < float(kWindows)) w.held |= 1u << int(fmaxf(x - 1e-3f, 0.0f)) | 1u << int(x + 1e-3f);
                        }
                    });
    w.held |= __shfl_xor_sync(0xffffffffu, w.held, 1);
    w.held |= __shfl_xor_sync(0xffffffffu, w.held, 2);
    w.held &= (1u << kWindows) - 1;
    return w;
}

// Sums of the pairs' probabilities 2^(lift + score - most) and of the values they weigh over these tiles, left in
// `part` as [kPairs][D] values, then [kPairs] sums of probabilities (`part` may be the ring).
template <class T, int D>
__device__ __noinline__ void sum_windows(const PagedArgs &a, float scale, const OwnedPair<T> p, int stream, int kvh,
                                         int t_begin, int t_end, uint8_t *ring, float most, uint32_t held, float lift,
                                         float *part) {
    constexpr int W = D / 64, NS = D == 192 ? 3 : 1;
    const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
    uint32_t q[D / 16][4];
    float us;
    {
        float qv[D / 32][8];
        load_queries<T, D>(p.query, p.live, false, qv);
        us = split_queries<D>(qv, scale, q);
    }
    float o[4 * W][4], l = 0.0f;
#pragma unroll
    for (int i = 0; i < 4 * W; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.0f;
    held = __reduce_or_sync(0xffffffffu, held);
    auto times = [&](float by) {
        l *= by;
#pragma unroll
        for (int i = 0; i < 4 * W; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][e] *= by;
    };
#pragma unroll 1
    for (int k = kWindows - 1; k >= 0; --k) {
        times(exp2f(-kWindowBits));
        if (!((held >> k) & 1u)) continue;
        const float from = -kWindowBits * float(k + 1), to = -kWindowBits * float(k), up = kWindowLift - to;
        score_all<T, D>(
            a, p, stream, kvh, t_begin, t_end, q, ring,
            [&](const uint8_t *stage, const LanePlaces<D> &at, int there, int t, const float(&s)[2][4]) {
                uint32_t hi[2][2], lo[2][2];
                bool any = false;
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        float e[2];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float x = (s[z][2 * u + h] - most) * us;
                            const bool in = x > from && x <= to;
                            e[h] = in ? ex2(x + up) : 0.0f;
                            any |= in;
                        }
                        l += e[0] + e[1];
                        const __half2 f = __floats2half2_rn(e[0], e[1]);
                        const float2 back = __half22float2(f);
                        hi[z][u] = h2u(f);
                        lo[z][u] = h2u(__floats2half2_rn(e[0] - back.x, e[1] - back.y));
                    }
                if (!__any_sync(0xffffffffu, any)) return;
                uint2 vs[2][NS];
                value_scales<D>(stage, vs);
                // values that weigh nothing count as 0, whatever is there: tiles that are not, tokens that no pair sees
                const int any_first = __reduce_min_sync(0xffffffffu, p.live ? p.first : INT32_MAX);
                const int any_last = __reduce_max_sync(0xffffffffu, p.live ? p.position : -1);
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int token = 16 * (t + z) + 4 * lt + i;
                        const bool none = !((there >> z) & 1) || token < any_first || token > any_last;
#pragma unroll
                        for (int n = 0; n < NS; ++n) {
                            uint32_t &pair_of = i < 2 ? vs[z][n].x : vs[z][n].y;
                            const uint32_t half = i & 1 ? pair_of >> 16 : pair_of & 0xFFFFu;
                            if (none || (half & 0x7C00u) == 0x7C00u) pair_of &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                        }
                    }
                add_values<D, true>(stage, at, vs, hi, lo, o);
            });
    }
    times(exp2f(lift - kWindowLift));
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
#pragma unroll
    for (int w = 0; w < W; ++w)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) part[(2 * lt + (e & 1)) * D + 8 * (W * lg + w) + 2 * i + (e >> 1)] = o[4 * w + i][e];
    if (lt == 0) part[kPairs * D + lg] = l;
    __syncwarp();
}

}  // namespace si::dev
