// Attention over the paged 4-bit cache: the kernel of single tokens and of a
// few rows per stream.
//
// Bound: the cache's bytes (0.5625 B a value, read once per eight pairs of a
// row and a query head), so the loop is built to spend few instructions on a
// value. Both products run on the tensor cores (mma.m16n8k16, F16 operands,
// FP32 sums): a cached value code * scale is an F16 number, so unpacking is a
// shift, a mask and one FMA for two values, (16 + nibble) * s - 24 * s, exact.
//   scores  C[16, 8 tokens] += A[16, 16 channels] B[16 channels, 8 tokens]:
//     rows 0..7 of A are eight queries rounded to F16, rows 8..15 what the
//     rounding left over, so the sum of both halves of C has 22 bits of them;
//   values  C[16 channels, 8] += A[16 channels, 16 tokens] B[16 tokens, 8]:
//     a score's place in C is its probability's place in B, so probabilities
//     never leave their lanes; F32 calls add the product with what rounding
//     them to F16 left over. F16 calls leave that out: it is up to 2^-11 of a
//     probability, no more than the rounding of their outputs loses (relative
//     error of 16 streams of 2047 tokens 2.3e-4 .. 2.6e-4, rounding the outputs
//     alone 2.1e-4).
// The tiles of 16 tokens of all streams, heads and passes form one line that is
// cut evenly over the warps of the grid, so uneven lengths balance. A warp walks
// its cut with running maxima that move only when a score exceeds them by 2^2,
// the next two tiles on their way into its ring; items that a cut divides are put together
// in shared memory once per block, and over the blocks by the last to arrive.
// Measured: 64 streams of up to 4096 tokens (40 query, 10 key/value heads of 128,
// F32) 72 us, 3.2 TB/s: near half each of the ALU, FMA and tensor pipes at the
// three warps a scheduler that the registers allow. One stream of 32768 tokens (24, 8
// heads) 21.3 us, of which the tiles take about half.
// F16 probabilities end 2^-37 below a row's largest. In an F32 row that
// one token owns (all others together below 2^-16 of it) the channels in which
// that token's value is 0 consist of such small ones, so a warp that meets
// such rows goes over its tiles again for them (`sum_windows`). Where several
// tokens own a row and all are 0 in a channel, the rest keeps that floor: it is
// off by 2^-38 of the largest probability times a value (2^-33 where maxima may lag 2^7, at the same speed).
#include <type_traits>

#include "launch.cuh"
#include "paged_fragments.cuh"

namespace si::kernels {
namespace {

using namespace si::dev;

// Pairs of a row and a query head of a stream and key/value head; more go to paged_chunk.cu. Measured with 4
// key/value heads of 128, us here / there: 16 streams of 2047 tokens, F32 32 pairs 37/51, 64 pairs 57/66, 96 pairs
// 74/68, F16 24 pairs 30/36, 32 pairs 36/35, 44 pairs 44/35; 64 of 1500, F32 32 pairs 77/104, 44 pairs 104/106, F16
// 72/71 and 97/72; one of 32768, F32 64 pairs 55/53, 96 pairs 73/53, F16 44 pairs 42/54, 96 pairs 69/55.
constexpr int kFewPairs = 32;
constexpr float kSlack = 2.0f;    // log2 of what a score may exceed the running maximum by
constexpr float kLift = 13.0f;    // log2 of a probability at the maximum: F16 keeps more small ones
// The products truncate what they add up. F32 calls take the sums out of the accumulators every kFlush tiles and add
// them up rounded, in memory of their own (32768 tokens that one warp walks, values of one sign: off by 1.3e-4 of the
// output without, 1.9e-6 so; mixed signs 4.2e-5 and 1.4e-6). 64 streams of up to 4096 tokens, 92
// tiles a warp: 71.1 us without, 72.0 so, 71.6 with 64 tiles. F16 calls do so every 8192 tokens (131072 tokens of values
// of one sign: off by 5.2e-4 without, 7e-5 so; their rounding 2.1e-4).
constexpr int kFlush = 32, kFlushHalf = 512;
template <bool kFour>
constexpr int pass_pairs() {  // where rows or columns of the products hold a pair twice (`walk`)
    return kFour ? kPairs / 2 : kPairs;
}

// Warps of a block, one block to an SM: as many as registers and rings allow, equally many for each of the four
// schedulers. 64 streams of 3000 tokens, 16 query and 4 key/value heads, F32, us: heads of 128 with 8 / 12 / 14 / 16
// warps 43.7 / 41.8 / 46 / 46.5 (16 leave 128 registers, and spill), of 192 with 8 / 10 warps 56.8 / 70.7, of 64
// with 8 / 12 / 16 warps 31.8 / 29.4 / 30.0.
template <int D>
constexpr int warps() {
    return D <= 128 ? 12 : 8;
}

// What a warp holds of one item of the line: running maximum, sum and weighted
// values of eight pairs, in the lanes' fragment layout.
template <int D>
struct Sums {
    float o[4 * (D / 64)][4];
    float m, l;
    uint32_t bad;  // groups in which the lane's pair sees a value that is not finite
};

// An item: one pass of eight (four) pairs of one stream on one key/value head.
struct Item {
    StreamWork sw;
    int stream, kvh, pass;
    int at, tiles;  // its place on the line
};

// Sums of those pairs of an item anew that one token owns (the maxima before their scale).
template <class T, int D, bool kFour>
__device__ __noinline__ void look_again(const AttentionArgs<T> &g, const Item &it, int tile_a, int tile_b, bool owned,
                                        uint8_t *ring, Sums<D> &r) {
    constexpr int W = D / 64;
    const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
    const int pair = it.pass * pass_pairs<kFour>() + lg, row = pair / g.group;
    OwnedPair<T> p;
    p.live = owned;
    p.query = g.query + (it.sw.begin + row) * g.query_stride + int64_t(it.kvh * g.group + pair - row * g.group) * D;
    p.position = it.sw.length - it.sw.rows + row;
    p.first = g.window ? max(0, p.position - g.window + 1) : 0;
    const int t_begin = it.sw.first_tile + tile_a, t_end = it.sw.first_tile + tile_b;
    float us, *part = reinterpret_cast<float *>(ring);
    const Windows w = find_windows<T, D>(g.a, g.scale, p, it.stream, it.kvh, t_begin, t_end, ring, &us);
    sum_windows<T, D>(g.a, g.scale, p, it.stream, it.kvh, t_begin, t_end, ring, w.most, w.held, kLift, part);
    if (owned) r.m = w.most, r.l = part[kPairs * D + lg];
    const uint32_t rows = __ballot_sync(0xffffffffu, owned);
#pragma unroll
    for (int c = 0; c < 2; ++c)
        if ((rows >> (4 * (2 * lt + c))) & 1u)
#pragma unroll
            for (int n = 0; n < W; ++n)
#pragma unroll
                for (int i = 0; i < 8; ++i) r.o[4 * n + i / 2][2 * (i & 1) + c] = part[(2 * lt + c) * D + 8 * (W * lg + n) + i];
    __syncwarp();
}

// One warp over the tiles [tile_a, tile_b) of an item, two at a time through its
// ring of two stages. kFour (32-bit calls of up to four pairs a stream, passes of four): rows lg and
// lg + 4 of the scores are the same pair, and the probabilities' columns lg + 4
// hold what rounding left of columns lg, so that one product does for both (64
// streams of 4 pairs: 70.9 us against 75.1, both without the sums put away).
template <class T, int D, bool kFour>
__device__ __forceinline__ void walk(const AttentionArgs<T> &g, const Item &it, int tile_a, int tile_b, uint8_t *ring,
                                     Sums<D> &r) {
    constexpr int NG = D / 32, W = D / 64, NS = D == 192 ? 3 : 1, TB = tile_bytes(D);
    constexpr bool kWide = sizeof(T) == 4;
    const PagedArgs &a = g.a;
    const StreamWork &sw = it.sw;
    const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
    // this lane's pair: the queries as A fragments and its visible tokens
    const int pair = it.pass * pass_pairs<kFour>() + (kFour ? lg & 3 : lg), row_in = pair / g.group;
    const bool live = row_in < sw.rows;
    const T *src = g.query + (sw.begin + row_in) * g.query_stride + int64_t(it.kvh * g.group + pair - row_in * g.group) * D;
    const int position = live ? sw.length - sw.rows + row_in : -1;
    const int first = g.window ? max(0, position - g.window + 1) : 0;

    const int t_begin = sw.first_tile + tile_a, t_end = sw.first_tile + tile_b;
    // every token of a tile between these is seen by all pairs, none outside [any_first, any_last] by any
    const int all_first = __reduce_max_sync(0xffffffffu, live ? first : 0);
    const int all_last = __reduce_min_sync(0xffffffffu, live ? position : INT32_MAX);
    const int any_first = __reduce_min_sync(0xffffffffu, live ? first : INT32_MAX);
    const int any_last = min(__reduce_max_sync(0xffffffffu, position), (a.table_width << a.page_shift) - 1);

    // lane i holds where the i-th tile from `held` on lies in the pool, counted in tiles
    constexpr uint32_t kNone = 0xFFFFFFFFu;
    uint32_t places = kNone;
    int held = INT32_MIN;
    auto tile_at = [&](int tile) -> const uint8_t * {
        if (tile < held || tile >= held + 32) {
            held = tile;
            const int mine = tile + lane, shift = a.page_shift - 4, entry = mine >> shift;
            places = kNone;
            if (mine < t_end && 16 * mine <= any_last && 16 * mine + 15 >= any_first && entry < a.table_width) {
                const int page = a.page_table[int64_t(it.stream) * a.table_width + entry];
                if (uint32_t(page) < uint32_t(a.page_count))
                    places = ((uint32_t(page) * a.kv_heads + it.kvh) << shift) + (mine & ((1 << shift) - 1));
            }
        }
        const uint32_t place = __shfl_sync(0xffffffffu, places, tile - held);
        return place == kNone ? nullptr : a.pages + uint64_t(place) * TB;
    };
    // bit z of the result: tile t + z is there and travels into `stage`
    auto fetch = [&](int t, uint8_t *stage) {
        const uint8_t *p0 = tile_at(t), *p1 = tile_at(t + 1);
        if (p0) copy_tile<D>(stage, p0);
        if (p1) copy_tile<D>(stage + TB, p1);
        copy_commit();
        return (p0 ? 1 : 0) | (p1 ? 2 : 0);
    };
    float qv[NG][8];
    load_queries<T, D>(src, live, g.vec, qv);
    __syncwarp();
    int there = fetch(t_begin, ring), coming = 0;

    uint32_t q[2 * NG][4];
    const float unscale = split_queries<D>(qv, g.scale, q), slack = kSlack / unscale;  // the scores' scale, kSlack before it
#pragma unroll
    for (int i = 0; i < 4 * W; ++i) r.o[i][0] = r.o[i][1] = r.o[i][2] = r.o[i][3] = 0.0f;
    float m = -INFINITY, l = 0.0f, most = -INFINITY;
    r.bad = 0;
    float flushed = 1.0f;  // how far the maximum has moved since sums were put away
    bool begun = false;    // some are
    auto held_at = [&](int i) {
        return g.held + (int64_t(blockIdx.x) * warps<D>() + (threadIdx.x >> 5)) * (4 * W * 32) + 32 * i + lane;
    };
    const LanePlaces<D> at;  // this lane's places in a tile
    for (int t = t_begin;;) {
        const int stop = min(t + (kWide ? kFlush : kFlushHalf), t_end);
        for (; t < stop; t += 2, there = coming) {
            const int t0 = 16 * t;
            const uint8_t *stage = ring + ((t - t_begin) & 2) * TB;
            __syncwarp();  // the other stage's readers are done
            coming = fetch(t + 2, ring + ((t + 2 - t_begin) & 2) * TB);
            copy_wait<1>();
            __syncwarp();
            float s[2][4];
            score_two<D>(stage, at, q, s);
            uint2 vs[2][NS];
            value_scales<D>(stage, vs);
            if (t0 < all_first || t0 + 31 > all_last || there != 3) {
#pragma unroll
                for (int z = 0; z < 2; ++z)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int token = t0 + 16 * z + 4 * lt + i;
                        const bool none = !((there >> z) & 1);
                        if (none || token < first || token > position) s[z][i] = -INFINITY;
                        if (none || token < any_first || token > any_last) {  // whatever is there: zeros
#pragma unroll
                            for (int n = 0; n < NS; ++n) {
                                uint32_t &half_pair = i < 2 ? vs[z][n].x : vs[z][n].y;
                                half_pair &= i & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                            }
                        }
                    }
            }
            uint32_t odd = 0;
#pragma unroll
            for (int n = 0; n < 2 * NS; ++n) odd |= not_finite(vs[n & 1][n >> 1].x) | not_finite(vs[n & 1][n >> 1].y);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, fmaxf(s[0][i], s[1][i]));
            if constexpr (kWide) most = fmaxf(most, top);
            // rare: a NaN among the values' scales, a score above its maximum
            if (__any_sync(0xffffffffu, (odd & 0x80008000u) || top > m + slack)) {
                if (__any_sync(0xffffffffu, odd & 0x80008000u)) {
                    // a NaN in the cache reaches the pairs that see its token, not the others of the product
                    for (int i = 0; i < 32; ++i)
                        if ((there >> (i >> 4)) & 1)
                            for (int j = 0; j < NG; ++j) {
                                const uint32_t v =
                                    reinterpret_cast<const uint16_t *>(stage + (i >> 4) * TB + 17 * D)[j * 16 + (i & 15)];
                                if ((v & 0x7C00u) == 0x7C00u && t0 + i >= first && t0 + i <= position) r.bad |= 1u << j;
                            }
#pragma unroll
                    for (int n = 0; n < 4 * NS; ++n) {
                        uint2 &pair_of = vs[n & 1][n >> 2];
                        uint32_t &h = n & 2 ? pair_of.y : pair_of.x;
                        if ((h & 0x7C00u) == 0x7C00u) h &= 0xFFFF0000u;
                        if ((h & 0x7C000000u) == 0x7C000000u) h &= 0x0000FFFFu;
                    }
                }
                // a pair's maximum moves by its own scores alone
                float up = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                up = fmaxf(up, __shfl_xor_sync(0xffffffffu, up, 2));
                const bool moves = up > m + slack;
                const float alpha = moves ? ex2((m - up) * unscale) : 1.0f;
                if (moves) m = up;
                l *= alpha;
                flushed *= alpha;
                const float a0 = __shfl_sync(0xffffffffu, alpha, 8 * lt), a1 = __shfl_sync(0xffffffffu, alpha, 8 * lt + 4);
#pragma unroll
                for (int i = 0; i < 4 * W; ++i) {
                    r.o[i][0] *= a0, r.o[i][2] *= a0;
                    r.o[i][1] *= a1, r.o[i][3] *= a1;
                }
            }
            const float lift = kLift - (m == -INFINITY ? 0.0f : m) * unscale;
            uint32_t hi[2][2], lo[2][2];
#pragma unroll
            for (int z = 0; z < 2; ++z)
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float e0 = ex2(fmaf(s[z][2 * u], unscale, lift)), e1 = ex2(fmaf(s[z][2 * u + 1], unscale, lift));
                    l += e0 + e1;
                    const __half2 h = __floats2half2_rn(e0, e1);
                    hi[z][u] = h2u(h);
                    if constexpr (kWide) {
                        const float2 f = __half22float2(h);
                        lo[z][u] = h2u(__floats2half2_rn(e0 - f.x, e1 - f.y));
                        if (kFour && lg >= 4) hi[z][u] = lo[z][u];
                    }
                }
            add_values<D, kWide && !kFour>(stage, at, vs, hi, lo, r.o);
        }
        if (begun) {
            const float f0 = __shfl_sync(0xffffffffu, flushed, 8 * lt), f1 = __shfl_sync(0xffffffffu, flushed, 8 * lt + 4);
#pragma unroll
            for (int i = 0; i < 4 * W; ++i) {
                const float4 y = __ldcg(held_at(i));
                r.o[i][0] = fmaf(y.x, f0, r.o[i][0]), r.o[i][1] = fmaf(y.y, f1, r.o[i][1]);
                r.o[i][2] = fmaf(y.z, f0, r.o[i][2]), r.o[i][3] = fmaf(y.w, f1, r.o[i][3]);
            }
        }
        if (t >= t_end) break;
#pragma unroll
        for (int i = 0; i < 4 * W; ++i) {
            __stcg(held_at(i), make_float4(r.o[i][0], r.o[i][1], r.o[i][2], r.o[i][3]));
            r.o[i][0] = r.o[i][1] = r.o[i][2] = r.o[i][3] = 0.0f;
        }
        begun = true;
        flushed = 1.0f;
    }
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    if constexpr (kFour) {
#pragma unroll
        for (int i = 0; i < 4 * W; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) r.o[i][e] += __shfl_xor_sync(0xffffffffu, r.o[i][e], 2);
    }
    if constexpr (kWide) {
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const float largest = ex2(fmaf(most, unscale, kLift - (m == -INFINITY ? 0.0f : m) * unscale));
        // a token that is alone needs no second look
        const bool owned = most > -INFINITY && l - largest < kOwned * largest && (!kFour || lg < 4) &&
                           min(position, 16 * t_end - 1) > max(first, 16 * t_begin);
        if (__any_sync(0xffffffffu, owned)) {
            // by way of memory, so that the sums' registers need not outlive the call
            const Item again = it;
            Sums<D> copy = r;
            copy.m = m, copy.l = l;
            look_again<T, D, kFour>(g, again, tile_a, tile_b, owned, ring, copy);
            r = copy;
            m = r.m, l = r.l;
        }
    }
    r.m = m * unscale;
    r.l = l;
}

// A partial result: [8][D] weighted values, then the maxima and the sums.
template <int D>
constexpr int part_floats() {
    return kPairs * (D + 2);
}

// Floats of a warp's ring (two stages of two tiles, at least a partial result)
// and of all its shared memory.
template <int D>
constexpr int ring_floats() {
    return 4 * tile_bytes(D) / 4;
}
template <int D>
constexpr int warp_floats() {
    static_assert(ring_floats<D>() >= part_floats<D>(), "the ring takes a part");
    return ring_floats<D>() + (part_floats<D>() + 31) / 32 * 32;
}

// The eight values of pair 2 lt + c in word w of this lane, NaN where the pair sees one.
template <int D>
__device__ __forceinline__ void lane_values(const Sums<D> &r, int w, int c, uint32_t bad, float (&v)[8]) {
    constexpr int W = D / 64;
    const int lg = (threadIdx.x & 31) >> 2;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = r.o[4 * w + i][c], v[2 * i + 1] = r.o[4 * w + i][2 + c];
    if ((bad >> ((W * lg + w) >> 2)) & 1u)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = NAN;
}

template <int D>
__device__ __forceinline__ void deposit(const Sums<D> &r, float *slot) {
    constexpr int W = D / 64;
    const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint32_t bad = __shfl_sync(0xffffffffu, r.bad, 8 * lt + 4 * c);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            float v[8];
            lane_values<D>(r, w, c, bad, v);
            store8_shared(slot + (2 * lt + c) * D + 8 * (W * lg + w), v);
        }
    }
    if (lt == 0) {
        slot[kPairs * D + lg] = r.m;
        slot[kPairs * D + kPairs + lg] = r.l;
    }
}

// Output row and head of a pair of an item; null for a pair without an output.
template <class T, int D, bool kFour>
__device__ __forceinline__ T *pair_output(const AttentionArgs<T> &g, const Item &it, int pr) {
    const int pair = it.pass * pass_pairs<kFour>() + pr, row = pair / g.group;
    if (pr >= pass_pairs<kFour>() || row >= it.sw.rows) return nullptr;
    const int p = it.sw.length - it.sw.rows + row;
    if (p < 0 || (p >> g.a.page_shift) >= g.a.table_width) return nullptr;
    return g.output + (it.sw.begin + row) * g.output_stride + int64_t(it.kvh * g.group + pair - row * g.group) * D;
}

// Parts of an item, in the item's order: part 0, then parts at equal distances.
struct Parts {
    const float *first, *rest;
    int stride, n;
    __device__ __forceinline__ const float *at(int i) const { return i == 0 ? first : rest + int64_t(i) * stride; }
};

template <bool kFour>
__device__ __forceinline__ int live_pairs(const Item &it, int group) {
    return min(pass_pairs<kFour>(), it.sw.rows * group - it.pass * pass_pairs<kFour>());
}

// Adds the parts of an item up, in their order: the pairs who, who + many, .. by
// this warp, written as output (`part` null) or as one part of the whole. A lane
// holds a part's factor; there are no more parts than warps in a block.
template <class T, int D, bool kFour>
__device__ __forceinline__ void combine(const AttentionArgs<T> &g, const Item &it, const Parts &ps, int who, int many,
                                        float *part) {
    constexpr int V = D % 128 ? 2 : 4, C = D / 32 / V;  // a lane's channels: C vectors of V
    using Vec = typename std::conditional<V == 4, float4, float2>::type;
    const int lane = threadIdx.x & 31, live = live_pairs<kFour>(it, g.group);
#pragma unroll 1
    for (int pr = who; pr < live; pr += many) {
        float m = -INFINITY, l = 0.0f;
        if (lane < ps.n) {
            const float *p = ps.at(lane) + kPairs * D + pr;
            m = p[0], l = p[kPairs];
        }
        float top = m;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float x = m == -INFINITY ? 1.0f : ex2(m - top);  // without a score a part keeps its sums: zeros, or NaN
        float sum = x * l;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        sum = __shfl_sync(0xffffffffu, sum, 0);
        float acc[C][V];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int v = 0; v < V; ++v) acc[c][v] = 0.0f;
#pragma unroll 4
        for (int i = 0; i < ps.n; ++i) {
            const float by = __shfl_sync(0xffffffffu, x, i);
            const Vec *p = reinterpret_cast<const Vec *>(ps.at(i) + pr * D) + lane;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const Vec y = p[32 * c];
                acc[c][0] = fmaf(by, y.x, acc[c][0]);
                acc[c][1] = fmaf(by, y.y, acc[c][1]);
                if constexpr (V == 4) {
                    acc[c][2] = fmaf(by, y.z, acc[c][2]);
                    acc[c][3] = fmaf(by, y.w, acc[c][3]);
                }
            }
        }
        if (part) {
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int v = 0; v < V; ++v) __stcg(part + pr * D + (32 * c + lane) * V + v, acc[c][v]);
            if (lane == 0) {
                __stcg(part + kPairs * D + pr, top);
                __stcg(part + kPairs * D + kPairs + pr, sum);
            }
        } else if (T *out = pair_output<T, D, kFour>(g, it, pr)) {
            const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int v = 0; v < V; ++v) stf(out + (32 * c + lane) * V + v, sum != 0.0f ? acc[c][v] * inv : 0.0f);
        }
    }
}

// The same for parts that blocks left in memory, into the output. A warp takes a
// pair, and the loads of a run of parts travel together, their maxima and sums
// with them: what this costs is its loads' latency (one stream of 32768 tokens: 28 us so, 35 us with a pass over the
// maxima first and four loads at a time). Both joins are inlined: handed over in
// local memory, their arguments cost the 64 streams 10 us of 86.
template <class T, int D, bool kFour, int NW>
__device__ __forceinline__ void combine_blocks(const AttentionArgs<T> &g, const Item &it, const Parts &ps, int warp) {
    constexpr int CH = D / 32;  // a lane's channels
    constexpr int V = CH % 4 == 0 ? 4 : CH % 2 == 0 ? 2 : 1, RUN = CH <= 2 ? 16 : 8;
    using Vec = typename std::conditional<V == 4, float4, typename std::conditional<V == 2, float2, float>::type>::type;
    const int lane = threadIdx.x & 31;
#pragma unroll 1
    for (int pr = warp; pr < pass_pairs<kFour>(); pr += NW) {
        const int from = pr * D;
        T *out = pair_output<T, D, kFour>(g, it, pr);
        if (!out) continue;
        float acc[CH], top = -INFINITY, sum = 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) acc[c] = 0.0f;
#pragma unroll 1
        for (int i0 = 0; i0 < ps.n; i0 += RUN) {
            const int n = min(RUN, ps.n - i0);
            float m = -INFINITY, l = 0.0f;
            if (lane < n) {
                const float *p = ps.at(i0 + lane) + kPairs * D + pr;
                m = __ldcg(p), l = __ldcg(p + kPairs);
            }
            Vec y[RUN][CH / V];
#pragma unroll
            for (int i = 0; i < RUN; ++i)
                if (i < n)
#pragma unroll
                    for (int c = 0; c < CH / V; ++c)
                        y[i][c] = __ldcg(reinterpret_cast<const Vec *>(ps.at(i0 + i) + from) + 32 * c + lane);
            float most = m;
#pragma unroll
            for (int o = 1; o < RUN; o <<= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
            most = fmaxf(top, __shfl_sync(0xffffffffu, most, 0));
            const float keep = top == -INFINITY ? 1.0f : ex2(top - most);
            top = most;
            const float x = m == -INFINITY ? 1.0f : ex2(m - top);  // without a score a part keeps its sums: zeros, or NaN
            float add = x * l;
#pragma unroll
            for (int o = 1; o < RUN; o <<= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
            sum = fmaf(sum, keep, __shfl_sync(0xffffffffu, add, 0));
#pragma unroll
            for (int c = 0; c < CH; ++c) acc[c] *= keep;
#pragma unroll
            for (int i = 0; i < RUN; ++i) {
                const float by = __shfl_sync(0xffffffffu, x, i);
                if (i < n)
#pragma unroll
                    for (int c = 0; c < CH; ++c)
                        acc[c] = fmaf(by, reinterpret_cast<const float *>(&y[i][c / V])[c % V], acc[c]);
            }
        }
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
#pragma unroll
        for (int c = 0; c < CH; ++c) stf(out + (c / V * 32 + lane) * V + c % V, sum != 0.0f ? acc[c] * inv : 0.0f);
    }
}

template <class T, int D, bool kFour>
__device__ __forceinline__ void finish(const AttentionArgs<T> &g, const Item &it, const Sums<D> &r) {
    constexpr int W = D / 64;
    const int lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        const uint32_t bad = __shfl_sync(0xffffffffu, r.bad, 8 * lt + 4 * c);
        const float l = __shfl_sync(0xffffffffu, r.l, 8 * lt + 4 * c);
        T *out = pair_output<T, D, kFour>(g, it, 2 * lt + c);
        const float inv = l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            float v[8];
            lane_values<D>(r, w, c, bad, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = l != 0.0f ? v[e] * inv : 0.0f;
            if (out) store8(out + 8 * (W * lg + w), v, g.vec_out);
        }
    }
}

// The line of all items' tiles and this warp's cut of it. Where every item can
// have blocks of its own without longer cuts, items are padded to whole blocks,
// so that few or none are divided between blocks.
struct Cut {
    int share, block;       // tiles of a warp, of a block
    bool padded;
    int begin, end;         // this warp's
    int stream, stream_at;  // the stream that it begins in, and where that begins
    StreamWork sw;          // of that stream
};

__device__ __forceinline__ int line_tiles(const PagedArgs &a, const StreamWork &w, const Cut &c) {
    const int items = w.passes * a.kv_heads;
    return items * (c.padded ? (w.tiles + c.block - 1) / c.block * c.block : w.tiles);
}

__device__ __forceinline__ int inclusive(int v) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, v, o);
        if (int(threadIdx.x & 31) >= o) v += y;
    }
    return v;
}

// Every warp finds its cut by itself: a lane adds up a run of streams, the lane
// whose run the cut begins in is found, then the stream in the run.
template <int NW, int kPass>
__device__ __forceinline__ bool find_cut(const PagedArgs &a, int group, int window, int min_share, Cut &c) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, per = (a.streams + 31) / 32;
    const int b0 = min(lane * per, a.streams), b1 = min(b0 + per, a.streams);
    c.padded = false;
    int mine = 0;
    StreamWork w;
    for (int b = b0; b < b1; ++b) {
        w = stream_work(a, b, group, window, kPass);
        mine += line_tiles(a, w, c);
    }
    const int total = __reduce_add_sync(0xffffffffu, mine), warps_all = int(gridDim.x) * NW;
    c.share = max((total + warps_all - 1) / warps_all, min_share);
    c.share += c.share & 1;  // tiles go in twos
    c.block = NW * c.share;
    int blocks = 0;  // at most the tiles, so no overflow
    for (int b = b0; b < b1; ++b) {
        if (per > 1) w = stream_work(a, b, group, window, kPass);
        blocks += w.passes * a.kv_heads * ((w.tiles + c.block - 1) / c.block);
    }
    c.padded = __reduce_add_sync(0xffffffffu, blocks) <= int(gridDim.x);
    if (c.padded) mine = blocks * c.block;
    const int incl = inclusive(mine), line = __shfl_sync(0xffffffffu, incl, 31);
    const int block_begin = int(min(int64_t(blockIdx.x) * c.block, int64_t(line)));
    if (block_begin >= line) return false;
    c.begin = min(block_begin + warp * c.share, line);
    c.end = min(c.begin + c.share, line);
    if (c.begin >= c.end) return true;
    int k = __ffs(__ballot_sync(0xffffffffu, incl > c.begin)) - 1;  // the run, then the lane that has the stream
    c.stream_at = __shfl_sync(0xffffffffu, incl - mine, k);
    c.stream = k * per;
    while (per > 1) {
        const int b = c.stream + lane;
        w = stream_work(a, min(b, a.streams - 1), group, window, kPass);
        const int tiles = b < a.streams ? line_tiles(a, w, c) : 0;
        const int upto = c.stream_at + inclusive(tiles);
        const uint32_t past = __ballot_sync(0xffffffffu, upto > c.begin);
        if (past) {
            k = __ffs(past) - 1;
            c.stream += k;
            c.stream_at = __shfl_sync(0xffffffffu, upto - tiles, k);
            break;
        }
        c.stream += 32;
        c.stream_at = __shfl_sync(0xffffffffu, upto, 31);
    }
    c.sw.begin = __shfl_sync(0xffffffffu, w.begin, k), c.sw.rows = __shfl_sync(0xffffffffu, w.rows, k);
    c.sw.length = __shfl_sync(0xffffffffu, w.length, k), c.sw.first_tile = __shfl_sync(0xffffffffu, w.first_tile, k);
    c.sw.tiles = __shfl_sync(0xffffffffu, w.tiles, k), c.sw.passes = __shfl_sync(0xffffffffu, w.passes, k);
    return true;
}

template <class T, int D, bool kFour>
__global__ void __launch_bounds__(warps<D>() * 32, 1) paged_attention_kernel(const __grid_constant__ AttentionArgs<T> g) {
    constexpr int NW = warps<D>(), PF = part_floats<D>();
    // of each warp: its ring, which then takes the item that it left, and the item that it found begun
    extern __shared__ __align__(128) float smem[];
    constexpr int WF = warp_floats<D>(), RF = ring_floats<D>();
    __shared__ Item merge_item[2];
    __shared__ int merge_first[2], merge_last[2], is_last[2];
    pdl_trigger();
    pdl_wait();
    const PagedArgs &a = g.a;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Cut cut;
    if (!find_cut<NW, pass_pairs<kFour>()>(a, g.group, g.window, g.min_share, cut)) return;
    if (threadIdx.x < 2) merge_first[threadIdx.x] = -1;

    float *tail_slot = smem + warp * WF, *head_slot = tail_slot + RF;
    Item it, head;
    bool has_head = false, has_tail = false;
    if (cut.begin < cut.end) {
        it.stream = cut.stream;
        it.sw = cut.sw;
        int x = cut.begin;
        while (x < cut.end) {
            const int items = it.sw.passes * a.kv_heads;
            const int span = cut.padded ? (it.sw.tiles + cut.block - 1) / cut.block * cut.block : it.sw.tiles;
            if (x >= cut.stream_at + span * items) {
                cut.stream_at += span * items;
                it.sw = stream_work(a, ++it.stream, g.group, g.window, pass_pairs<kFour>());
                continue;
            }
            const int index = (x - cut.stream_at) / span;
            it.kvh = index / it.sw.passes;
            it.pass = index - it.kvh * it.sw.passes;
            it.at = cut.stream_at + index * span;
            it.tiles = it.sw.tiles;
            const int stop = min(it.at + it.tiles, cut.end);
            if (x >= stop) break;  // padding
            Sums<D> r;
            walk<T, D, kFour>(g, it, x - it.at, stop - it.at, reinterpret_cast<uint8_t *>(tail_slot), r);
            has_tail = it.at >= x && it.at + it.tiles > cut.end;
            if (it.at < x) {
                head = it;
                has_head = true;
            }
            if (it.at < x || has_tail) {
                __syncwarp();
                deposit<D>(r, has_tail ? tail_slot : head_slot);
            } else {
                finish<T, D, kFour>(g, it, r);
            }
            x = stop;
        }
    }
    __syncthreads();

    // An item that cuts divide is added up by the warps that hold parts of it.
    const int block_begin = int(blockIdx.x) * cut.block, block_end = block_begin + cut.block;
    bool divided = false;
#pragma unroll 1
    for (int e = 0; e < 2; ++e) {
        if (!(e ? has_tail : has_head)) continue;
        const Item c = e ? it : head;
        const int end = c.at + c.tiles;
        const bool here = c.at >= block_begin, whole = here && end <= block_end;
        const int lead = here ? (c.at - block_begin) / cut.share : 0;
        Parts ps;
        ps.first = smem + lead * WF + (here ? 0 : RF);
        ps.rest = smem + lead * WF + RF;
        ps.stride = WF;
        ps.n = (min(end, block_end) - block_begin + cut.share - 1) / cut.share - lead;
        // slot 0 of a block: an item that began in an earlier one, slot 1: in it
        combine<T, D, kFour>(g, c, ps, warp - lead, ps.n,
                      whole ? nullptr : g.parts + (2 * int64_t(blockIdx.x) + here) * PF);
        if (!whole) {
            divided = true;
            if (warp == lead && lane == 0) {
                merge_item[here] = c;
                merge_first[here] = c.at / cut.block;
                merge_last[here] = (end - 1) / cut.block;
            }
        }
    }
    if (divided) __threadfence();
    if (!__syncthreads_or(divided)) return;
    if (threadIdx.x < 2 && merge_first[threadIdx.x] >= 0) {
        const int slot = threadIdx.x, parts = merge_last[slot] - merge_first[slot] + 1;
        is_last[slot] = atomicAdd(g.tickets + merge_first[slot], 1u) == uint32_t(parts - 1);
        if (is_last[slot]) g.tickets[merge_first[slot]] = 0;
    }
    __syncthreads();
    // the block that comes last to an item adds up the blocks' parts
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
        if (merge_first[slot] < 0 || !is_last[slot]) continue;
        __threadfence();
        Parts ps;
        ps.first = g.parts + (2 * int64_t(merge_first[slot]) + 1) * PF;
        ps.rest = ps.first - PF;
        ps.stride = 2 * PF;
        ps.n = merge_last[slot] - merge_first[slot] + 1;
        combine_blocks<T, D, kFour, NW>(g, merge_item[slot], ps, warp);
    }
}

uint64_t ticket_bytes() { return (uint64_t(device_sm_count()) * 4 + 255) / 256 * 256; }

template <class T, int D, bool kFour>
si_status launch(const AttentionArgs<T> &g, void *stream) {
    constexpr int NW = warps<D>();
    const double tiles = double(int64_t(g.a.table_width) << (g.a.page_shift - 4));
    constexpr int kPass = pass_pairs<kFour>();
    const double passes = double((g.a.rows * g.group + kPass - 1) / kPass + g.a.streams);
    const double most = tiles * passes * g.a.kv_heads;
    if (most > double(INT32_MAX / 2))
        return fail(SI_ERR_UNSUPPORTED, "paged-attention: rows times the table's tokens exceed 2^30 tiles.");
    // blocks of their own for all items, if there are so many
    const double blocks = passes * g.a.kv_heads * double(int64_t(tiles + NW * g.min_share - 1) / (NW * g.min_share));
    const unsigned grid = unsigned(blocks < device_sm_count() ? blocks : device_sm_count());
    return launch_pdl("paged-attention", paged_attention_kernel<T, D, kFour>, dim3(grid), dim3(NW * 32),
                      size_t(NW) * warp_floats<D>() * 4, 1, stream, g);
}

template <class T, bool kFour>
si_status launch_size(const AttentionArgs<T> &g, void *stream) {
    switch (g.a.head_size) {
    case 64: return launch<T, 64, kFour>(g, stream);
    case 128: return launch<T, 128, kFour>(g, stream);
    case 192: return launch<T, 192, kFour>(g, stream);
    default: return launch<T, 256, kFour>(g, stream);
    }
}

// Bytes of the blocks' parts (two to a block), then of the sums that their warps put away.
uint64_t part_bytes(int head_size) { return uint64_t(device_sm_count()) * 2 * kPairs * (uint64_t(head_size) + 2) * 4; }
uint64_t held_bytes(int head_size) {
    return uint64_t(device_sm_count()) * (head_size <= 128 ? warps<128>() : warps<256>()) * kPairs * uint64_t(head_size) * 4;
}

template <class T>
si_status run(const PagedArgs &a, const PagedAttention &q, void *stream) {
    const int capacity = a.table_width << a.page_shift;
    uint8_t *const parts = static_cast<uint8_t *>(q.workspace) + ticket_bytes();
    const AttentionArgs<T> g{a, static_cast<const T *>(q.query), static_cast<T *>(q.output), q.query_stride,
                             q.output_stride, q.query_heads, q.query_heads / a.kv_heads,
                             q.window < capacity ? q.window : 0, 2, q.scale * 1.44269504088896340736f,
                             whole8<T>(q.query, q.query_stride * int64_t(sizeof(T))),
                             whole8<T>(q.output, q.output_stride * int64_t(sizeof(T))),
                             static_cast<uint32_t *>(q.workspace), reinterpret_cast<float *>(parts),
                             reinterpret_cast<float4 *>(parts + part_bytes(a.head_size)), device_sm_count(), 1};
    if (int64_t(q.max_rows) * g.group > kFewPairs) return paged_chunk_attention(g, stream);
    if (sizeof(T) == 4 && int64_t(q.max_rows) * g.group <= pass_pairs<true>()) return launch_size<T, sizeof(T) == 4>(g, stream);
    return launch_size<T, false>(g, stream);
}

}  // namespace

uint64_t paged_attention_workspace(const PagedArgs &a, int64_t, int max_rows, int query_heads) {
    if (int64_t(max_rows) * (query_heads / a.kv_heads) > kFewPairs) return ticket_bytes() + paged_chunk_workspace(a.head_size);
    return ticket_bytes() + part_bytes(a.head_size) + held_bytes(a.head_size);
}

si_status paged_attention(const PagedArgs &a, uint32_t type, const PagedAttention &q, void *stream) {
    return type == SI_TYPE_F32 ? run<float>(a, q, stream) : run<__half>(a, q, stream);
}

}  // namespace si::kernels
