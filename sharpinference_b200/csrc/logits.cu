// Penalties, biases and token masks of logits, and the greedy pick.
#include <cooperative_groups.h>

#include <algorithm>

#include "device_common.cuh"
#include "launch.cuh"

namespace si::kernels {
namespace {

using namespace si::dev;
namespace cg = cooperative_groups;

constexpr int kTokens = 16;      // of a thread in a chunk: 8 bytes of shared memory each
constexpr int kFewRows = 4;
constexpr int kBatch = 8;        // list entries of a thread on the way at a time

template <class T>
struct LogitArgs {
    const T *logits;
    T *output;
    int32_t *next;
    int64_t stride, output_stride, vocab;
    int chunk;  // tokens a block takes at a time, a multiple of 128
    si_logit_controls c;
};

// [begin, end) of a row's list, bounded to the list.
__device__ __forceinline__ void list_range(const int32_t *starts, int64_t row, int64_t count, int64_t &begin,
                                           int64_t &end) {
    begin = end = 0;
    if (!starts) return;
    begin = max(int64_t(starts[row]), int64_t(0));
    end = min(int64_t(starts[row + 1]), count);
}

// VEC neighbouring logits, one access where VEC is 4.
template <int VEC>
__device__ __forceinline__ void load_logits(const float *p, float (&x)[VEC]) {
    if constexpr (VEC == 4) {
        const float4 v = *reinterpret_cast<const float4 *>(p);
        x[0] = v.x, x[1] = v.y, x[2] = v.z, x[3] = v.w;
    } else {
        x[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void load_logits(const __half *p, float (&x)[VEC]) {
    if constexpr (VEC == 4) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&v.x)),
                     b = __half22float2(*reinterpret_cast<const __half2 *>(&v.y));
        x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y;
    } else {
        x[0] = __half2float(*p);
    }
}
template <int VEC>
__device__ __forceinline__ void store_logits(float *p, const float (&x)[VEC]) {
    if constexpr (VEC == 4) *reinterpret_cast<float4 *>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else *p = x[0];
}
template <int VEC>
__device__ __forceinline__ void store_logits(__half *p, const float (&x)[VEC]) {
    if constexpr (VEC == 4) {
        const __half2 a = __floats2half2_rn(x[0], x[1]), b = __floats2half2_rn(x[2], x[3]);
        *reinterpret_cast<uint2 *>(p) =
            make_uint2(*reinterpret_cast<const uint32_t *>(&a), *reinterpret_cast<const uint32_t *>(&b));
    } else {
        *p = __float2half_rn(x[0]);
    }
}

// One cluster per row; its blocks take the vocabulary in chunks. A chunk's
// history counts and last bias entries are tables in shared memory with one bit
// for every token that either has; the pass over the logits looks at the bits
// and, where one is set, at the tables, which it leaves cleared for the next
// chunk. Bound: the logits' bytes; a chunk's logits are on the way to registers
// while its lists are counted. 128 rows of 100352 FP32 logits with 3000 tokens of
// history, 50 biases and masks: 40.7 us, 2.6 TB/s; held by issue (50 % of slots:
// tests of bits, the few listed tokens' arithmetic) and the chunks' barriers.
// VEC 4: rows on 16-byte boundaries (8 for F16) and vocab a multiple of 4.
template <class T, int VEC, int kThreads>
__global__ void __launch_bounds__(kThreads, 1024 / kThreads) process_logits_kernel(const LogitArgs<T> g) {
    constexpr int kMaxChunk = kTokens * kThreads;
    extern __shared__ __align__(16) uint32_t count[];  // [chunk], then bias entries + 1 [chunk]
    __shared__ uint32_t listed[kMaxChunk / 32];        // a bit for every token
    __shared__ unsigned long long best_of[kThreads / 32];
    __shared__ unsigned long long block_best;
    cg::cluster_group cluster = cg::this_cluster();
    pdl_trigger();
    pdl_wait();
    constexpr int kStep = kThreads * VEC, kLoads = VEC == 4 ? kMaxChunk / kStep : 8;
    const int ranks = int(cluster.num_blocks()), rank = int(cluster.block_rank()), tid = threadIdx.x, lane = tid & 31;
    const int64_t row = blockIdx.x / ranks;
    const si_logit_controls &c = g.c;
    int64_t hb, he, bb, be;
    list_range(c.history ? c.history_starts : nullptr, row, c.history_count, hb, he);
    list_range(c.bias_tokens ? c.bias_starts : nullptr, row, c.bias_count, bb, be);
    const int32_t *history = c.history + hb, *bias_tokens = c.bias_tokens + bb;
    const float *bias_values = c.bias_values + bb;
    const int seen = int(max(he - hb, int64_t(0))), biases = int(max(be - bb, int64_t(0)));
    const bool lists = seen > 0 || biases > 0;
    const float rep = c.repetition ? c.repetition[row] : 1.0f, freq = c.frequency ? c.frequency[row] : 0.0f,
                pres = c.presence ? c.presence[row] : 0.0f;
    const uint32_t *mask = nullptr;
    if (c.allowed) {
        const int64_t m = c.allowed_index ? int64_t(c.allowed_index[row]) : row;
        if (m >= 0 && m < c.allowed_rows) mask = c.allowed + m * c.allowed_stride;
    }
    uint32_t *entry = count + g.chunk;
    if (lists) {
        for (int v = 4 * tid; v < 2 * g.chunk; v += 4 * kThreads)
            *reinterpret_cast<uint4 *>(count + v) = make_uint4(0, 0, 0, 0);
        for (int v = tid; v < kMaxChunk / 32; v += kThreads) listed[v] = 0;
    }
    float best = -INFINITY;
    uint32_t best_at = 0;
    for (int64_t c0 = int64_t(rank) * g.chunk; c0 < g.vocab; c0 += int64_t(ranks) * g.chunk) {
        const int n = int(min(int64_t(g.chunk), g.vocab - c0));
        const T *in = g.logits + row * g.stride + c0;
        T *out = g.output ? g.output + row * g.output_stride + c0 : nullptr;
        const uint32_t *words = mask ? mask + (c0 >> 5) : nullptr;
        float x[kLoads][VEC];
        uint32_t bits[kLoads];
        auto fetch = [&](int b) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int v = b + i * kStep;
                bits[i] = 0xffffffffu;
                if (v < n) {
                    load_logits<VEC>(in + v, x[i]);
                    if (words) bits[i] = words[v >> 5];
                }
            }
        };
        fetch(VEC * tid);
        if (lists) {
            __syncthreads();  // the tables are clear
            // those of a list's tokens that are in the chunk, a batch of loads ahead
            auto each = [&](const int32_t *tokens, int many, auto &&f) {
                for (int b = tid; b < many; b += kBatch * kThreads) {
                    uint32_t v[kBatch];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        v[i] = b + i * kThreads < many ? uint32_t(tokens[b + i * kThreads]) - uint32_t(c0) : 0xffffffffu;
#pragma unroll
                    for (int i = 0; i < kBatch; ++i)
                        if (v[i] < uint32_t(n)) {
                            f(v[i], b + i * kThreads);
                            atomicOr(listed + (v[i] >> 5), 1u << (v[i] & 31));
                        }
                }
            };
            each(history, seen, [&](uint32_t v, int) { atomicAdd(count + v, 1u); });
            each(bias_tokens, biases, [&](uint32_t v, int i) { atomicMax(entry + v, uint32_t(i) + 1u); });
            __syncthreads();
        }
        for (int b = VEC * tid;; ) {
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const int v = b + i * kStep;
                if (v >= n) continue;
                const uint32_t hits = lists ? listed[v >> 5] >> (v & 31) : 0u, allowed = bits[i] >> (v & 31);
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    if ((hits >> e) & 1u) {
                        float y = x[i][e];
                        if (const uint32_t k = count[v + e]) {
                            y = y > 0.0f ? __fdiv_rn(y, rep) : __fmul_rn(y, rep);
                            y = __fsub_rn(__fsub_rn(y, __fmul_rn(freq, float(k))), pres);
                            count[v + e] = 0;
                        }
                        if (const uint32_t k = entry[v + e]) {
                            y = __fadd_rn(y, bias_values[k - 1]);
                            entry[v + e] = 0;
                        }
                        x[i][e] = y;
                    }
                    if (!((allowed >> e) & 1u)) x[i][e] = -INFINITY;
                    if (x[i][e] > best) {  // never for NaN; a thread's tokens come in their order
                        best = x[i][e];
                        best_at = uint32_t(c0) + uint32_t(v + e);
                    }
                }
                if (out) store_logits<VEC>(out + v, x[i]);
            }
            b += kLoads * kStep;
            if (b - VEC * tid >= n) break;
            fetch(b);
        }
        if (lists) {
            __syncthreads();  // the chunk's bits are no longer read
            for (int v = tid; v < kMaxChunk / 32; v += kThreads) listed[v] = 0;
        }
    }
    if (!g.next) return;
    unsigned long long key = 0;  // larger value first (-0 counts as +0), then the smaller token
    if (best > -INFINITY) {
        const uint32_t u = __float_as_uint(best + 0.0f), order = u & 0x80000000u ? ~u : u | 0x80000000u;
        key = (static_cast<unsigned long long>(order) << 32) | (0xffffffffu - best_at);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
    if (lane == 0) best_of[tid >> 5] = key;
    __syncthreads();
    if (tid < 32) {
        key = tid < kThreads / 32 ? best_of[tid] : 0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) key = max(key, __shfl_xor_sync(0xffffffffu, key, o));
        if (tid == 0) block_best = key;
    }
    cluster.sync();
    if (rank == 0 && tid == 0) {
        for (int r = 1; r < ranks; ++r) key = max(key, *cluster.map_shared_rank(&block_best, r));
        g.next[row] = key ? int32_t(0xffffffffu - uint32_t(key)) : -1;
    }
    cluster.sync();  // no block leaves while its shared memory is read
}

template <class T, int VEC, int kThreads>
si_status launch(LogitArgs<T> &g, int64_t rows, void *stream) {
    constexpr int kMaxChunk = kTokens * kThreads;
    // as many blocks to a row (16 is beyond the portable 8) as run at once: a second wave would pay every block's
    // start again (128 rows of 100352: 39.5 us, 45.6 with four blocks to a row; one row of 200064: 8.5 us, 11.4 with 8)
    const int64_t room = int64_t(1024 / kThreads) * device_sm_count() / rows;
    const int64_t want = std::min<int64_t>(room, (g.vocab + 2047) / 2048);
    const int cluster = int(want >= 16 ? 16 : std::max<int64_t>(1, std::min<int64_t>(want, 8)));
    if (cluster > 8)
        if (const int e = allow_cluster_16(reinterpret_cast<const void *>(process_logits_kernel<T, VEC, kThreads>)))
            return cuda_error(e, "process-logits");
    const int64_t per_round = int64_t(cluster) * kMaxChunk, rounds = (g.vocab + per_round - 1) / per_round;
    const int64_t share = (g.vocab + cluster * rounds - 1) / (cluster * rounds);
    g.chunk = int((share + 127) / 128 * 128);
    return launch_pdl("process-logits", process_logits_kernel<T, VEC, kThreads>, dim3(unsigned(rows * cluster)), dim3(kThreads),
                      size_t(g.chunk) * 8, cluster, stream, g);
}

// Few rows of a vocabulary that 16 blocks of 512 threads take in two chunks: blocks twice as large, one to an SM,
// take it in one (200064 tokens, one row 8.6 us against 9.3, four rows 8.7 against 10.2; eight such clusters do
// not run at once: 17.0 against 12.0; 32064 tokens, one row 6.7 against 6.0).
template <class T, int VEC>
si_status launch_threads(LogitArgs<T> &g, int64_t rows, void *stream) {
    return rows <= kFewRows && g.vocab > 16 * 512 * kTokens ? launch<T, VEC, 1024>(g, rows, stream) : launch<T, VEC, 512>(g, rows, stream);
}

template <class T>
si_status run(const void *logits, int64_t stride, const si_logit_controls &c, void *output, int64_t output_stride,
              int32_t *next, int64_t rows, int64_t vocab, void *stream) {
    LogitArgs<T> g{static_cast<const T *>(logits), static_cast<T *>(output), next, stride, output_stride, vocab, 0, c};
    auto wide = [](const void *p, int64_t row) { return reinterpret_cast<uintptr_t>(p) % (4 * sizeof(T)) == 0 && row % 4 == 0; };
    if (vocab % 4 == 0 && wide(logits, stride) && (!output || wide(output, output_stride)))
        return launch_threads<T, 4>(g, rows, stream);
    return launch_threads<T, 1>(g, rows, stream);
}

}  // namespace

si_status process_logits(uint32_t type, const void *logits, int64_t stride, const si_logit_controls &c, void *output,
                         int64_t output_stride, int32_t *next, int64_t rows, int64_t vocab, void *stream) {
    return type == SI_TYPE_F32 ? run<float>(logits, stride, c, output, output_stride, next, rows, vocab, stream)
                               : run<__half>(logits, stride, c, output, output_stride, next, rows, vocab, stream);
}

}  // namespace si::kernels
