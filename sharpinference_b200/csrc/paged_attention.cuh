// What the kernels of attention over the paged 4-bit cache share: their
// arguments, unpacking, and a stream's share of the work.
#pragma once

#include "device_common.cuh"
#include "paged.cuh"

namespace si::dev {

constexpr float kOwned = 0x1p-16f; // share of all other tokens in a row that one token owns

template <class T>
struct AttentionArgs {
    PagedArgs a;
    const T *query;
    T *output;
    int64_t query_stride, output_stride;
    int query_heads, group, window;
    int min_share;  // tiles of a warp at least, while there are blocks to spare (2; 4 costs 1 us on 4096 tokens)
    float scale;    // of the scores, times log2(e)
    bool vec, vec_out;  // whole accesses of eight: query rows, output rows
    uint32_t *tickets;  // [slots], zero between calls
    float *parts;
    float4 *held;       // [blocks][warps][4 words of a lane's values][lanes]: sums that left a warp's accumulators
    int slots;          // SMs
    int splits;         // parts of a block's tokens (prompt chunks)
};

__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<const uint32_t *>(&h); }
__device__ __forceinline__ __half2 u2h(uint32_t u) { return *reinterpret_cast<const __half2 *>(&u); }

// Nibble I of both halves of x times the scales s, off = -24 s: exact.
template <int I>
__device__ __forceinline__ uint32_t unpack(uint32_t x, __half2 s, __half2 off) {
    const uint32_t at = I == 0 ? x << 6 : I == 1 ? x << 2 : I == 2 ? x >> 2 : x >> 6;
    uint32_t h;  // (at & 0x03C003C0) | 0x4C004C00, one instruction
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(h) : "r"(at), "r"(0x03C003C0u), "r"(0x4C004C00u));
    return h2u(__hfma2(u2h(h), s, off));
}

// Bits 15 and 31: whether the halves are a NaN or an infinity.
__device__ __forceinline__ uint32_t not_finite(uint32_t halves) { return (halves & 0x7C007C00u) + 0x04000400u; }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A stream's share of the work: its rows make ceil(n * group / pairs) passes per
// key/value head over the tiles of 16 tokens that any of them sees.
struct StreamWork {
    int begin, rows, length, first_tile, tiles, passes;
};

__device__ __forceinline__ StreamWork stream_work(const PagedArgs &a, int b, int group, int window, int pairs) {
    StreamWork w;
    w.begin = stream_start(a.row_starts, b, a.rows);
    w.rows = max(stream_start(a.row_starts, b + 1, a.rows) - w.begin, 0);
    w.length = max(a.lengths[b], 0);
    const int capacity = a.table_width << a.page_shift;
    const int first = window ? max(0, w.length - w.rows - window + 1) : 0;
    w.first_tile = first >> 4;
    w.tiles = w.rows ? max((min(w.length, capacity) + 15) / 16 - w.first_tile, 0) : 0;
    // rows that see no tile still get their zeros
    w.tiles = w.rows ? max(w.tiles, 1) : 0;
    w.passes = (w.rows * group + pairs - 1) / pairs;
    return w;
}

}  // namespace si::dev

namespace si::kernels {
// Prompt chunks (paged_chunk.cu), and the bytes behind AttentionArgs::parts that they need.
uint64_t paged_chunk_workspace(int head_size);
si_status paged_chunk_attention(const dev::AttentionArgs<float> &g, void *stream);
si_status paged_chunk_attention(const dev::AttentionArgs<__half> &g, void *stream);
}  // namespace si::kernels
