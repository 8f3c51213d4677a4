// Attention over the paged 4-bit cache for many rows: prompt chunks.
//
// Bound: the tensor pipe, then the issue of what feeds it. A block takes 256
// pairs of a row and a query head of one stream and key/value head (128 for
// head sizes above 128: tensor memory) as groups of 128 and walks the tokens
// that any of them sees, 64 at a time. For each group
//   S[128, 64] = Q K^T   tcgen05.mma, both operands in shared memory;
//   P = 2^(scale S - m)  by 128 threads, a row each, back into tensor memory
//                        over S as F16 (F32 calls: also what rounding left);
//   O[128, D] += P V     tcgen05.mma with P from tensor memory.
// Cached values are F16 numbers, so K and V are unpacked without a rounding,
// once for both groups: two warps write K as [token][channel], four V
// transposed as [channel][token] (eight tokens of one word give eight 16-byte
// runs), both in the 128-byte swizzled layout. F32 queries are two F16 numbers,
// products with both added in the same accumulator; F16 calls round probabilities
// to one F16 number (relative error of 4096 rows on 8192 tokens 2.7e-4, of which
// rounding the outputs is 2.1e-4). Running maxima move only
// when a score exceeds them by 2^7; then the row's O is scaled in tensor memory.
// One group's exponentials run under the other's products. Blocks start with
// the rows that see most. Measured: 4096 rows on 8192 tokens (24 query, 8
// key/value heads of 128) F16 391 us, 0.79 PFLOP/s; F32, 3 chunks of up to 777
// rows on 1500 tokens (40, 10 heads) 120 us.
//
// While there are fewer blocks than SMs, each block's tokens are cut into parts
// of two steps or more, for as many blocks as fit; a part's sums lie in its slot of
// the workspace and a second launch joins them. 16 rows of 4 heads a key/value
// head on 32768 tokens, 4 key/value heads, F32: 50 us, 758 uncut; on 4096: 27 and 105.
//
// Every wait is bounded (device error word, no trap): a thread whose wait runs
// out leaves its loop, and the block frees its tensor memory and ends.
#include <algorithm>

#include "launch.cuh"
#include "paged_fragments.cuh"

namespace si::kernels {
namespace {

using namespace si::dev;

constexpr int kRows = 128;   // pairs of a group: MMA M, tensor memory lanes
constexpr int kTokens = 64;  // of one step: N of the scores, K of the values
// tcgen05 aligns the sum and 16 products to the largest of them, cuts each towards zero 25 places below that, and
// cuts what they add up to 23 places below itself (that gives the kernel's sums to 0.5 of 2^-23 in the mean). F32
// calls put back what the second cut loses: half a last place in the mean, for a value of mantissa m in [1, 2)
// 2^-24 / m of itself, and m with density 1 / (m ln 2) gives 2^-24 / (2 ln 2); a sum that n additions build up from
// nothing loses that for every value on its way, n / 2 times its last one. The first cut goes by each product's sign:
// little where signs are mixed, but as much again where all products of 1024 tokens have one (2.5e-6 of their sum
// stays lost; a factor that put that back too would be 2.4e-6 too large for mixed signs).
constexpr float kTruncated = 0.72134752f * 0x1p-24f;
constexpr float kSlack = 7.0f;  // log2 of what a score may exceed the running maximum by (2 makes chunks 8 to 11 % slower)
constexpr float kLift = 8.0f;   // log2 of a probability at the maximum: F16 keeps more small ones
constexpr int kMostParts = 32;
constexpr int kUnpackK = 64, kUnpackV = 128;  // threads: with the rest 16 warps, which leaves 128 registers to each

template <class T, int D>
struct Chunk {
    static constexpr bool kWide = sizeof(T) == 4;
    static constexpr int kGroups = D <= 128 ? 2 : 1;
    // F32 calls take O out of tensor memory every so many steps and add it up rounded, in a slot of the workspace
    // ([four channels][row]) for every block that runs, since what truncation loses
    // grows with the tokens (6.5e-5 of O at 32768 without either, 3.8e-6 with this, 1.9e-6 with kTruncated too; at
    // 2048 tokens 4.7e-6, 3.0e-6 and 1.1e-6; values of one sign at 32768 2e-4 without either, 5.3e-6, 2.5e-6). Three
    // chunks of up to 777 rows on 1500 tokens (40 query heads, 10 of 128) take 119 us so, 138 with 8 steps, 154 with
    // 4, 114 with 32
    static constexpr int kFlush = 16;
    static constexpr int kSoftmax = kGroups * kRows, kThreads = kSoftmax + kUnpackK + kUnpackV + 32 * kGroups;
    static constexpr int kMmaWarp = kThreads / 32 - kGroups;  // the first of one for every group
    static constexpr int kPart = kRows * D * 2;                  // one F16 part of a group's queries
    static constexpr int kGroupBytes = kPart * (kWide ? 2 : 1);  // and all parts
    static constexpr int kTile = kTokens * D * 2;                // K of a step, V of a step
    static constexpr int kQBytes = kGroups * kGroupBytes, kLimit = 225 * 1024;
    static constexpr int kStagesK = kQBytes + 3 * kTile <= kLimit ? 2 : 1;
    static constexpr int kStagesV = kQBytes + 4 * kTile <= kLimit ? 2 : 1;
    static constexpr int kSlot = kGroups * kRows * (D + 4);  // floats: O, then four numbers of each row
    static constexpr size_t kSmem = kQBytes + size_t(kStagesK + kStagesV) * kTile;
    // tensor memory: S / P of even and odd steps of the groups, then their O
    static constexpr int kOut = kGroups * 2 * kTokens;
    static constexpr int kColumns = kOut + kGroups * D <= 256 ? 256 : 512;
    static constexpr uint32_t kScores = (1u << 4) | (uint32_t(kTokens >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
    static constexpr uint32_t kValues = (1u << 4) | (uint32_t(D >> 3) << 17) | (uint32_t(kRows >> 4) << 24);
    static_assert(kSmem <= kLimit && kOut + kGroups * D <= 512, "shared and tensor memory");
};

// Shared-memory descriptor of a K-major tile in the 128-byte swizzled layout:
// rows of 128 B, groups of eight rows 1024 B apart.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
    return uint64_t((addr & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) |
           (uint64_t(2) << 61);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
// mbar_wait behind a test that does not suspend: the phase has mostly completed.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t parity, uint32_t err) {
    uint32_t done;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(smem_u32(bar)), "r"(parity)
        : "memory");
    return done || mbar_wait(bar, parity, err);
}
__device__ __forceinline__ bool elect_one() {
    uint32_t yes;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
    return yes != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Loads of tensor memory with their wait: the values are there when they return.
__device__ __forceinline__ void tm_load16(uint32_t t, uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15"
        "}, [%16];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tm_load32(uint32_t t, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31"
        "}, [%32];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tm_load64(uint32_t t, uint32_t (&v)[64]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
        "}, [%64];\n tcgen05.wait::ld.sync.aligned;"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31]),
          "=r"(v[32]), "=r"(v[33]), "=r"(v[34]), "=r"(v[35]), "=r"(v[36]), "=r"(v[37]), "=r"(v[38]), "=r"(v[39]),
          "=r"(v[40]), "=r"(v[41]), "=r"(v[42]), "=r"(v[43]), "=r"(v[44]), "=r"(v[45]), "=r"(v[46]), "=r"(v[47]),
          "=r"(v[48]), "=r"(v[49]), "=r"(v[50]), "=r"(v[51]), "=r"(v[52]), "=r"(v[53]), "=r"(v[54]), "=r"(v[55]),
          "=r"(v[56]), "=r"(v[57]), "=r"(v[58]), "=r"(v[59]), "=r"(v[60]), "=r"(v[61]), "=r"(v[62]), "=r"(v[63])
        : "r"(t)
        : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t t, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            t),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
        "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
        : "memory");
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void put16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// What one unpacking thread loads of a step: a token's key words, or
// words of eight tokens' values.
template <int D>
struct RawK {
    static constexpr int NG = D / 32;
    uint32_t w[4 * NG], s[NG / 2];
};
template <int D>
struct RawV {
    static constexpr int NG = D / 32, N = (NG + 3) / 4;
    uint32_t w[N][8];
    uint4 s[N];
};

__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// a * b + c and a + b of two floats at once.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)),
          "l"(reinterpret_cast<unsigned long long &>(c)));
    return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long &>(d))
        : "l"(reinterpret_cast<unsigned long long &>(a)), "l"(reinterpret_cast<unsigned long long &>(b)));
    return d;
}

__device__ __forceinline__ void add_global(float4 *at, float4 x) {
    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(x.x), "f"(x.y), "f"(x.z),
                 "f"(x.w)
                 : "memory");
}
__device__ __forceinline__ float4 fma_all(float4 a, float b, float4 c) {
    return make_float4(fmaf(a.x, b, c.x), fmaf(a.y, b, c.y), fmaf(a.z, b, c.z), fmaf(a.w, b, c.w));
}

// What one block of the chunk kernel works on.
struct Place {
    int stream, pass, kvh;
    StreamWork sw;
    int any_last, any_first;  // the tokens that any of its rows sees
    int step0, steps;         // in steps of 64; this part's
    int parts;                // that the tokens are cut into
};

// Stream and pass of the block of 256 (128) pairs `at`, later rows first, by one
// warp; stream -1 past the last.
__device__ __forceinline__ void find_pass(const PagedArgs &a, int group, int window, int pairs, int at, int &stream,
                                          int &pass) {
    const int lane = threadIdx.x & 31;
    int total = 0;
    for (int b0 = 0; b0 < a.streams; b0 += 32) {
        const int b = b0 + lane;
        total += b < a.streams ? stream_work(a, b, group, window, pairs).passes : 0;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    int left = total - 1 - at;
    stream = -1;
    if (left >= 0)
        for (int b0 = 0; b0 < a.streams; b0 += 32) {
            const int b = b0 + lane;
            const int n = b < a.streams ? stream_work(a, b, group, window, pairs).passes : 0;
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += y;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, incl > left);
            if (past) {
                const int k = __ffs(past) - 1;
                stream = b0 + k;
                left -= __shfl_sync(0xffffffffu, incl - n, k);
                break;
            }
            left -= __shfl_sync(0xffffffffu, incl, 31);
        }
    pass = left;
}

__device__ __forceinline__ Place place_at(const PagedArgs &a, int group, int window, int pairs, int splits, int stream,
                                          int pass, int kvh, int part) {
    Place p;
    p.stream = stream, p.pass = pass, p.kvh = kvh;
    p.sw = stream_work(a, stream, group, window, pairs);
    const int capacity = a.table_width << a.page_shift;
    const int row_first = pass * pairs / group, row_last = min((pass * pairs + pairs - 1) / group, p.sw.rows - 1);
    p.any_last = min(p.sw.length - p.sw.rows + row_last, capacity - 1);
    p.any_first = window ? max(0, p.sw.length - p.sw.rows + row_first - window + 1) : 0;
    const int step0 = p.any_first / kTokens, steps = p.any_last < p.any_first ? 0 : p.any_last / kTokens - step0 + 1;
    // a part's steps against the parts' join: the best number grows with the root of the steps (us of 64 pairs on 16,
    // 64, 128 steps: F16 20, 27, 32; with parts of 4 steps 19, 27, 37, of 8 22, 26, 32; F32 20, 27, 30; 20, 24, 28; 27,
    // 28, 30)
    p.parts = max(min(min(splits, int(sqrtf(2.0f * float(steps)))), steps / 2), 1);
    const int from = int(int64_t(steps) * part / p.parts);
    p.step0 = step0 + from;
    p.steps = int(int64_t(steps) * (part + 1) / p.parts) - from;
    return p;
}

// A pair of a place: `pair` counts within the stream.
template <class T>
struct PairOf {
    int row, head, position, first;
    bool live;
    T *out;  // null: past the stream's rows, or without a place in the table
    __device__ __forceinline__ PairOf(const AttentionArgs<T> &g, const Place &p, int pair, int head_size) {
        row = pair / g.group;
        live = row < p.sw.rows;
        position = live ? p.sw.length - p.sw.rows + row : -1;
        first = g.window ? max(0, position - g.window + 1) : 0;
        head = p.kvh * g.group + pair - row * g.group;
        out = nullptr;
        if (live && position >= 0 && (position >> g.a.page_shift) < g.a.table_width)
            out = g.output + (p.sw.begin + row) * g.output_stride + int64_t(head) * head_size;
    }
};

// Rows that one token owns, summed again by the NW warps of a block, eight at a time: of the pairs from `pair0` on that
// have a bit in the `words` words `rows`, every `many`-th from the `which`-th on. The place's tokens are spread over the
// warps, whose sums are added up in their order. `smem`: a ring for every warp, then its rows' maxima.
template <int D, int NW>
constexpr int owned_bytes() {
    return NW * (4 * tile_bytes(D) + kPairs * 4);
}
template <class T, int D, int NW>
__device__ __noinline__ void sum_owned(const AttentionArgs<T> &g, const Place &at, int pair0, const uint32_t *rows, int words,
                                       const uint32_t *bad, int which, int many, uint8_t *smem) {
    constexpr int kRing = 4 * tile_bytes(D), kStepTiles = kTokens / kTileTokens;
    static_assert(kRing >= kPairs * (D + 1) * 4, "the ring takes a warp's sums");
    float *most_of = reinterpret_cast<float *>(smem + NW * kRing);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, lg = lane >> 2, lt = lane & 3;
    uint8_t *ring = smem + warp * kRing;
    const int tiles = at.steps * kStepTiles, share = (tiles + 2 * NW - 1) / (2 * NW) * 2;
    const int begin = at.step0 * kStepTiles + min(warp * share, tiles), end = min(begin + share, (at.step0 + at.steps) * kStepTiles);
    int total = 0;
    for (int i = 0; i < words; ++i) total += __popc(rows[i]);
    for (int done = which; done < total; done += kPairs * many) {
        // lane group lg takes the row with done + lg * many owned ones before it
        int left = done + lg * many, mine = -1;
        for (int i = 0; i < words && mine < 0; ++i) {
            const int n = __popc(rows[i]);
            if (left < n) mine = 32 * i + int(__fns(rows[i], 0, left + 1));
            left -= n;
        }
        const PairOf<T> of(g, at, pair0 + max(mine, 0), D);
        const OwnedPair<T> p{g.query + (at.sw.begin + of.row) * g.query_stride + int64_t(of.head) * D, of.position, of.first,
                             mine >= 0};
        float us;
        const Windows w = find_windows<T, D>(g.a, g.scale, p, at.stream, at.kvh, begin, end, ring, &us);
        if (lt == 0) most_of[warp * kPairs + lg] = w.most;
        __syncthreads();
        float most = -INFINITY;
        for (int i = 0; i < NW; ++i) most = fmaxf(most, most_of[i * kPairs + lg]);
        float *part = reinterpret_cast<float *>(ring);
        sum_windows<T, D>(g.a, g.scale, p, at.stream, at.kvh, begin, end, ring, most, w.below(most, us), kLift, part);
        __syncthreads();
        for (int pr = warp; pr < kPairs; pr += NW) {
            const int r = __shfl_sync(0xffffffffu, mine, 4 * pr);
            T *out = reinterpret_cast<T *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(of.out), 4 * pr));
            if (r < 0) continue;
            float l = 0.0f;
            for (int i = 0; i < NW; ++i) l += reinterpret_cast<const float *>(smem + i * kRing)[kPairs * D + pr];
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            for (int c = lane; c < D; c += 32) {
                float o = 0.0f;
                for (int i = 0; i < NW; ++i) o += reinterpret_cast<const float *>(smem + i * kRing)[pr * D + c];
                stf(out + c, (bad[r] >> (c >> 5)) & 1u ? NAN : o * inv);
            }
        }
        __syncthreads();
    }
}

template <class T, int D, bool kCut>
__global__ void __launch_bounds__(Chunk<T, D>::kThreads, 1) paged_chunk_kernel(const __grid_constant__ AttentionArgs<T> g) {
    using C = Chunk<T, D>;
    constexpr int NG = D / 32, TB = tile_bytes(D), KST = C::kStagesK, VST = C::kStagesV;
    constexpr bool kWide = C::kWide;
    constexpr int G = C::kGroups, kSoftmax = C::kSoftmax, kBlockRows = G * kRows;
    extern __shared__ __align__(1024) uint8_t q_tile[];  // then the K stages, the V stages
    __shared__ __align__(8) uint64_t k_full[2], v_full[2], s_full[G][2], p_full[G][2], pv_done[G][2];
    __shared__ uint32_t tmem_slot, mapped[8], poisoned[8];  // of the last eight steps: K runs ahead of the softmax by fewer
    __shared__ int found[2], slot_of;
    __shared__ uint32_t owned_rows[kWide ? kSoftmax / 32 : 1], bad_of[kWide ? kSoftmax : 1];  // of rows that one token owns
    const PagedArgs &a = g.a;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    pdl_trigger();
    pdl_wait();

    const int splits = kCut ? g.splits : 1;
    const int item = int(blockIdx.x) / splits, part = int(blockIdx.x) - item * splits, kvh = item % a.kv_heads;
    if (warp == 0) {
        int stream, pass;
        find_pass(a, g.group, g.window, kBlockRows, item / a.kv_heads, stream, pass);
        if (lane == 0) found[0] = stream, found[1] = pass;
    }
    if (tid == 32) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&k_full[i], kUnpackK);
            mbar_init(&v_full[i], kUnpackV);
            for (int n = 0; n < G; ++n) {
                mbar_init(&s_full[n][i], 2);  // the products, and the thread that saw K: its look-ups are ordered too
                mbar_init(&p_full[n][i], kRows);
                mbar_init(&pv_done[n][i], 1);
            }
        }
        for (int i = 0; i < 8; ++i) poisoned[i] = 0;
        fence_barrier_init();
    }
    // a slot of the workspace: the block's own while there is one for each, else a free one
    constexpr bool borrow = kWide && !kCut;
    if (tid == 64) {
        slot_of = int(blockIdx.x);
        if (borrow) {
            // registers allow one block an SM, so its SM's is free; were it not, another is
            uint32_t sm;
            asm volatile("mov.u32 %0, %%smid;" : "=r"(sm));
            slot_of = -1;
            for (int k = 0; k < g.slots && slot_of < 0; ++k) {
                const int slot = int((sm + k) % uint32_t(g.slots));
                if (atomicCAS(g.tickets + slot, 0u, 1u) == 0u) slot_of = slot;
            }
            // none: the workspace was not zeroed, or another call uses it at the same time
            if (slot_of < 0) atomicOr(&g_error_word, kErrNoSlot);
        }
    }
    __syncthreads();
    const int stream = found[0], pass = found[1];
    if (borrow && slot_of < 0) return;
    Place at;
    if (stream >= 0) at = place_at(a, g.group, g.window, kBlockRows, splits, stream, pass, kvh, part);
    if (stream < 0 || (kCut && part >= at.parts)) {
        if (borrow && tid == 0) atomicExch(g.tickets + slot_of, 0u);
        return;
    }
    const StreamWork &sw = at.sw;
    const int any_first = at.any_first, any_last = at.any_last, step0 = at.step0, steps = at.steps;
    const int groups = min(G, (sw.rows * g.group - pass * kBlockRows + kRows - 1) / kRows);  // that have rows

    if (warp == C::kMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)),
                     "n"(C::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // blocks and groups take turns, by what their own rows are: together they would queue for the L2 cache
    auto flush_phase = [&](int n) { return kWide ? (pass * 5 + kvh * 3 + n * (C::kFlush / 2)) % C::kFlush : 0; };
    uint8_t *k_tiles = q_tile + C::kQBytes, *v_tiles = k_tiles + KST * C::kTile;

    // softmax threads: pair `tid` of the block, row `tid % 128` of its group
    const int own = G == 2 ? warp >> 2 : 0;
    const PairOf<T> mine(g, at, pass * kBlockRows + tid, D);
    const bool live = tid < kSoftmax && mine.live;
    const int position = tid < kSoftmax ? mine.position : -1, first = mine.first;
    const T *src = g.query + (sw.begin + mine.row) * g.query_stride + int64_t(mine.head) * D;
    float unscale = 1.0f, slack = kSlack;
    if (tid < kSoftmax) {
        // the row's queries as one or two F16 numbers each, scaled by a power of two into F16's range
        float top = 0.0f;
        if (live)
            for (int d = 0; d < D; d += 8) {
                float v[8];
                load8(src + d, v, g.vec);
#pragma unroll
                for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[e]));
            }
        int ex = top > 0.0f && top < INFINITY ? int(__float_as_uint(top) >> 23) - 127 : 0;
        ex = min(max(ex, -100), 126);
        const float down = __uint_as_float(uint32_t(127 - ex) << 23);
        unscale = fminf(fmaxf(g.scale * __uint_as_float(uint32_t(127 + ex) << 23), 1e-30f), 1e30f);
        slack = kSlack / unscale;
        if (kWide) unscale *= 1.0f + 1.5f * (D / 16) * kTruncated;  // the low parts are added to the whole score
        for (int d = 0; d < D; d += 8) {
            float v[8];
            if (live) {
                load8(src + d, v, g.vec);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = 0.0f;
            }
            uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x0 = v[2 * i] * down, x1 = v[2 * i + 1] * down;
                const __half2 h = __floats2half2_rn(x0, x1);
                const float2 back = __half22float2(h);
                hi[i] = h2u(h);
                lo[i] = h2u(__floats2half2_rn(x0 - back.x, x1 - back.y));
            }
            uint8_t *at = q_tile + own * C::kGroupBytes + (d >> 6) * (kRows * 128) + (tid & 127) * 128 +
                          ((((d >> 3) & 7) ^ (tid & 7)) << 4);
            *reinterpret_cast<uint4 *>(at) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
            if constexpr (kWide)
                *reinterpret_cast<uint4 *>(at + C::kPart) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
        }
        fence_async();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_slot;
    bool healthy = true;  // no wait of this thread's rows ran out

    if (warp >= C::kMmaWarp) {
        // ---- the products of a group: one elected thread issues ------------------------------------------
        // The warp stays together otherwise, so that descriptors are formed in uniform registers.
        const bool leader = elect_one();
        const uint64_t q0 = tile_desc(smem_u32(q_tile)), k0 = tile_desc(smem_u32(k_tiles)), v0 = tile_desc(smem_u32(v_tiles));
        const int n = warp - C::kMmaWarp, phase = flush_phase(n);
        const uint64_t q = q0 + uint32_t(n * (C::kGroupBytes / 16));
        bool ok = n < groups;
#pragma unroll 1
        for (int i = -1; ok && i < steps; ++i) {
            if (i + 1 < steps) {
                // the next scores go where the last probabilities were
                ok = wait_phase(&k_full[(i + 1) % KST], ((i + 1) / KST) & 1, kErrFullBarrierTimeout) &&
                     (i < 1 || wait_phase(&pv_done[n][(i - 1) & 1], ((i - 1) >> 1) & 1, kErrMmaBarrierTimeout));
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint64_t k_desc = k0 + uint32_t(((i + 1) % KST) * (C::kTile / 16));
                const uint32_t d = tmem + uint32_t(2 * n + ((i + 1) & 1)) * kTokens;
                if (leader) {
#pragma unroll
                    for (int half = 0; half < (kWide ? 2 : 1); ++half)
#pragma unroll
                        for (int k = 0; k < D / 16; ++k)  // descriptors count 16 bytes
                            mma_ss(d, q + (half * C::kPart + (k >> 2) * (kRows * 128) + (k & 3) * 32) / 16,
                                   k_desc + ((k >> 2) * (kTokens * 128) + (k & 3) * 32) / 16, C::kScores, half | k);
                    mma_commit(&s_full[n][(i + 1) & 1]);
                    mbar_arrive(&s_full[n][(i + 1) & 1]);
                }
                __syncwarp();
            }
            if (i < 0) continue;
            ok = wait_phase(&p_full[n][i & 1], (i >> 1) & 1, kErrFullBarrierTimeout) &&
                 wait_phase(&v_full[i % VST], (i / VST) & 1, kErrFullBarrierTimeout);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
            const uint32_t p = tmem + uint32_t(2 * n + (i & 1)) * kTokens;
            const uint64_t v = v0 + uint32_t((i % VST) * (C::kTile / 16));
            if (leader) {
#pragma unroll
                for (int half = 0; half < (kWide ? 2 : 1); ++half)
#pragma unroll
                    for (int k = 0; k < kTokens / 16; ++k)
                        mma_ts(tmem + C::kOut + n * D, p + (k >> 1) * 32 + half * 16 + (k & 1) * 8, v + k * 2, C::kValues,
                               (kWide && (i + phase) % C::kFlush == 0 ? 0 : i) | half | k);
                mma_commit(&pv_done[n][i & 1]);
            }
            __syncwarp();
        }
    } else if (tid >= kSoftmax) {
        // ---- unpacking ---------------------------------------------------------------------
        const int t = tid < kSoftmax + kUnpackK ? tid - kSoftmax : tid - kSoftmax - kUnpackK;
        const __half2 minus = __float2half2_rn(-24.0f);
        // lane i holds where the i-th tile of 16 tokens from `held` on lies in the pool, counted in tiles
        constexpr uint32_t kNone = 0xFFFFFFFFu;
        uint32_t places = kNone;
        int held = INT32_MIN;
        auto place_of = [&](int sub) {  // asked by all lanes, for tiles of one step
            const int low = sub & ~3;
            if (low < held || low + 3 >= held + 32) {
                held = low;
                const int mine = low + lane, shift = a.page_shift - 4, entry = mine >> shift;
                places = kNone;
                if (16 * mine <= any_last && 16 * mine + 15 >= any_first && entry < a.table_width) {
                    const int page = a.page_table[int64_t(stream) * a.table_width + entry];
                    if (uint32_t(page) < uint32_t(a.page_count))
                        places = ((uint32_t(page) * a.kv_heads + kvh) << shift) + (mine & ((1 << shift) - 1));
                }
            }
            return __shfl_sync(0xffffffffu, places, sub - held);
        };
        // Pages are read by ordinary loads: this grid may have started beside the append that writes them, and only
        // those see after pdl_wait() what it wrote (the non-coherent path wants memory that nobody writes while a
        // grid runs). The loads of step i + 1 travel while step i waits for its place and the products of step i run;
        // one copy of the code, because the block's four roles share the instruction cache
        auto walk = [&](auto &x, auto &&load, auto &&put) {
            if (steps > 0) load(0, x);
#pragma unroll 1
            for (int i = 0; i < steps; ++i) {
                if (!put(i, x)) break;
                if (i + 1 < steps) load(i + 1, x);
            }
        };
        // a stage of K or V is free when all groups' products of step i have read it
        auto read_by_all = [&](uint64_t (&bars)[G][2], int i) {
            for (int n = 0; n < groups; ++n)
                if (!wait_phase(&bars[n][i & 1], (i >> 1) & 1, kErrEmptyBarrierTimeout)) return false;
            return true;
        };
        if (tid < kSoftmax + kUnpackK) {  // K rows by token, one to a thread
            const int token = t, slot = token & 15;
            uint32_t put_at[4];
#pragma unroll
            for (int n = 0; n < 4; ++n) put_at[n] = token * 128 + ((n ^ (token & 7)) << 4);
            RawK<D> x;
            walk(
                x,
                [&](int i, RawK<D> &x) {
                    const uint32_t place = place_of((step0 + i) * (kTokens / 16) + (token >> 4));
                    const uint8_t *tile = a.pages + uint64_t(place) * TB;
                    if (place != kNone) {
                        const uint4 *w = reinterpret_cast<const uint4 *>(tile + slot * (D / 2));
#pragma unroll
                        for (int n = 0; n < NG; ++n) {
                            const uint4 y = w[n];
                            x.w[4 * n] = y.x, x.w[4 * n + 1] = y.y, x.w[4 * n + 2] = y.z, x.w[4 * n + 3] = y.w;
                        }
#pragma unroll
                        for (int n = 0; n < NG / 2; ++n)
                            x.s[n] = reinterpret_cast<const uint32_t *>(tile + 16 * D + slot * (2 * NG))[n];
                    } else {
#pragma unroll
                        for (int n = 0; n < NG; ++n) x.w[4 * n] = x.w[4 * n + 1] = x.w[4 * n + 2] = x.w[4 * n + 3] = 0;
#pragma unroll
                        for (int n = 0; n < NG / 2; ++n) x.s[n] = 0;
                    }
                    if (slot == 0)
                        reinterpret_cast<uint8_t *>(&mapped[i & 7])[token >> 4] = place != kNone;
                },
                [&](int i, RawK<D> &x) {
                    // this stage was read by the scores of step i - KST
                    if (i >= KST && !read_by_all(s_full, i - KST)) return false;
                    const uint32_t stage = smem_u32(k_tiles) + (i % KST) * C::kTile;
#pragma unroll
                    for (int j = 0; j < NG; ++j) {
                        const __half2 both = u2h(x.s[j / 2]), offs = __hmul2(both, minus);
                        const __half2 s = j & 1 ? __high2half2(both) : __low2half2(both);
                        const __half2 o = j & 1 ? __high2half2(offs) : __low2half2(offs);
#pragma unroll
                        for (int n = 0; n < 4; ++n) {  // word (n, j): chunk 4 j + n of the row
                            const uint32_t w = x.w[n * NG + j];
                            put16(((stage + put_at[n]) ^ ((j & 1) << 6)) + (j >> 1) * (kTokens * 128), unpack<0>(w, s, o),
                                  unpack<1>(w, s, o), unpack<2>(w, s, o), unpack<3>(w, s, o));
                        }
                    }
                    fence_async();
                    mbar_arrive(&k_full[i % KST]);
                    return true;
                });
        } else {  // V rows by channel: thread (eight tokens, word), eight tokens' places side by side
            RawV<D> x;
            walk(
                x,
                [&](int i, RawV<D> &x) {
#pragma unroll
                    for (int n = 0; n < RawV<D>::N; ++n) {
                        const int item = t + kUnpackV * n, tg = item & 7, w = item >> 3;
                        const uint32_t place = place_of((step0 + i) * (kTokens / 16) + (tg >> 1));
                        x.s[n] = make_uint4(0, 0, 0, 0);
                        if (item >= 32 * NG) continue;
                        if (place == kNone) {
#pragma unroll
                            for (int e = 0; e < 8; ++e) x.w[n][e] = 0;
                            continue;
                        }
                        const uint8_t *tile = a.pages + uint64_t(place) * TB;
                        const uint32_t *p =
                            reinterpret_cast<const uint32_t *>(tile + 8 * D + 8 * (tg & 1) * (D / 2)) + w;
#pragma unroll
                        for (int e = 0; e < 8; ++e) x.w[n][e] = p[e * (D / 8)];
                        x.s[n] = *reinterpret_cast<const uint4 *>(tile + 17 * D + (w >> 2) * 32 + 16 * (tg & 1));
                    }
                },
                [&](int i, RawV<D> &x) {
                    const int t0 = (step0 + i) * kTokens;
                    const uint32_t stage = smem_u32(v_tiles) + (i % VST) * C::kTile;
                    // values that no row sees weigh nothing, whatever is there; NaN scales are taken out and reported
#pragma unroll
                    for (int n = 0; n < RawV<D>::N; ++n) {
                        uint32_t *s = &x.s[n].x;
                        const int tok = t0 + 8 * ((t + kUnpackV * n) & 7);
                        if (tok < any_first || tok + 7 > any_last) {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (tok + e < any_first || tok + e > any_last) s[e >> 1] &= e & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                        }
                        if ((not_finite(s[0]) | not_finite(s[1]) | not_finite(s[2]) | not_finite(s[3])) & 0x80008000u) {
                            poisoned[i & 7] = uint32_t(i) + 1u;
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                if ((s[e] & 0x7C00u) == 0x7C00u) s[e] &= 0xFFFF0000u;
                                if ((s[e] & 0x7C000000u) == 0x7C000000u) s[e] &= 0x0000FFFFu;
                            }
                        }
                    }
                    if (i >= VST && !read_by_all(pv_done, i - VST)) return false;
#pragma unroll
                    for (int n = 0; n < RawV<D>::N; ++n) {
                        const int item = t + kUnpackV * n, tg = item & 7, w = item >> 3;
                        if (item >= 32 * NG) continue;
                        const uint32_t *sv = &x.s[n].x;
                        uint32_t lo[4], hi[4];
                        __half2 s[4], o[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) {
                            lo[p] = __byte_perm(x.w[n][2 * p], x.w[n][2 * p + 1], 0x5410);
                            hi[p] = __byte_perm(x.w[n][2 * p], x.w[n][2 * p + 1], 0x7632);
                            s[p] = u2h(sv[p]);
                            o[p] = __hmul2(s[p], minus);
                        }
                        const uint32_t at = stage + (8 * w) * 128 + (tg << 4);
                        auto row = [&](int e, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3) {
                            put16((at ^ (e << 4)) + e * 128, a0, a1, a2, a3);
                        };
#define SI_ROW(E, I, X)                                                                                    \
    row(E, unpack<I>(X[0], s[0], o[0]), unpack<I>(X[1], s[1], o[1]), unpack<I>(X[2], s[2], o[2]), \
        unpack<I>(X[3], s[3], o[3]))
                        SI_ROW(0, 0, lo);
                        SI_ROW(1, 0, hi);
                        SI_ROW(2, 1, lo);
                        SI_ROW(3, 1, hi);
                        SI_ROW(4, 2, lo);
                        SI_ROW(5, 2, hi);
                        SI_ROW(6, 3, lo);
                        SI_ROW(7, 3, hi);
#undef SI_ROW
                    }
                    fence_async();
                    mbar_arrive(&v_full[i % VST]);
                    return true;
                });
        }
    } else {
        // ---- softmax: a row to a thread ----------------------------------------------------
        const uint32_t lanes = tmem + (uint32_t((warp & 3) * 32) << 16);
        const uint32_t out_at = lanes + C::kOut + own * D;
        const int my_steps = own < groups ? steps : 0;
        uint32_t bad = 0;  // groups in which the row sees a value that is not finite
        // the row's O into its slot: added there when that holds something, which `by` scales first. A slot has
        // one writer, so the additions have one order; they return nothing that a thread would wait for
        auto slot4 = [&](int c) {
            float *slot = g.parts + int64_t(slot_of) * C::kSlot + own * (kRows * D) + (tid & 127) * 4;
            return reinterpret_cast<float4 *>(slot + (c >> 2) * (4 * kRows));
        };
        auto flush = [&](bool more, float by, float whole) {
            const bool scale = more && __any_sync(0xffffffffu, by != 1.0f);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                tm_load32(out_at + c, o);
#pragma unroll
                for (int j = 0; j < 32; j += 4) {
                    float4 x = make_float4(__uint_as_float(o[j]) * whole, __uint_as_float(o[j + 1]) * whole,
                                           __uint_as_float(o[j + 2]) * whole, __uint_as_float(o[j + 3]) * whole);
                    if (more && !scale) {
                        add_global(slot4(c + j), x);
                    } else {
                        if (scale) x = fma_all(__ldcg(slot4(c + j)), by, x);
                        __stcg(slot4(c + j), x);
                    }
                }
            }
        };
        const int phase = flush_phase(own);
        bool begun = false;    // the slot holds something
        int summed = 0;        // products of 16 tokens that put something into the present sums of the row
        // what the mean of their truncations makes good: one product adds either half; where the row sees none of the
        // 16 tokens it adds zeros, which lose nothing
        auto untruncated = [&] { return kWide ? 1.0f + kTruncated * float(summed) : 1.0f; };
        float flushed = 1.0f;  // how far the maximum has moved since the slot was written
        float m = -INFINITY, l = 0.0f, most = -INFINITY;
        bool ok = true;
        for (int i = 0; i < my_steps; ++i) {
            const int t0 = (step0 + i) * kTokens;
            const uint32_t scores = lanes + uint32_t(2 * own + (i & 1)) * kTokens;
            ok = wait_phase(&s_full[own][i & 1], (i >> 1) & 1, kErrMmaBarrierTimeout);
            if (__any_sync(0xffffffffu, !ok)) {
                ok = false;
                break;
            }
            tc_fence_after();
            const bool fresh = i == 0 || (kWide && (i + phase) % C::kFlush == 0);  // the step's product replaces O
            if (kWide && fresh && i > 0) {
                ok = wait_phase(&pv_done[own][(i - 1) & 1], ((i - 1) >> 1) & 1, kErrMmaBarrierTimeout);
                if (__any_sync(0xffffffffu, !ok)) {
                    ok = false;
                    break;
                }
                tc_fence_after();
                flush(begun, flushed, untruncated());
                begun = true;
                summed = 0;
                flushed = 1.0f;
            }
            const uint32_t have = mapped[i & 7];
            const bool cut = __any_sync(0xffffffffu, have != 0x01010101u || t0 < first || t0 + kTokens - 1 > position);
            uint32_t v[kTokens];
            tm_load64(scores, v);
            if (cut) {  // tokens that the row does not see at -inf
#pragma unroll
                for (int c = 0; c < kTokens; c += 32) {
                    const int lo = first - t0 - c, hi = position - t0 - c;
                    uint32_t sees = hi < 0 || lo > 31 ? 0u : 0xffffffffu;
                    if (hi >= 0 && hi < 31) sees &= (2u << hi) - 1u;
                    if (lo > 0 && lo < 32) sees &= 0xffffffffu << lo;
                    if (!((have >> (c / 2)) & 1u)) sees &= 0xffff0000u;
                    if (!((have >> (c / 2 + 8)) & 1u)) sees &= 0x0000ffffu;
                    if constexpr (kWide) summed += int((sees & 0xffffu) != 0) + int((sees >> 16) != 0);
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[c + j] = (sees >> j) & 1u ? v[c + j] : 0xff800000u;
                }
            } else if constexpr (kWide) {
                summed += kTokens / 16;
            }
            float top = -INFINITY, other = -INFINITY;
#pragma unroll
            for (int j = 0; j < kTokens; j += 4) {
                top = max3(top, __uint_as_float(v[j]), __uint_as_float(v[j + 1]));
                other = max3(other, __uint_as_float(v[j + 2]), __uint_as_float(v[j + 3]));
            }
            top = fmaxf(top, other);
            if constexpr (kWide) most = fmaxf(most, top);
            const bool moves = top > m + slack;
            if (__any_sync(0xffffffffu, moves)) {
                const float alpha = moves ? ex2((m - top) * unscale) : 1.0f;
                if (moves) m = top;
                l *= alpha;
                flushed *= alpha;
                if (!fresh) {
                    ok = wait_phase(&pv_done[own][(i - 1) & 1], ((i - 1) >> 1) & 1, kErrMmaBarrierTimeout);
                    if (__any_sync(0xffffffffu, !ok)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t o[16];
                        tm_load16(out_at + c, o);
#pragma unroll
                        for (int j = 0; j < 16; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * alpha);
                        tm_store16(out_at + c, o);
                    }
                    tc_wait_st();
                }
            }
            const float lift = kLift - (m == -INFINITY ? 0.0f : m) * unscale;
            const float2 lift2 = make_float2(lift, lift), unscale2 = make_float2(unscale, unscale);
            // 32 scores become 16 columns of probabilities and 16 of what rounding left, in the same place
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < kTokens; c += 32) {
                uint32_t h[16], r[16];
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    float2 e = fma2(make_float2(__uint_as_float(v[c + 2 * j]), __uint_as_float(v[c + 2 * j + 1])), unscale2,
                                    lift2);
                    e = make_float2(ex2(e.x), ex2(e.y));
                    sum = add2(sum, e);
                    const __half2 p = __floats2half2_rn(e.x, e.y);
                    h[j] = h2u(p);
                    if constexpr (kWide) {
                        const float2 f = __half22float2(p);
                        r[j] = h2u(__floats2half2_rn(e.x - f.x, e.y - f.y));
                    }
                }
                tm_store16(scores + c, h);
                if constexpr (kWide) tm_store16(scores + c + 16, r);
            }
            l += sum.x + sum.y;
            // reported while V was unpacked, which the product waits for anyway
            ok = wait_phase(&v_full[i % VST], (i / VST) & 1, kErrFullBarrierTimeout);
            if (__any_sync(0xffffffffu, !ok)) {
                ok = false;
                break;
            }
            if (poisoned[i & 7] == uint32_t(i) + 1u) {
                for (int j = 0; j < kTokens; ++j) {
                    if (t0 + j < first || t0 + j > position || !((have >> (8 * (j >> 4))) & 1u)) continue;
                    const uint8_t *tile = tile_of(a, stream, t0 + j, kvh);
                    if (!tile) continue;
                    for (int n = 0; n < NG; ++n) {
                        const uint32_t x = reinterpret_cast<const uint16_t *>(tile + 17 * D)[n * 16 + (j & 15)];
                        if ((x & 0x7C00u) == 0x7C00u) bad |= 1u << n;
                    }
                }
            }
            tc_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[own][i & 1]);
        }
        if (my_steps > 0 && ok) ok = wait_phase(&pv_done[own][(steps - 1) & 1], ((steps - 1) >> 1) & 1, kErrMmaBarrierTimeout);
        ok = !__any_sync(0xffffffffu, !ok);
        tc_fence_after();
        T *const out = PairOf<T>(g, at, pass * kBlockRows + tid, D).out;
        if constexpr (kWide) {  // rows that one token owns: a token that is alone needs no second look
            const float largest = ex2(fmaf(most, unscale, kLift - (m == -INFINITY ? 0.0f : m) * unscale));
            const bool owned = (!kCut || at.parts == 1) && ok && out && most > -INFINITY && l - largest < kOwned * largest &&
                               min(position, any_last) > first;
            const uint32_t rows = __ballot_sync(0xffffffffu, owned);
            if (lane == 0) owned_rows[warp] = rows;
            bad_of[tid] = bad;
            healthy = ok;
        }
        if (kCut && ok && at.parts > 1) {  // one part of the row's sums, for the join
            if (my_steps > 0) {
                flush(begun, flushed, untruncated());
                float *stats = g.parts + int64_t(slot_of) * C::kSlot + kBlockRows * D + tid;
                __stcg(stats, m * unscale);
                __stcg(stats + kBlockRows, l);
                __stcg(stats + 2 * kBlockRows, most * unscale);
                __stcg(stats + 3 * kBlockRows, __uint_as_float(bad));
            }
        } else if (ok) {
            const float inv = l != 0.0f ? 1.0f / l : 0.0f;
            const float whole = untruncated();
            float4 held[8];  // what the slot holds of the next 32 channels
            auto fetch = [&](int c) {
#pragma unroll
                for (int j = 0; j < 8; ++j) held[j] = __ldcg(slot4(c + 4 * j));
            };
            if (kWide && begun) fetch(0);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                float v[32];
                if (my_steps > 0) tm_load32(out_at + c, o);
                const float times = (bad >> (c >> 5)) & 1u ? NAN : inv;
#pragma unroll
                for (int j = 0; j < 32; ++j) v[j] = my_steps > 0 ? __uint_as_float(o[j]) * whole : 0.0f;
                if (kWide && begun) {
#pragma unroll
                    for (int j = 0; j < 32; j += 4) {
                        const float4 x = fma_all(held[j / 4], flushed, make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]));
                        v[j] = x.x, v[j + 1] = x.y, v[j + 2] = x.z, v[j + 3] = x.w;
                    }
                    if (c + 32 < D) fetch(c + 32);
                }
                if (out) {
#pragma unroll
                    for (int j = 0; j < 32; j += 8) {
                        const float u[8] = {v[j] * times,     v[j + 1] * times, v[j + 2] * times, v[j + 3] * times,
                                            v[j + 4] * times, v[j + 5] * times, v[j + 6] * times, v[j + 7] * times};
                        store8(out + c + j, u, g.vec_out);
                    }
                }
                __syncwarp();
            }
        }
    }
    if constexpr (kWide) {
        static_assert(owned_bytes<D, C::kThreads / 32>() <= C::kSmem, "operands make room for the second look");
        // all products are done where every row's last one is
        if (!__syncthreads_or(!healthy)) {
            uint32_t any = 0;
            for (int i = 0; i < kSoftmax / 32; ++i) any |= owned_rows[i];
            if (any) {
                const Place copy = at;  // `at` itself stays in registers
                sum_owned<T, D, C::kThreads / 32>(g, copy, pass * kBlockRows, owned_rows, kSoftmax / 32, bad_of, 0, 1, q_tile);
            }
        }
    }
    if (borrow) __threadfence();
    tc_fence_before();
    __syncthreads();
    if (borrow && tid == 0) atomicExch(g.tickets + slot_of, 0u);
    if (warp == C::kMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(C::kColumns) : "memory");
    }
}

// Adds the parts of a block's tokens up: 128 rows and 16 channels a block, a row
// a thread. Bound: the parts' latency, four of them on their way at a time.
template <class T, int D>
__global__ void __launch_bounds__(kRows) paged_chunk_join_kernel(const __grid_constant__ AttentionArgs<T> g) {
    using C = Chunk<T, D>;
    constexpr int G = C::kGroups, kBlockRows = G * kRows, kChannels = 16;
    __shared__ int found[2];
    pdl_trigger();
    pdl_wait();
    const int tid = threadIdx.x, item = int(blockIdx.x) / G, own = int(blockIdx.x) - item * G, c = int(blockIdx.y) * kChannels;
    if (tid < 32) {
        int stream, pass;
        find_pass(g.a, g.group, g.window, kBlockRows, item / g.a.kv_heads, stream, pass);
        if (tid == 0) found[0] = stream, found[1] = pass;
    }
    __syncthreads();
    if (found[0] < 0) return;
    const Place at = place_at(g.a, g.group, g.window, kBlockRows, g.splits, found[0], found[1], item % g.a.kv_heads, 0);
    if (at.parts == 1) return;
    const int pair = at.pass * kBlockRows + own * kRows + tid;
    const PairOf<T> of(g, at, pair, D);
    const float *slot = g.parts + int64_t(item) * g.splits * C::kSlot;
    const float *stats = slot + kBlockRows * D + own * kRows + tid, *o = slot + own * (kRows * D) + tid * 4 + c * kRows;
    bool owned = false;
    uint32_t bad = 0;
    if (of.out) {
        float top = -INFINITY, most = -INFINITY;
#pragma unroll 4
        for (int k = 0; k < at.parts; ++k) {
            top = fmaxf(top, __ldcg(stats + int64_t(k) * C::kSlot));
            most = fmaxf(most, __ldcg(stats + int64_t(k) * C::kSlot + 2 * kBlockRows));
        }
        float l = 0.0f;
        float4 acc[kChannels / 4];
#pragma unroll
        for (int j = 0; j < kChannels / 4; ++j) acc[j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
        for (int k = 0; k < at.parts; ++k) {
            const float *p = stats + int64_t(k) * C::kSlot;
            const float m = __ldcg(p);
            const float by = m == -INFINITY ? 1.0f : ex2(m - top);  // without a score a part keeps its sums: zeros, or NaN
            l = fmaf(by, __ldcg(p + kBlockRows), l);
            bad |= __float_as_uint(__ldcg(p + 3 * kBlockRows));
#pragma unroll
            for (int j = 0; j < kChannels / 4; ++j)
                acc[j] = fma_all(__ldcg(reinterpret_cast<const float4 *>(o + int64_t(k) * C::kSlot + j * (4 * kRows))), by, acc[j]);
        }
        if constexpr (C::kWide) {
            const float largest = ex2(most - (top == -INFINITY ? 0.0f : top) + kLift);
            owned = most > -INFINITY && l - largest < kOwned * largest && min(of.position, at.any_last) > of.first;
        }
        if (!owned) {
            const float times = (bad >> (c >> 5)) & 1u ? NAN : l != 0.0f ? 1.0f / l : 0.0f;
#pragma unroll
            for (int j = 0; j < kChannels / 4; j += 2) {
                const float v[8] = {acc[j].x * times,     acc[j].y * times,     acc[j].z * times,     acc[j].w * times,
                                    acc[j + 1].x * times, acc[j + 1].y * times, acc[j + 1].z * times, acc[j + 1].w * times};
                store8(of.out + c + 4 * j, v, g.vec_out);
            }
        }
    }
    if constexpr (C::kWide) {  // owned rows go round the blocks of all channels
        extern __shared__ __align__(128) uint8_t rings[];
        __shared__ uint32_t owned_rows[kRows / 32], bad_of[kRows];
        const uint32_t rows = __ballot_sync(0xffffffffu, owned);
        if ((tid & 31) == 0) owned_rows[tid >> 5] = rows;
        bad_of[tid] = bad;
        if (__syncthreads_or(owned)) {
            const Place whole =
                place_at(g.a, g.group, g.window, kBlockRows, 1, found[0], found[1], item % g.a.kv_heads, 0);
            sum_owned<T, D, kRows / 32>(g, whole, at.pass * kBlockRows + own * kRows, owned_rows, kRows / 32, bad_of,
                                        int(blockIdx.y), int(gridDim.y), rings);
        }
    }
}

template <class T, int D>
si_status launch(const AttentionArgs<T> &all, void *stream) {
    constexpr int kBlockRows = Chunk<T, D>::kGroups * kRows;
    // the most blocks that the streams' pairs can be: each stream rounds up once
    const int64_t items = all.a.kv_heads * ((all.a.rows * all.group + int64_t(kBlockRows - 1) * all.a.streams) / kBlockRows);
    if (items > INT32_MAX) return fail(SI_ERR_UNSUPPORTED, "paged-attention: too many rows.");
    if (items == 0) return SI_OK;
    AttentionArgs<T> g = all;
    g.splits = int(std::max<int64_t>(1, std::min<int64_t>(g.slots / items, kMostParts)));
    const dim3 grid(unsigned(items * g.splits)), block(Chunk<T, D>::kThreads);
    if (g.splits == 1)
        return launch_pdl("paged-attention", paged_chunk_kernel<T, D, false>, grid, block, Chunk<T, D>::kSmem, 1, stream, g);
    if (const si_status e =
            launch_pdl("paged-attention", paged_chunk_kernel<T, D, true>, grid, block, Chunk<T, D>::kSmem, 1, stream, g))
        return e;
    return launch_pdl("paged-attention", paged_chunk_join_kernel<T, D>,
                      dim3(unsigned(items) * Chunk<T, D>::kGroups, D / 16), dim3(kRows),
                      Chunk<T, D>::kWide ? owned_bytes<D, kRows / 32>() : 0, 1, stream, g);
}

template <class T>
si_status run(const AttentionArgs<T> &g, void *stream) {
    switch (g.a.head_size) {
    case 64: return launch<T, 64>(g, stream);
    case 128: return launch<T, 128>(g, stream);
    case 192: return launch<T, 192>(g, stream);
    default: return launch<T, 256>(g, stream);
    }
}

}  // namespace

si_status paged_chunk_attention(const AttentionArgs<float> &g, void *stream) { return run(g, stream); }
si_status paged_chunk_attention(const AttentionArgs<__half> &g, void *stream) { return run(g, stream); }

uint64_t paged_chunk_workspace(int head_size) {
    return uint64_t(device_sm_count()) * (head_size <= 128 ? 2 : 1) * kRows * (uint64_t(head_size) + 4) * 4;
}

si_status take_error_paged(int device, uint32_t *code) {
    int prev = 0;
    cudaGetDevice(&prev);
    if (cudaSetDevice(device) != cudaSuccess) return fail(SI_ERR_CUDA, "cudaSetDevice(%d) failed", device);
    uint32_t v = 0, zero = 0;
    cudaError_t e = cudaMemcpyFromSymbol(&v, g_error_word, sizeof v);
    if (e == cudaSuccess) e = cudaMemcpyToSymbol(g_error_word, &zero, sizeof zero);
    cudaSetDevice(prev);
    if (e != cudaSuccess) return fail(SI_ERR_CUDA, "device error word: %s", cudaGetErrorString(e));
    *code |= v;
    return SI_OK;
}

}  // namespace si::kernels
