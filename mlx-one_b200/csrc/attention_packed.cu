// Attention of single tokens over a cache held in 4 bits (packed_cache.cuh has the format).
//
//   s_j = scale q . k_j = scale sum_g (step_jg (q_g . code_jg) + lowest_jg sum(q_g))
//   o   = sum_j p_j v_j,  v_jg = step_jg code_jg + lowest_jg,  p = softmax of s over the keys seen (and a sink)
//
// Codes are whole numbers of 0..15, so they go into the matrix instructions as they are: the steps and lowest
// values stay outside, in 32 bits. Scores are computed transposed (keys are the 16 rows of a product, up to
// eight query heads that share the key head its 8 columns), so that GQA's few heads waste no rows, and a unit's
// codes are operand registers after two shifts' worth of masking: four bits at the bottom of a half-precision
// number are the subnormal number code * 2^-24, four bits above them 16 times that. So one shift and four ANDs
// make the eight operands of a word; the factor 16 is in the queries of those dimensions, or taken off those
// dimensions of the output at the end.
//
// Roundings (bfloat16 queries): a query becomes half-precision times a power of two that brings the
// block's largest to 2^13, exact but for what is 2^-26 of the largest and less. A weight p step becomes
// half-precision times a power of two that keeps the largest step near 2^9 (11 bits of every weight down to
// 2^-24 of the largest; as bfloat16 with its 8 bits the result was off by 0.003 to 0.008 of itself, now by
// 0.0003 and its own rounding). Sums, scores, exponentials and the lowest values' share are in 32 bits.
//
// float32 queries: every value cut into three bfloat16 parts, which hold its 24 bits, and so are the weights
// of the values; the codes are centred (code - 8, exact in bfloat16) and the outputs added up in 32-bit
// registers, tile by tile, so that no sum is longer or larger than it must be.
//
// What bounds it: latency. Of the time of 32 requests of 4,096 keys, the bytes of the codes (72 a key and key head of
// 64, keys and values) keep DRAM busy for 38 %, 290 instructions of a warp for 32 keys the issue slots for 47 % (61 %
// of the cycles in which an SM works), the ALU pipe 47 %, the tensor pipe 21 %: with the 16 warps an SM that 128
// registers and the rings allow, 0.97 of 3.25 warps a scheduler are ready on average. One block = one
// (request, key head, up to 8 of its query heads, split of the keys); its 8 warps take tiles of 64 keys (Ring) in
// turn, each through a ring of its own that bulk copies fill (one copy brings the keys and values of 16 tokens):
// no barrier of the block before the end. The warps are merged in shared memory, the splits of up to 8 blocks
// through a cluster's shared memory, more by a second kernel.
//
// Measured, 32 heads over 8 key heads of 64, us on the GPU: 32 requests of 4,096 keys 24.1 (75.5 MB, 3.1 TB/s; 11.3
// at the copy rate; issue slots taken in 61 % of the cycles that an SM works, 256 blocks on 296 places), one of
// 509 keys 4.0 (launch and three loads one after the other), four of 30,011 keys with heads of 128 38.2 (3.8
// TB/s). 10 to 16 warps a block (26.8 to 30.3 against 24.2 us; an SM then has room for one block) or tiles of 32 keys with
// heads of 64 (26.9) are slower, and so is more than one block a request and key head where the blocks find no
// place at once (packed_splits in kernels/cuda_ops.py has the rule).
//
// The running maximum moves only when a score passes it by more than 2^4 (in powers of two), the steps'
// power of two only when one outgrows it: most tiles need no exchange between lanes and no pass over the
// output.
#include <cooperative_groups.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "by_words.cuh"
#include "packed_cache.cuh"

namespace cg = cooperative_groups;

namespace {

using bf16 = __nv_bfloat16;
constexpr int WARPS = 8;
constexpr int HEADS = 8;               // query heads of a block
constexpr int CLUSTER = 8;             // splits that a cluster merges
constexpr int WAIT_LIMIT = 1 << 22;
constexpr int ERROR_WAIT = 9;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NOTHING = -1e30f;      // a maximum of no scores: finite, so that differences stay numbers
constexpr float LAZY = 4.f;

// Keys of a tile, and tiles of a warp's ring. 64 keys with heads of up to 64 values (what a tile costs beside its
// keys, the look-up of pages, the copies, the wait and the vote, is paid half as often), 32 where registers
// are short.
template <typename T, int HD>
struct Ring {
    static constexpr int KEYS = HD <= 64 && sizeof(T) == 2 ? 64 : 32;
    static constexpr int UNITS = KEYS / 16;
    static constexpr int STAGES = HD == 32 ? 4 : 3;
    static constexpr int STAGE = UNITS * Packed<HD>::UNIT;
    static constexpr int BYTES = WARPS * STAGES * STAGE;
    // what the merge needs: a maximum, a sum and an output per head, for every warp and then for the block
    static constexpr int MERGE = (WARPS + 1) * HEADS * (HD + 2) * 4;
    static constexpr int SHARED = (BYTES > MERGE ? BYTES : MERGE) + 128;
};

__device__ __forceinline__ uint32_t shared_address(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void barrier_init(uint32_t bar) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bar));
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool barrier_test(uint32_t bar, uint32_t parity) {
    uint32_t done;
    asm volatile(
        "{\n.reg .pred p;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "selp.b32 %0, 1, 0, p;\n}\n"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
    return done != 0;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
        ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
        : "memory");
}
// d += a (16x16, row) * b (16x8, col), bfloat16 in, float accumulate
__device__ __forceinline__ void mma_16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                          uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with half-precision operands
__device__ __forceinline__ void mma_half(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// ... and nothing to add to
__device__ __forceinline__ void mma_half_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                               uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
        "{%8,%9}, {%10,%10,%10,%10};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float max_of_three(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float low_of(uint32_t pair) { return __uint_as_float(pair << 16); }
__device__ __forceinline__ float high_of(uint32_t pair) { return __uint_as_float(pair & 0xffff0000u); }

// The operand pairs of a word's eight codes, in the order of their bits: code - 8 as bfloat16 ...
__device__ __forceinline__ void expand_centred(uint32_t word, uint32_t (&pair)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        pair[i] = ((word >> (4 * i)) & 0x000f000fu) | 0x43004300u;       // 128 + code
        const uint32_t middle = 0x43084308u;                             // 136
        const __nv_bfloat162 v = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&pair[i]),
                                         *reinterpret_cast<const __nv_bfloat162*>(&middle));
        pair[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
}
// ... or in half-precision code * 2^-24, the second and the fourth pair 16 times that.
__device__ __forceinline__ void expand_small(uint32_t word, uint32_t (&pair)[4]) {
    pair[0] = word & 0x000f000fu;
    pair[1] = word & 0x00f000f0u;
    word >>= 8;
    pair[2] = word & 0x000f000fu;
    pair[3] = word & 0x00f000f0u;
}
constexpr float CODE_UNIT = 16777216.f;                // 2^24

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

// Cuts a pair of 32-bit values into NP pairs of bfloat16 parts, the largest first: their sum is the value.
template <int NP>
__device__ __forceinline__ void parts_of(float a, float b, uint32_t (&part)[NP]) {
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        part[i] = pack_pair(a, b);
        a -= low_of(part[i]);
        b -= high_of(part[i]);
    }
}

__device__ __forceinline__ void load_words(const unsigned char* at, uint32_t (&words)[4]) {
    const uint4 w = *reinterpret_cast<const uint4*>(at);
    words[0] = w.x; words[1] = w.y; words[2] = w.z; words[3] = w.w;
}
__device__ __forceinline__ void load_words(const unsigned char* at, uint32_t (&words)[2]) {
    const uint2 w = *reinterpret_cast<const uint2*>(at);
    words[0] = w.x; words[1] = w.y;
}

template <typename T>
__device__ __forceinline__ void store_pair(T* dst, float a, float b);
template <>
__device__ __forceinline__ void store_pair<float>(float* dst, float a, float b) {
    *reinterpret_cast<float2*>(dst) = make_float2(a, b);
}
template <>
__device__ __forceinline__ void store_pair<bf16>(bf16* dst, float a, float b) {
    *reinterpret_cast<uint32_t*>(dst) = pack_pair(a, b);
}

template <typename T, int HD>
__global__ void __launch_bounds__(WARPS * 32, HD <= 64 || sizeof(T) == 2 ? 2 : 1)
attention_packed_kernel(const T* q, const unsigned char* cache,
                        const int* block_table, int table_width, int page_shift, int pages,
                        const int* positions, T* out, float* partial,
                        int heads, int kv_heads, int splits, float scale_log2, int window,
                        const float* sinks, int* error_flag) {
    using P = Packed<HD>;
    using R = Ring<T, HD>;
    constexpr int KEYS = R::KEYS, UNITS = R::UNITS;
    constexpr bool WIDE = sizeof(T) == 4;                  // 32-bit queries
    constexpr int NP = WIDE ? 3 : 1;                       // bfloat16 parts of a value
    constexpr int RUNS = P::RUNS, GROUPS = P::GROUPS, GROUP_RUNS = P::GROUP / 16;
    constexpr float MIDDLE = 8.f;                          // of the centred codes
    extern __shared__ unsigned char shared_raw[];
    __shared__ __align__(8) unsigned long long barriers[WARPS * R::STAGES];
    unsigned char* shared = reinterpret_cast<unsigned char*>((reinterpret_cast<size_t>(shared_raw) + 127) &
                                                             ~(size_t)127);
    const int group = heads / kv_heads;
    const int blocks_of_heads = (group + HEADS - 1) / HEADS;
    const int kv_head = blockIdx.y / blocks_of_heads;
    const int head0 = kv_head * group + (blockIdx.y % blocks_of_heads) * HEADS;
    const int rows = min(HEADS, kv_head * group + group - head0);
    const int request = blockIdx.z, split = blockIdx.x;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, c = lane & 3;

    griddep_launch();
    // (a warp's barriers are its own: nobody else waits for them or for their making)
    if (lane == 0) {
#pragma unroll
        for (int k = 0; k < R::STAGES; ++k) barrier_init(shared_address(&barriers[warp * R::STAGES + k]));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    // Queries, and pages: the kernel before this one may have written this step's tokens there.
    griddep_wait();
    const T* queries = settled(q);
    const unsigned char* codes = settled(cache);

    const int position = positions[request];
    const int lowest_key = first_visible_key(position, window);
    const int tile_first = lowest_key / KEYS;
    const int tiles = position < 0 ? 0 : position / KEYS - tile_first + 1;
    const int share = (tiles + splits - 1) / splits;
    const int from = tile_first + min(split * share, tiles), to = tile_first + min(split * share + share, tiles);

    const int* table = block_table + (size_t)request * table_width;
    const int units_per_page = 1 << (page_shift - 4);
    unsigned char* ring = shared + warp * R::STAGES * R::STAGE;
    auto barrier = [&](int stage) { return shared_address(&barriers[warp * R::STAGES + stage]); };
    // Where the units of a warp's tiles lie, a lane each for AHEAD tiles at a time (lane = tile of these * UNITS +
    // unit; -1: no key of it is seen); the next ones are looked up half a turn before the first is wanted. A unit
    // that has keys to be seen but no page makes every tile go by the mask, which then looks at the pages.
    constexpr int AHEAD = 32 / UNITS;
    bool holes = false;
    auto look_up = [&](int first_tile) -> int {
        const int tile = first_tile + lane / UNITS * WARPS;
        const int key = tile * KEYS + 16 * (lane % UNITS);
        if (tile >= to || key > position || key + 15 < lowest_key) return -1;
        const int block = key >> page_shift;
        const int page = block < table_width ? table[block] : -1;
        if (page < 0 || page >= pages) {
            holes = true;
            return -1;
        }
        return (page * kv_heads + kv_head) * units_per_page + ((key & ((1 << page_shift) - 1)) >> 4);
    };
    int tile = from + warp, turn = 0;          // turn: of AHEAD, the place of the next tile to be asked for
    int units_now = look_up(tile), units_next = -1;
    const uint32_t my_ring = shared_address(ring) + lane * P::UNIT;
    auto fetch = [&](int stage, int asked) {
        const int unit = __shfl_sync(0xffffffffu, units_now, turn * UNITS + (lane & (UNITS - 1)));
        const unsigned live = __ballot_sync(0xffffffffu, lane < UNITS && unit >= 0);
        if (lane == 0) barrier_expect(barrier(stage), (uint32_t)__popc(live) * P::UNIT);
        __syncwarp();
        if (lane < UNITS && unit >= 0)
            bulk_load(my_ring + stage * R::STAGE, codes + (size_t)unit * P::UNIT, P::UNIT, barrier(stage));
        if (turn == AHEAD / 2) units_next = look_up(asked + (AHEAD - AHEAD / 2) * WARPS);
        if (++turn == AHEAD) {
            turn = 0;
            units_now = units_next;
        }
    };
#pragma unroll
    for (int ahead = 0; ahead < R::STAGES - 1; ++ahead)
        if (tile + ahead * WARPS < to) fetch(ahead, tile + ahead * WARPS);

    // q^T as the 8-column operand (head r, dims 16 s + 2c, + 1 and + 8), in NP parts
    uint32_t qb[RUNS][2][NP];
    {
        const bool live = r < rows;
        const T* row = queries + ((size_t)request * heads + head0 + (live ? r : 0)) * HD;
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const T* at = row + 16 * s + 8 * half + 2 * c;
                if constexpr (WIDE) {
                    const float2 v = *reinterpret_cast<const float2*>(at);
                    parts_of<NP>(live ? v.x : 0.f, live ? v.y : 0.f, qb[s][half]);
                } else {
                    qb[s][half][0] = live ? *reinterpret_cast<const uint32_t*>(at) : 0u;
                }
            }
    }
    // scale sum(q) of every group for heads 2c and 2c + 1, by a product with ones
    constexpr uint32_t ONES = 0x3f803f80u;
    float sums[GROUPS][2];
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
        float small[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = g * GROUP_RUNS; s < (g + 1) * GROUP_RUNS; ++s)
#pragma unroll
            for (int n = NP - 1; n >= 0; --n)
                mma_16816(n ? small : sum, ONES, ONES, ONES, ONES, qb[s][0][n], qb[s][1][n]);
        sums[g][0] = (sum[0] + small[0]) * scale_log2;
        sums[g][1] = (sum[1] + small[1]) * scale_log2;
    }

    // bfloat16 queries as half-precision, and what a score's product with the codes is then to be multiplied by
    float code_scale = scale_log2;
    if constexpr (!WIDE) {
        float most = 0.f;
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float a = fabsf(low_of(qb[s][half][0])), b = fabsf(high_of(qb[s][half][0]));
                if (a < INFINITY) most = fmaxf(most, a);
                if (b < INFINITY) most = fmaxf(most, b);
            }
        float inverse;
        const float by = power_towards(warp_max(most), 13, inverse);
        code_scale = scale_log2 * CODE_UNIT * inverse;
#pragma unroll
        for (int s = 0; s < RUNS; ++s)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const float to = half ? by * 0.0625f : by;
                qb[s][half][0] = pack_half(low_of(qb[s][half][0]) * to, high_of(qb[s][half][0]) * to);
            }
    }

    // heads 2c, 2c + 1: what scores are taken against, whether that has come from a score yet, this lane's
    // share of the sum
    float m[2] = {0.f, 0.f}, l[2] = {0.f, 0.f};
    bool begun[2] = {false, false};
    if (sinks != nullptr && split == 0 && warp == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (2 * c + i < rows) {
                // a sink: a term of the denominator with neither key nor value
                const float sink = sinks[head0 + 2 * c + i] * LOG2E;
                begun[i] = !(sink < NOTHING);
                if (begun[i]) {
                    m[i] = sink;
                    l[i] = r == 0 ? 1.f : 0.f;
                }
            }
    }
    float o[RUNS][4], lows[GROUPS][2];     // outputs, sums of p lowest
    float grown = 1.2676506e30f, shrunk = 7.8886091e-31f;    // (not WIDE) the weights' power of two, 2^100 at first
#pragma unroll
    for (int s = 0; s < RUNS; ++s)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[s][k] = 0.f;
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) lows[g][0] = lows[g][1] = 0.f;

    // One tile: `held` its units, `first` its first key, `some` whether a unit with keys to be seen has no page.
    auto attend = [&](auto masked, const unsigned char* held, int first, bool some) {
        constexpr bool MASKED = decltype(masked)::value;
        // which of this lane's keys are seen: two bits a unit, r and r + 8
        uint32_t seen = 0;
        if (MASKED) {
#pragma unroll
            for (int i = 0; i < 2 * UNITS; ++i) {
                const int key = first + 8 * i + r;
                bool there = key >= lowest_key && key <= position;
                if (some && there) {
                    const int block = key >> page_shift;
                    const int page = block < table_width ? table[block] : -1;
                    there = page >= 0 && page < pages;
                }
                if (there) seen |= 1u << i;
            }
        }
        // scores (times log2 e), less what they are taken against
        float s[UNITS][4];
#pragma unroll
        for (int u = 0; u < UNITS; ++u) {
            const unsigned char* part = held + u * P::UNIT;
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) {
                float acc[4], small[4];
                if constexpr (WIDE) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) acc[k] = small[k] = 0.f;
                }
                uint32_t words[GROUP_RUNS];
                load_words(part + P::word_at(lane, g * GROUP_RUNS), words);
#pragma unroll
                for (int k = 0; k < GROUP_RUNS; ++k) {
                    uint32_t a[4];
                    const auto& b = qb[g * GROUP_RUNS + k];
                    if constexpr (WIDE) {
                        expand_centred(words[k], a);
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n)
                            mma_16816(n ? small : acc, a[0], a[2], a[1], a[3], b[0][n], b[1][n]);
                    } else {
                        expand_small(words[k], a);
                        if (k == 0) mma_half_first(acc, a[0], a[2], a[1], a[3], b[0][0], b[1][0]);
                        else mma_half(acc, a[0], a[2], a[1], a[3], b[0][0], b[1][0]);
                    }
                }
                const uint2 scale = *reinterpret_cast<const uint2*>(part + P::scale_at(r, g));
                const float step[2] = {packed_step(scale.x) * code_scale, packed_step(scale.y) * code_scale};
                float low[2] = {packed_lowest(scale.x), packed_lowest(scale.y)};
                if (WIDE) {
                    low[0] = fmaf(MIDDLE, packed_step(scale.x), low[0]);
                    low[1] = fmaf(MIDDLE, packed_step(scale.y), low[1]);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    s[u][k] = fmaf(low[k >> 1], sums[g][k & 1], g ? s[u][k] : -m[k & 1]);
                    s[u][k] = fmaf(step[k >> 1], NP > 1 ? acc[k] + small[k] : acc[k], s[u][k]);
                }
            }
            if (MASKED) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (!(seen >> (2 * u + (k >> 1)) & 1u)) s[u][k] = -INFINITY;
            }
        }
        // the values' steps and lowest values of this lane's keys; of keys that are not seen, whatever lies
        // there, zeros
        float step[GROUPS][UNITS][2], low[GROUPS][UNITS][2], largest = 0.f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                const uint2 scale = *reinterpret_cast<const uint2*>(held + u * P::UNIT + P::PART + P::scale_at(r, g));
                step[g][u][0] = packed_step(scale.x); step[g][u][1] = packed_step(scale.y);
                low[g][u][0] = packed_lowest(scale.x); low[g][u][1] = packed_lowest(scale.y);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    if (MASKED && !(seen >> (2 * u + i) & 1u)) step[g][u][i] = low[g][u][i] = 0.f;
                    if (WIDE) low[g][u][i] = fmaf(MIDDLE, step[g][u][i], low[g][u][i]);
                }
                if (!WIDE) largest = max_of_three(largest, step[g][u][0], step[g][u][1]);
            }
        float top[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            top[i] = fmaxf(s[0][i], s[0][i + 2]);
#pragma unroll
            for (int u = 1; u < UNITS; ++u) top[i] = max_of_three(top[i], s[u][i], s[u][i + 2]);
        }
        if (__any_sync(0xffffffffu, fmaxf(top[0], top[1]) > LAZY || !(begun[0] && begun[1]) ||
                                        (!WIDE && largest * grown > 1024.f))) {
            float resized = 1.f;
            if constexpr (!WIDE) {
                largest = warp_max(largest);
                if (largest * grown > 1024.f) {
                    const float before = shrunk;
                    grown = power_towards(largest, 9, shrunk);
                    resized = grown * before;
                }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int offset = 4; offset < 32; offset <<= 1)
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], offset));
                // (the first score of a head may lie anywhere; from then on the maximum only rises)
                const bool any = top[i] > -INFINITY;
                const float rise = begun[i] ? fmaxf(top[i], 0.f) : any ? top[i] : 0.f;
                const float by = begun[i] ? fast_exp2(-rise) : 1.f, of_output = by * resized;
                begun[i] = begun[i] || any;
                m[i] += rise;
                l[i] *= by;
#pragma unroll
                for (int u = 0; u < UNITS; ++u) {
                    s[u][i] -= rise;
                    s[u][i + 2] -= rise;
                }
#pragma unroll
                for (int g = 0; g < GROUPS; ++g) lows[g][i] *= by;
#pragma unroll
                for (int k = 0; k < RUNS; ++k) {
                    o[k][i] *= of_output;
                    o[k][i + 2] *= of_output;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < UNITS; ++u)
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                s[u][k] = fast_exp2(s[u][k]);                // from here on p
                l[k & 1] += s[u][k];
            }
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
#pragma unroll
            for (int u = 0; u < UNITS; ++u) {
                // the group's weights p step, transposed: keys 2c, + 1 (and + 8), head r
                uint32_t pb[2][NP];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const float factor = WIDE ? step[g][u][half] : step[g][u][half] * grown;
                    lows[g][0] = fmaf(s[u][2 * half], low[g][u][half], lows[g][0]);
                    lows[g][1] = fmaf(s[u][2 * half + 1], low[g][u][half], lows[g][1]);
                    const float a = s[u][2 * half] * factor, b = s[u][2 * half + 1] * factor;
                    if constexpr (WIDE) parts_of<NP>(a, b, pb[half]);
                    else pb[half][0] = pack_half(a, b);
#pragma unroll
                    for (int n = 0; n < NP; ++n) pb[half][n] = transpose_8x8(pb[half][n]);
                }
                uint32_t words[GROUP_RUNS];
                load_words(held + u * P::UNIT + P::PART + P::word_at(lane, g * GROUP_RUNS), words);
#pragma unroll
                for (int k = 0; k < GROUP_RUNS; ++k) {
                    uint32_t a[4];
                    float (&to)[4] = o[g * GROUP_RUNS + k];
                    if constexpr (WIDE) {
                        expand_centred(words[k], a);
                        float small[4] = {0.f, 0.f, 0.f, 0.f}, large[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int n = NP - 1; n >= 0; --n)
                            mma_16816(n ? small : large, a[0], a[1], a[2], a[3], pb[0][n], pb[1][n]);
#pragma unroll
                        for (int x = 0; x < 4; ++x) to[x] += large[x] + small[x];
                    } else {
                        expand_small(words[k], a);
                        mma_half(to, a[0], a[1], a[2], a[3], pb[0][0], pb[1][0]);
                    }
                }
            }
    };

    bool ok = true;
    int stage = 0;
    uint32_t parity = 0;
    for (; tile < to; tile += WARPS) {
        {
            const int next = tile + (R::STAGES - 1) * WARPS;
            __syncwarp();                  // every lane is done with the stage that is filled now
            if (next < to) fetch(stage == 0 ? R::STAGES - 1 : stage - 1, next);
        }
        for (int i = 0; !barrier_test(barrier(stage), parity); ++i)
            if (i >= WAIT_LIMIT) { ok = false; break; }
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const unsigned char* held = ring + stage * R::STAGE;
        const int first = tile * KEYS;
        // (a tile whose keys are all seen needs no mask)
        const bool some = __any_sync(0xffffffffu, holes);
        if (first >= lowest_key && first + KEYS - 1 <= position && !some)
            attend(std::false_type{}, held, first, false);
        else
            attend(std::true_type{}, held, first, some);
        stage = stage + 1 == R::STAGES ? 0 : stage + 1;
        if (stage == 0) parity ^= 1;
    }
    if (!ok && lane == 0) atomicExch(error_flag, ERROR_WAIT);

    // the lanes' shares of the sums; every lane has its own dimensions of the output
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int offset = 4; offset < 32; offset <<= 1) {
            l[i] += __shfl_xor_sync(0xffffffffu, l[i], offset);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g) lows[g][i] += __shfl_xor_sync(0xffffffffu, lows[g][i], offset);
        }
    }
    // A warp that gave up leaves no copy of its own behind: a bounded wait for the stages that it had asked for.
    if (!ok)
        for (int k = 0; k < R::STAGES; ++k)
            for (int i = 0; i < WAIT_LIMIT / 16 && !barrier_test(barrier(k), k >= stage ? parity : parity ^ 1); ++i) {}
    __syncthreads();
    // [warp][head][HD + 2]: outputs, maximum, sum, where the rings were
    float* merge = reinterpret_cast<float*>(shared);
    constexpr int ROW = HD + 2;
    {
        float* mine = merge + warp * HEADS * ROW;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            float* row = mine + (2 * c + i) * ROW;
#pragma unroll
            for (int k = 0; k < RUNS; ++k) {
                const int g = k / GROUP_RUNS;
                // (not WIDE: codes were 2^-24 of themselves, 2^-20 in dimensions r + 8, weights `grown` times)
                const float a = WIDE ? o[k][i] : o[k][i] * CODE_UNIT * shrunk;
                const float b = WIDE ? o[k][i + 2] : o[k][i + 2] * (CODE_UNIT / 16.f) * shrunk;
                row[16 * k + r] = a + lows[g][i];
                row[16 * k + r + 8] = b + lows[g][i];
            }
            if (r == 0) {
                row[HD] = begun[i] ? m[i] : NOTHING;
                row[HD + 1] = l[i];
            }
        }
    }
    __syncthreads();
    if (splits == 1) {
        // no key and no sink: zeros; a sum that is no number stays one
        for (int i = threadIdx.x; i < rows * HD / 2; i += WARPS * 32) {
            const int head = i / (HD / 2), d = i % (HD / 2) * 2;
            float top = NOTHING;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) top = fmaxf(top, merge[(w * HEADS + head) * ROW + HD]);
            float sum = 0.f, a = 0.f, b = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float* row = merge + (w * HEADS + head) * ROW;
                const float by = fast_exp2(row[HD] - top);
                sum = fmaf(by, row[HD + 1], sum);
                a = fmaf(by, row[d], a);
                b = fmaf(by, row[d + 1], b);
            }
            const float inverse = sum == 0.f ? 0.f : 1.f / sum;
            store_pair(out + ((size_t)request * heads + head0 + head) * HD + d, a * inverse, b * inverse);
        }
        return;
    }
    // the block's result behind the warps' rows
    float* block_row = merge + WARPS * HEADS * ROW;
    for (int i = threadIdx.x; i < HEADS * HD; i += WARPS * 32) {
        const int head = i / HD, d = i % HD;
        float top = NOTHING;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, merge[(w * HEADS + head) * ROW + HD]);
        float sum = 0.f, value = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float* row = merge + (w * HEADS + head) * ROW;
            const float by = fast_exp2(row[HD] - top);
            sum = fmaf(by, row[HD + 1], sum);
            value = fmaf(by, row[d], value);
        }
        block_row[head * ROW + d] = value;
        if (d == 0) {
            block_row[head * ROW + HD] = top;
            block_row[head * ROW + HD + 1] = sum;
        }
    }
    if (partial != nullptr) {
        __syncthreads();
        for (int i = threadIdx.x; i < rows * ROW; i += WARPS * 32)
            partial[(((size_t)request * heads + head0 + i / ROW) * splits + split) * ROW + i % ROW] = block_row[i];
        return;
    }
    // the splits are a cluster: block `split` adds up every splits-th pair of dimensions
    cg::cluster_group cluster = cg::this_cluster();
    cluster.sync();
    for (int i = split * WARPS * 32 + threadIdx.x; i < rows * HD / 2; i += splits * WARPS * 32) {
        const int head = i / (HD / 2), d = i % (HD / 2) * 2;
        float top = NOTHING;
        for (int k = 0; k < splits; ++k) top = fmaxf(top, cluster.map_shared_rank(block_row, k)[head * ROW + HD]);
        float sum = 0.f, a = 0.f, b = 0.f;
        for (int k = 0; k < splits; ++k) {
            const float* row = cluster.map_shared_rank(block_row, k) + head * ROW;
            const float by = fast_exp2(row[HD] - top);
            sum = fmaf(by, row[HD + 1], sum);
            a = fmaf(by, row[d], a);
            b = fmaf(by, row[d + 1], b);
        }
        const float inverse = sum == 0.f ? 0.f : 1.f / sum;
        store_pair(out + ((size_t)request * heads + head0 + head) * HD + d, a * inverse, b * inverse);
    }
    cluster.sync();                        // nobody leaves while its rows are read
}

// The merge of more splits than a cluster holds: partial [rows, splits, HD + 2] -> out [rows, HD], a warp a row.
template <typename T, int HD>
__global__ void __launch_bounds__(128)
merge_kernel(const float* partial, T* out, int rows, int splits) {
    griddep_launch();
    griddep_wait();
    const float* written = settled(partial);
    const int row = blockIdx.x * 4 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (row >= rows) return;
    const float* from = written + (size_t)row * splits * (HD + 2);
    float top = NOTHING;
    for (int k = lane; k < splits; k += 32) top = fmaxf(top, from[k * (HD + 2) + HD]);
    top = warp_max(top);
    float sum = 0.f, value[HD / 32];
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) value[i] = 0.f;
    for (int k = 0; k < splits; ++k) {
        const float* at = from + k * (HD + 2);
        const float by = fast_exp2(at[HD] - top);
        sum = fmaf(by, at[HD + 1], sum);
#pragma unroll
        for (int i = 0; i < HD / 32; ++i) value[i] = fmaf(by, at[lane + 32 * i], value[i]);
    }
    const float inverse = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) out[(size_t)row * HD + lane + 32 * i] = from_float<T>(value[i] * inverse);
}

template <typename T, int HD>
int launch_packed(const void* q, const void* cache, const int* block_table, int table_width, int page_shift,
                  int pages, const int* positions, void* out, float* partial, int requests, int heads,
                  int kv_heads, int splits, float scale, int window, const float* sinks, int* error_flag,
                  cudaStream_t stream) {
    auto kernel = attention_packed_kernel<T, HD>;
    static thread_local int prepared = -1;                 // (the device that the attribute was set on)
    int device = 0;
    cudaGetDevice(&device);
    if (prepared != device) {
        const cudaError_t error =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<T, HD>::SHARED);
        MLXONE_REQUIRE(error == cudaSuccess, "attention_packed: %s", cudaGetErrorString(error));
        prepared = device;
    }
    const int groups = kv_heads * ceil_div_host(heads / kv_heads, HEADS);
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(splits, groups, requests);
    config.blockDim = dim3(WARPS * 32);
    config.dynamicSmemBytes = Ring<T, HD>::SHARED;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    int count = 0;
    if (partial == nullptr && splits > 1) {
        attributes[count].id = cudaLaunchAttributeClusterDimension;
        attributes[count].val.clusterDim.x = splits;
        attributes[count].val.clusterDim.y = 1;
        attributes[count].val.clusterDim.z = 1;
        ++count;
    }
    if (mlxone_pdl_enabled()) {
        attributes[count].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attributes[count].val.programmaticStreamSerializationAllowed = 1;
        ++count;
    }
    config.attrs = attributes;
    config.numAttrs = count;
    cudaLaunchKernelEx(&config, kernel, (const T*)q, (const unsigned char*)cache, block_table, table_width,
                       page_shift, pages, positions, (T*)out, partial, heads, kv_heads, splits,
                       scale * LOG2E, window, sinks, error_flag);
    MLXONE_LAUNCH_CHECK("attention_packed");
    if (partial != nullptr) {
        const int rows = requests * heads;
        launch_kernel(merge_kernel<T, HD>, dim3(ceil_div_host(rows, 4)), dim3(128), 0, stream, true,
                      (const float*)partial, (T*)out, rows, splits);
        MLXONE_LAUNCH_CHECK("attention_packed merge");
    }
    return 0;
}

}  // namespace

// Splits that a cluster merges; more need `partial`.
MLXONE_API int mlxone_attention_packed_cluster() { return CLUSTER; }

// One token a request: q [requests, heads, head_dim], positions [requests] (each token's own position: the last key
// that it sees; below 0: none). window: as first_visible_key's span. sinks: float32 [heads] or null. partial:
// null where `splits` is at most mlxone_attention_packed_cluster(), else requests * heads * splits *
// (head_dim + 2) floats. Keys without a page are not seen.
MLXONE_API int mlxone_attention_packed(const void* q, const void* cache, const int* block_table, int table_width,
                                       int page_size, int pages, const int* positions, void* out, float* partial,
                                       int requests, int heads, int kv_heads, int head_dim, int splits, float scale,
                                       int window, const float* sinks, int dtype, int* error_flag,
                                       cudaStream_t stream) {
    if (requests == 0) return 0;
    MLXONE_REQUIRE(requests > 0 && requests <= 65535 && heads > 0 && kv_heads > 0 && heads % kv_heads == 0,
                   "attention_packed: bad sizes");
    MLXONE_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0 && pages > 0 && table_width > 0,
                   "attention_packed: pages hold a power of two of tokens, 16 or more, not %d", page_size);
    MLXONE_REQUIRE(splits >= 1 && splits <= 65535 && (partial != nullptr || splits <= CLUSTER),
                   "attention_packed: %d splits need scratch", splits);
    MLXONE_REQUIRE(kv_heads * (long long)ceil_div_host(heads / kv_heads, HEADS) <= 65535,
                   "attention_packed: too many heads");
    MLXONE_REQUIRE((long long)pages * kv_heads * (page_size / 16) <= 0x7fffffff,
                   "attention_packed: a cache of more than 2^31 units of 16 tokens of a head");
    MLXONE_REQUIRE((((size_t)cache | (size_t)q) & 15) == 0,
                   "attention_packed: cache and queries start at multiples of 16 bytes");
    const int page_shift = 31 - __builtin_clz((unsigned)page_size);
#define CALL(HD)                                                                                               \
    if (dtype == MLXONE_BF16)                                                                                  \
        return launch_packed<bf16, HD>(q, cache, block_table, table_width, page_shift, pages, positions, out,  \
                                       partial, requests, heads, kv_heads, splits, scale, window, sinks,       \
                                       error_flag, stream);                                                    \
    else                                                                                                       \
        return launch_packed<float, HD>(q, cache, block_table, table_width, page_shift, pages, positions, out, \
                                        partial, requests, heads, kv_heads, splits, scale, window, sinks,      \
                                        error_flag, stream)
    MLXONE_PACKED_DIMS(CALL)
#undef CALL
    return 0;
}
MLXONE_BY_WORDS(mlxone_attention_packed)
