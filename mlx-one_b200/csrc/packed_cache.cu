// Keys and values of a step's tokens written to pages of 4-bit codes (packed_cache.cuh has the format),
// read back, and whole requests opened into pages of plain values.
//
// Writing. For a group of a token's values: lowest = bfloat16(min), step = bfloat16(max(max - lowest, 0) * (1 / 15),
// difference, inverse and product in 32 bits: not always the quotient's bits, so it is the product that defines
// the format, as a tensor divided by the number 15 on this GPU), code = (x - lowest) / step to the nearest whole number, ties to
// even, cut to 0..15. The codes are those of exact arithmetic on the stored lowest and step (codes_of). A group
// with a value that is not finite, or whose range is none, gets NaN as step and lowest: it stays visible.
//
// Measured, us on the GPU, written and read back (two launches): 16 tokens of 8 heads of 64 5.3 (loads one after the
// other: owner and position, the row and its page), two portions of 2,048 tokens 16.7 (24 MB; 3.7 at the copy rate),
// of which the writing takes 10: about 50 instructions for 32 values, and three loads in a row before the first.
// A portion of 1,024 tokens behind 3,076 keys, opened in half-precision and attended to, 71.3; over pages of bfloat16 66.8.
#include <cuda_fp16.h>

#include "by_words.cuh"
#include "packed_cache.cuh"

namespace {

using bf16 = __nv_bfloat16;
constexpr int ERROR_WRITE = 2;        // a key written to a position that has no page
constexpr int ERROR_READ = 3;         // a key read from a position that has no page
constexpr int TOKENS = 16;            // of a block

template <typename T>
__device__ __forceinline__ void load_eight(const T* src, bool wide, float (&x)[8]) {
    if (wide) {
        if constexpr (sizeof(T) == 2) {
            const uint4 raw = *reinterpret_cast<const uint4*>(src);
            const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = __uint_as_float(words[i] << 16);
                x[2 * i + 1] = __uint_as_float(words[i] & 0xffff0000u);
            }
        } else {
            const float4 a = *reinterpret_cast<const float4*>(src);
            const float4 b = *reinterpret_cast<const float4*>(src + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_float<T>(src[i]);
    }
}

// Whether x lies above the tie between code and code + 1 (on it: whether code is odd), in exact arithmetic: the
// difference from lowest with its own rounding (a two-term sum), and the tie, (code + 1/2) step, a number of 13
// bits, which the difference is near enough to be taken from without rounding.
__device__ __forceinline__ bool above_tie(float x, float lowest, float step, int code) {
    const float above = x - lowest, back = above - x;
    const float lost = (x - (above - back)) - (lowest + back);
    const float rest = above - ((float)code + 0.5f) * step;
    return rest > 0.f || (rest == 0.f && (lost > 0.f || (lost == 0.f && (code & 1))));
}

// The codes of eight values, four bits each. The quotient is the 32-bit one: a product with the inverse, corrected
// once by the inverse times its remainder, which one fused operation gives exactly (P. Markstein, "Computation of
// elementary functions on the IBM RISC System/6000 processor", 1990); adding 1.5 * 2^23 rounds to a whole number, ties to even, that lies in the sum's last bits. With
// bfloat16 values that is exact unless one is below 2^-15 of lowest: x - lowest has 24 bits, and a quotient of
// a number of 24 bits by one of 8 either is a tie or lies 2^-18 of itself away from it. What may be decided
// wrongly by it (32-bit values within 1e-5 of a tie) is decided again, exactly.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float lowest, float step) {
    const float inverse = 1.f / step;
    constexpr float WHOLE = 12582912.f;
    uint32_t codes = 0;
    float furthest = 0.f, least = INFINITY;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float above = x[i] - lowest, near = above * inverse;
        const float ratio = fminf(fmaxf(fmaf(fmaf(-near, step, above), inverse, near), 0.f), 15.f);
        const float raised = ratio + WHOLE;
        furthest = fmaxf(furthest, fabsf(ratio - (raised - WHOLE)));
        if (sizeof(T) == 2) least = fminf(least, fabsf(x[i]));
        codes = codes * 16u + (__float_as_uint(raised) - __float_as_uint(WHOLE));
    }
    const bool doubtful = sizeof(T) == 4 || least < fabsf(lowest) * 3.0517578e-5f;
    // (or a step so small that its inverse, or what the correction works with, is none)
    if ((doubtful && !(furthest <= 0.49999f)) || !(inverse < 1e30f)) {
        codes = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float ratio = fminf(fmaxf((x[i] - lowest) / step, 0.f), 15.f);
            int code = (int)ratio;
            const float past = ratio - (float)code;
            if (fabsf(past - 0.5f) > 2e-5f) code += past > 0.5f;
            else code += above_tie(x[i], lowest, step, code);
            codes |= (uint32_t)min(code, 15) << (4 * i);
        }
    }
    return codes;
}
// the larger (smaller) of two and NaN if either is
__device__ __forceinline__ float max_nan(float a, float b) {
    float c;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
__device__ __forceinline__ float min_nan(float a, float b) {
    float c;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(c) : "f"(a), "f"(b));
    return c;
}
// four neighbouring codes (16 bits) to a byte each
__device__ __forceinline__ uint32_t spread(uint32_t four) {
    four = (four | four << 8) & 0x00ff00ffu;
    return (four | four << 4) & 0x0f0f0f0fu;
}

// One block: the runs of tokens that begin among 16 tokens of the step and share a unit (a run ends with its
// unit or its request), for one key head. HD / 8 lanes take a token's row, eight neighbouring values each: the
// group's extremes by shuffles, and one exchange of codes with the neighbour that holds the run's other
// eight dimensions, whose codes share its bytes. The 16 tokens of a whole unit (at most one begins in a block)
// are put together in shared memory and leave in 16-byte pieces; tokens of a unit's part write their bytes
// one by one, since the others' stay as they are.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
pack_kernel(const T* keys, long long key_stride, const T* values,
            long long value_stride, int wide, const int* positions,
            const int* token_request, const int* request_start,
            const int* block_table, int table_width, int page_shift, int pages, int kv_heads,
            int tokens, unsigned char* cache, int* error_flag) {
    using P = Packed<HD>;
    constexpr int LANES = HD == 96 ? 16 : HD / 8;            // lanes of a row (four of 16 idle with 96 values)
    constexpr int GROUP_LANES = P::GROUP / 8;
    __shared__ __align__(16) unsigned char image[P::UNIT];
    __shared__ int span[3];                                  // first and last + 1 token, the whole unit's first
    griddep_launch();
    griddep_wait();
    const int head = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (warp == 0) {
        const int t = blockIdx.x * TOKENS + lane;
        bool begins = false;
        int length = 0;
        if (lane < TOKENS && t < tokens) {
            const int r = token_request[t], inside = positions[t] & 15;
            begins = inside == 0 || t == request_start[r];
            length = min(16 - inside, request_start[r + 1] - t);
        }
        const unsigned starts = __ballot_sync(0xffffffffu, begins);
        const unsigned full = __ballot_sync(0xffffffffu, begins && length == 16);
        const int last = 31 - __clz((int)(starts | 1u));
        const int end = __shfl_sync(0xffffffffu, t + length, last);
        if (lane == 0) {
            span[0] = blockIdx.x * TOKENS + (starts ? __ffs((int)starts) - 1 : 0);
            span[1] = starts ? min(end, tokens) : span[0];
            span[2] = full ? blockIdx.x * TOKENS + __ffs((int)full) - 1 : -1;
        }
    }
    __syncthreads();
    const int first = span[0], count = span[1] - span[0], whole = span[2];
    const int units = 1 << (page_shift - 4);
    auto unit_of = [&](int t) -> unsigned char* {
        const int position = positions[t], block = position >> page_shift;
        const int page = position >= 0 && block < table_width
                             ? block_table[(size_t)token_request[t] * table_width + block] : -1;
        if (page < 0 || page >= pages) return nullptr;
        return cache + (((size_t)page * kv_heads + head) * units + (position >> 4 & (units - 1))) * P::UNIT;
    };
    const int sub = threadIdx.x % LANES;                     // this thread's place in its row
    const bool live_lane = sub * 8 < HD;
    const int rows = 2 * count;                              // keys' rows, then values'
    // (where a row goes is looked up beside its load, not behind it)
    unsigned char* const whole_unit = whole >= 0 ? unit_of(whole) : nullptr;
    for (int base = 0; base < rows; base += blockDim.x / LANES) {
        const int row = base + threadIdx.x / LANES;
        const bool live = row < rows && live_lane;
        const int part = row >= count ? 1 : 0;
        const int t = first + (live ? row - part * count : 0);
        const bool imaged = whole >= 0 && t >= whole && t < whole + 16;
        const int key = live ? positions[t] & 15 : 0;
        unsigned char* unit = imaged ? image : live ? unit_of(t) : nullptr;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (live) {
            const T* src = (part ? values + (size_t)t * value_stride : keys + (size_t)t * key_stride) +
                           head * HD + sub * 8;
            load_eight<T>(src, wide, x);
        }
        float least = x[0], most = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            least = min_nan(least, x[i]);
            most = max_nan(most, x[i]);
        }
#pragma unroll
        for (int offset = 1; offset < GROUP_LANES; offset <<= 1) {
            least = min_nan(least, __shfl_xor_sync(0xffffffffu, least, offset));
            most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, offset));
        }
        const bf16 lowest_stored = __float2bfloat16_rn(least);
        const float lowest = __bfloat162float(lowest_stored);
        const bf16 step_stored = __float2bfloat16_rn(fmaxf(most - lowest, 0.f) * (1.f / 15.f));
        const float step = __bfloat162float(step_stored);
        const bool fine = isfinite(least) && isfinite(most) && isfinite(lowest) && isfinite(step);
        const uint32_t mine = fine && step > 0.f ? codes_of<T>(x, lowest, step) : 0u;
        // this lane's four bytes: dimensions e and e + 8 of the run, e from 4 (sub & 1) on
        const uint32_t other = __shfl_xor_sync(0xffffffffu, mine, 1);
        const uint32_t bytes = sub & 1 ? spread(other >> 16) | spread(mine >> 16) << 4
                                       : spread(mine & 0xffffu) | spread(other & 0xffffu) << 4;
        if (live) {
            if (unit == nullptr) {
                atomicExch(error_flag, ERROR_WRITE);
            } else {
                unit += part * P::PART;
                const int run = sub >> 1;
                const uint32_t words = fine ? (uint32_t)__bfloat16_as_ushort(step_stored) |
                                                  (uint32_t)__bfloat16_as_ushort(lowest_stored) << 16
                                            : 0x7fc07fc0u;
                // bytes e = 4 (sub & 1) + 0 .. 3: neighbouring pairs of a key's lanes, or every fourth lane
                const int half = sub & 1, lane_bytes = 4 * P::block_runs(run);
                unsigned char* at = unit + (part ? P::value_byte(key, run, 4 * half) : P::key_byte(key, run, 4 * half));
                const int second = part ? 4 * lane_bytes : 2, third = part ? 8 * lane_bytes : lane_bytes;
                at[0] = (unsigned char)bytes;
                at[second] = (unsigned char)(bytes >> 8);
                at[third] = (unsigned char)(bytes >> 16);
                at[third + second] = (unsigned char)(bytes >> 24);
                if (sub % GROUP_LANES == 0)
                    *reinterpret_cast<uint32_t*>(unit + P::scale_at(key, sub / GROUP_LANES)) = words;
            }
        }
    }
    if (whole >= 0) {
        __syncthreads();
        if (whole_unit == nullptr) {
            if (threadIdx.x == 0) atomicExch(error_flag, ERROR_WRITE);
        } else {
            for (int i = threadIdx.x; i < P::UNIT / 16; i += blockDim.x)
                reinterpret_cast<uint4*>(whole_unit)[i] = reinterpret_cast<const uint4*>(image)[i];
        }
    }
}

// Sixteen neighbouring values (run s of a key) from a part's codes, as one thread reads them.
template <int HD>
__device__ __forceinline__ void read_run(const unsigned char* part, int which, int key, int s, float (&x)[16]) {
    using P = Packed<HD>;
    const uint32_t word = *reinterpret_cast<const uint32_t*>(part + P::scale_at(key, s * 16 / P::GROUP));
    const float step = packed_step(word), lowest = packed_lowest(word);
    if (which) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t both = part[P::value_byte(key, s, e)];
            x[e] = fmaf(step, (float)(both & 15u), lowest);
            x[e + 8] = fmaf(step, (float)(both >> 4), lowest);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            // (dimensions e and e + 1 lie in one word)
            const uint32_t both = *reinterpret_cast<const uint32_t*>(part + (P::key_byte(key, s, e) & ~3)) >> (key & 8);
            x[e] = fmaf(step, (float)(both & 15u), lowest);
            x[e + 8] = fmaf(step, (float)(both >> 4 & 15u), lowest);
            x[e + 1] = fmaf(step, (float)(both >> 16 & 15u), lowest);
            x[e + 9] = fmaf(step, (float)(both >> 20 & 15u), lowest);
        }
    }
}

__device__ __forceinline__ void store_run(float* dst, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(dst + i) = make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]);
}
__device__ __forceinline__ void store_run(bf16* dst, const float (&x)[16]) {
    uint32_t words[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 pair = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        words[i] = *reinterpret_cast<const uint32_t*>(&pair);
    }
    *reinterpret_cast<uint4*>(dst) = make_uint4(words[0], words[1], words[2], words[3]);
    *reinterpret_cast<uint4*>(dst + 8) = make_uint4(words[4], words[5], words[6], words[7]);
}

// The values that the step's tokens find at their places: keys and values [tokens, kv_heads, HD]. A block
// takes 16 tokens of one head (neighbours share units, which the first reader brings into the cache), a
// thread a run of 16 values.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
read_kernel(const unsigned char* cache, const int* positions,
            const int* token_request, const int* block_table, int table_width,
            int page_shift, int pages, int kv_heads, int tokens, T* keys, T* values,
            int* error_flag) {
    using P = Packed<HD>;
    griddep_launch();
    griddep_wait();
    const int head = blockIdx.y, units = 1 << (page_shift - 4);
    const unsigned char* from = settled(cache);
    for (int i = threadIdx.x; i < TOKENS * 2 * P::RUNS; i += blockDim.x) {
        const int s = i % P::RUNS, which = i / P::RUNS & 1, t = blockIdx.x * TOKENS + i / (2 * P::RUNS);
        if (t >= tokens) continue;
        const int position = positions[t], block = position >> page_shift;
        const int page = position >= 0 && block < table_width
                             ? block_table[(size_t)token_request[t] * table_width + block] : -1;
        float x[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) x[e] = 0.f;
        if (page < 0 || page >= pages) {
            atomicExch(error_flag, ERROR_READ);
        } else {
            const unsigned char* unit =
                from + (((size_t)page * kv_heads + head) * units + (position >> 4 & (units - 1))) * P::UNIT;
            read_run<HD>(unit + which * P::PART, which, position & 15, s, x);
        }
        store_run((which ? values : keys) + ((size_t)t * kv_heads + head) * HD + s * 16, x);
    }
}

// Queries as half-precision, a row times the power of two that brings its largest to 2^10 (exact but for what is
// 2^-26 of the largest and less), whose inverse goes to `factors`. HD / 8 lanes a row, blocks of 256 threads.
template <int HD>
__device__ __forceinline__ void half_queries(const bf16* q, long long rows, uint4* out, float* factors,
                                             long long block, long long blocks) {
    constexpr int LANES = HD == 96 ? 16 : HD / 8, ROWS = 256 / LANES;
    const bf16* written = settled(q);
    const int sub = threadIdx.x % LANES;
    for (long long first = block * ROWS; first < rows; first += blocks * ROWS) {      // (one for a block)
        const long long row = first + threadIdx.x / LANES;
        const bool live = row < rows && sub * 8 < HD;
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.f;
        if (live) load_eight<bf16>(written + row * HD + sub * 8, true, x);
        float most = 0.f, inverse;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (fabsf(x[i]) < INFINITY) most = fmaxf(most, fabsf(x[i]));
#pragma unroll
        for (int offset = 1; offset < LANES; offset <<= 1)
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
        const float by = power_towards(most, 10, inverse);
        if (!live) continue;
        uint32_t pairs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 pair = __floats2half2_rn(x[2 * i] * by, x[2 * i + 1] * by);
            pairs[i] = *reinterpret_cast<const uint32_t*>(&pair);
        }
        out[row * (HD / 8) + sub] = make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
        if (sub == 0) factors[row] = inverse;
    }
}

// What opening into half-precision has to know ahead: the largest number, by its size, that the keys' and the
// values' part of `chunk_units` units of a request and key head may open to, largest [requests, open heads, 2,
// chunks]. And the queries in half-precision, by the layers of the grid behind the requests'.
template <int HD>
__global__ void __launch_bounds__(256)
range_kernel(const unsigned char* cache, const int* block_table, int table_width, int page_shift, int pages,
             const int* request_start, const int* history, int span, int first_request, int requests, int first_head,
             int kv_heads, int chunk_units, float* largest, const bf16* q, long long rows, uint4* halves,
             float* query_factors) {
    using P = Packed<HD>;
    __shared__ float scratch[33];
    griddep_launch();
    griddep_wait();
    if ((int)blockIdx.z >= requests) {
        const long long layer = (long long)gridDim.x * gridDim.y;
        half_queries<HD>(q, rows, halves, query_factors,
                         (blockIdx.z - requests) * layer + blockIdx.y * gridDim.x + blockIdx.x,
                         (gridDim.z - requests) * layer);
        return;
    }
    const unsigned char* from = settled(cache);
    const int chunk = blockIdx.x, head = first_head + blockIdx.y, request = first_request + blockIdx.z;
    const int held = history[request];
    const int length = held + request_start[request + 1] - request_start[request];
    const int lowest_key = first_visible_key(held, span), units = 1 << (page_shift - 4);
    float most[2] = {0.f, 0.f};
#pragma unroll 4
    for (int i = threadIdx.x; i < chunk_units * 16; i += 256) {
        const int first = (chunk * chunk_units + i / 16) * 16, place = i % 16;
        if (first + place / 2 + 8 * (place & 1) >= length || first + 15 < lowest_key) continue;
        const int block = first >> page_shift;
        const int page = block < table_width ? block_table[(size_t)request * table_width + block] : -1;
        if (page < 0 || page >= pages) continue;
        const unsigned char* part =
            from + (((size_t)page * kv_heads + head) * units + (first >> 4 & (units - 1))) * P::UNIT;
#pragma unroll
        for (int g = 0; g < 2 * P::GROUPS; ++g) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(part + g % 2 * P::PART + P::CODES + 64 * (g / 2) +
                                                                     4 * place);
            const float lowest = packed_lowest(word);
            // (what is no number counts as nothing)
            most[g % 2] = fmaxf(most[g % 2], fmaxf(fabsf(lowest), fabsf(fmaf(15.f, packed_step(word), lowest))));
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const float all = block_max(most[k], scratch);
        if (threadIdx.x == 0)
            largest[(((size_t)blockIdx.z * gridDim.y + blockIdx.y) * 2 + k) * gridDim.x + chunk] = all;
    }
}

// Requests opened: every unit that the requests' tables name, up to their last token, as plain values in
// pages [2, requests * blocks, open_heads, open_size, HD] of their own, request r's block b in page r * blocks
// + b, of the key heads from first_head on; rows behind the last token, and of units without a page, are zeros,
// so that no reader meets a number that is none. A token whose keys or values are none has NaN for its keys and
// zeros for its values: queries that see it get NaN by their scores, the others nothing, since a reader drops
// scores that are masked but multiplies every value. A key that a token of the step sees (by `window`, or as one
// of the first keep_first positions) but that has no page is told of: its row of zeros would count as a
// key, for the readers do not look whether an opened row had a page. So are keys behind the last opened page. `table` gets the page numbers and, behind them, where the
// requests' tokens start, counted from the first one's. With `largest` (range_kernel's, `chunks` of them each) the
// pages are half-precision, keys and values times the powers of two that bring the largest of a request and key
// head to 2^9, whose inverses go to `factors` [requests, open heads, 2]: 11 bits of every number of 2^-23 of the
// largest and more, where bfloat16 has 8. A thread takes a run of four keys, 2j, 2j + 1, 2j + 8 and 2j + 9: every byte of its
// eight words is theirs, of the keys' part as of the values'.
template <typename T, int HD>
__global__ void __launch_bounds__(256)
open_kernel(const unsigned char* cache, const int* block_table, int table_width, int page_shift, int pages,
            const int* request_start, const int* history, int span, int window, int keep_first, int first_request,
            int first_head, int kv_heads, int blocks, int open_size, long long half, T* opened, int* table,
            const float* largest, int chunks, float* factors, int* error_flag) {
    using P = Packed<HD>;
    constexpr int THREADS = 8 * P::RUNS;                         // of a unit
    griddep_launch();
    griddep_wait();
    const unsigned char* from = settled(cache);
    const int r = blockIdx.z, open_head = blockIdx.y, head = first_head + open_head;
    const int request = first_request + r;
    const int held = history[request];
    const int length = held + request_start[request + 1] - request_start[request];
    const int per_block = open_size / 16;
    const int inside = threadIdx.x % THREADS;
    const int unit = blockIdx.x * (blockDim.x / THREADS) + threadIdx.x / THREADS;
    float raise = 1.f;
    if (largest != nullptr) {
        const float* mine = settled(largest) + ((size_t)r * gridDim.y + open_head) * 2 * chunks;
        float most[2] = {0.f, 0.f}, inverse[2];
        for (int i = threadIdx.x & 31; i < chunks; i += 32) {
            most[0] = fmaxf(most[0], mine[i]);
            most[1] = fmaxf(most[1], mine[chunks + i]);
        }
        const float of_keys = power_towards(warp_max(most[0]), 9, inverse[0]);
        const float of_values = power_towards(warp_max(most[1]), 9, inverse[1]);
        raise = inside / P::RUNS & 1 ? of_values : of_keys;
        if (blockIdx.x == 0 && threadIdx.x < 2)
            factors[((size_t)r * gridDim.y + open_head) * 2 + threadIdx.x] = inverse[threadIdx.x];
    }
    if (unit >= blocks * per_block) return;
    const int open_block = unit / per_block;
    if (open_head == 0 && inside == 0 && unit % per_block == 0) {
        table[(size_t)r * blocks + open_block] = r * blocks + open_block;
        if (unit == 0) {
            // (keys behind the last opened page: `blocks` comes from a bound that the host knows)
            if (length > held && (length - 1) / open_size >= blocks) atomicExch(error_flag, ERROR_READ);
            int* starts = table + (size_t)gridDim.z * blocks;
            const int base = request_start[first_request];
            starts[r] = request_start[request] - base;
            if (r + 1 == (int)gridDim.z) starts[r + 1] = request_start[request + 1] - base;
        }
    }
    if (open_block * open_size >= length) return;
    const int s = inside % P::RUNS, which = inside / P::RUNS & 1, j = inside / (2 * P::RUNS);
    const int first = unit * 16;
    const bool seen = first < length && first + 15 >= first_visible_key(held, span);
    const int block = first >> page_shift;
    int page = seen && block < table_width ? block_table[(size_t)request * table_width + block] : -1;
    if (page >= pages) page = -1;
    if (page < 0 && first < length && length > held &&
        (first + 15 >= first_visible_key(held, window) || first < keep_first) && open_head == 0 && inside == 0)
        atomicExch(error_flag, ERROR_READ);
    uint32_t words[8];
    float step[4], lowest[4];
#pragma unroll
    for (int k = 0; k < 8; ++k) words[k] = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) step[k] = lowest[k] = 0.f;
    if (page >= 0) {
        const int units = 1 << (page_shift - 4);
        const unsigned char* part =
            from + (((size_t)page * kv_heads + head) * units + (first >> 4 & (units - 1))) * P::UNIT + which * P::PART;
#pragma unroll
        for (int k = 0; k < 8; ++k)      // keys: rows 2j and 2j + 1, c = k % 4; values: r = k, c = j
            words[k] = *reinterpret_cast<const uint32_t*>(
                part + P::word_at(which ? 4 * k + j : 4 * (2 * j + k / 4) + k % 4, s));
        // (the words of keys 2j, 2j + 8, 2j + 1, 2j + 9 lie side by side)
        uint32_t none = 0;
#pragma unroll
        for (int g = 0; g < 2 * P::GROUPS; ++g) {
            const uint4 scale = *reinterpret_cast<const uint4*>(part + (g % 2 - which) * P::PART + P::scale_at(2 * j, g / 2));
            const uint32_t of_key[4] = {scale.x, scale.z, scale.y, scale.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                if (!isfinite(packed_step(of_key[k]))) none |= 1u << k;
                if (g == 2 * (s * 16 / P::GROUP) + which) {
                    step[k] = packed_step(of_key[k]);
                    lowest[k] = packed_lowest(of_key[k]);
                }
            }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int key = first + 2 * j + (k & 1) + 8 * (k >> 1);
            const bool is_none = none >> k & 1u;
            if (key >= length || is_none) step[k] = 0.f;
            if (key >= length || is_none) lowest[k] = key < length && !which ? NAN : 0.f;
            step[k] *= raise;
            lowest[k] *= raise;
        }
    }
    T* to = opened + which * half + (((size_t)r * blocks + open_block) * gridDim.y + open_head) * open_size * HD +
            (size_t)(unit % per_block) * 16 * HD + s * 16;
#pragma unroll
    for (int k = 0; k < 4; ++k) {        // key 2j + (k & 1) + 8 (k / 2)
        float x[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // keys' words: row 2j + (k & 1), c = e / 2, the byte of the upper half of keys and of odd e; values'
            // words: r = e, the byte of the upper half of keys and of the odd key
            const uint32_t both = which ? words[e] >> (8 * (k >> 1) + 16 * (k & 1))
                                        : words[4 * (k & 1) + e / 2] >> (8 * (k >> 1) + 16 * (e & 1));
            x[e] = fmaf(step[k], (float)(both & 15u), lowest[k]);
            x[e + 8] = fmaf(step[k], (float)(both >> 4 & 15u), lowest[k]);
        }
        T* row = to + (2 * j + (k & 1) + 8 * (k >> 1)) * HD;
        if (sizeof(T) == 2 && largest != nullptr) {
            uint32_t pairs[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const __half2 pair = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
                pairs[e] = *reinterpret_cast<const uint32_t*>(&pair);
            }
            *reinterpret_cast<uint4*>(row) = make_uint4(pairs[0], pairs[1], pairs[2], pairs[3]);
            *reinterpret_cast<uint4*>(row + 8) = make_uint4(pairs[4], pairs[5], pairs[6], pairs[7]);
        } else {
            store_run(row, x);
        }
    }
}

int check_geometry(const char* name, int head_dim, int page_size, int pages, int kv_heads, int table_width,
                   const void* cache) {
    MLXONE_REQUIRE(page_size >= 16 && (page_size & (page_size - 1)) == 0,
                   "%s: pages of 4 bits hold a power of two of tokens, 16 or more, not %d", name, page_size);
    MLXONE_REQUIRE(pages > 0 && table_width > 0 && kv_heads > 0 && kv_heads <= 65535, "%s: bad page geometry", name);
    MLXONE_REQUIRE(((size_t)cache & 15) == 0, "%s: the cache starts at a multiple of 16 bytes", name);
    MLXONE_REQUIRE(head_dim % 32 == 0 && head_dim >= 32 && head_dim <= 128,
                   "%s: a cache of 4 bits takes heads of 32, 64, 96 or 128 values, not %d", name, head_dim);
    return 0;
}

}  // namespace

// Bytes of 16 tokens of one key head, keys and values; 0 for a head size that the format does not have.
MLXONE_API int mlxone_packed_unit_bytes(int head_dim) {
    if (head_dim % 32 != 0 || head_dim < 32 || head_dim > 128) return 0;
    return 2 * (8 * head_dim + 64 * (head_dim % 64 == 0 ? head_dim / 64 : head_dim / 32));
}

// keys, values: rows of kv_heads * head_dim values, `*_stride` values apart.
MLXONE_API int mlxone_pack_key_values(const void* keys, long long key_stride, const void* values,
                                      long long value_stride, const int* positions, const int* token_request,
                                      const int* request_start, const int* block_table, int table_width,
                                      int page_size, int pages, int kv_heads, int head_dim, int tokens,
                                      void* cache, int dtype, int* error_flag, cudaStream_t stream) {
    if (tokens == 0) return 0;
    if (check_geometry("pack_key_values", head_dim, page_size, pages, kv_heads, table_width, cache)) return 1;
    MLXONE_REQUIRE(tokens > 0, "pack_key_values: bad token count");
    const int size = dtype == MLXONE_BF16 ? 2 : 4;
    const int wide = ((size_t)keys & 15) == 0 && ((size_t)values & 15) == 0 && key_stride * size % 16 == 0 &&
                     value_stride * size % 16 == 0;
    const dim3 grid(ceil_div_host(tokens, TOKENS), kv_heads);
    const int page_shift = 31 - __builtin_clz((unsigned)page_size);
#define CALL(HD)                                                                                          \
    if (dtype == MLXONE_BF16)                                                                             \
        launch_kernel(pack_kernel<bf16, HD>, grid, dim3(256), 0, stream, true, (const bf16*)keys,         \
                      key_stride, (const bf16*)values, value_stride, wide, positions, token_request,      \
                      request_start, block_table, table_width, page_shift, pages, kv_heads, tokens,        \
                      (unsigned char*)cache, error_flag);                                                 \
    else                                                                                                  \
        launch_kernel(pack_kernel<float, HD>, grid, dim3(256), 0, stream, true, (const float*)keys,       \
                      key_stride, (const float*)values, value_stride, wide, positions, token_request,     \
                      request_start, block_table, table_width, page_shift, pages, kv_heads, tokens,        \
                      (unsigned char*)cache, error_flag)
    MLXONE_PACKED_DIMS(CALL)
#undef CALL
    MLXONE_LAUNCH_CHECK("pack_key_values");
    return 0;
}
MLXONE_BY_WORDS(mlxone_pack_key_values)

MLXONE_API int mlxone_read_key_values(const void* cache, const int* positions, const int* token_request,
                                      const int* block_table, int table_width, int page_size, int pages,
                                      int kv_heads, int head_dim, int tokens, void* keys, void* values,
                                      int dtype, int* error_flag, cudaStream_t stream) {
    if (tokens == 0) return 0;
    if (check_geometry("read_key_values", head_dim, page_size, pages, kv_heads, table_width, cache)) return 1;
    MLXONE_REQUIRE(tokens > 0, "read_key_values: bad token count");
    const dim3 grid(ceil_div_host(tokens, TOKENS), kv_heads);
    const int page_shift = 31 - __builtin_clz((unsigned)page_size);
#define CALL(HD)                                                                                          \
    if (dtype == MLXONE_BF16)                                                                             \
        launch_kernel(read_kernel<bf16, HD>, grid, dim3(256), 0, stream, true, (const unsigned char*)cache, \
                      positions, token_request, block_table, table_width, page_shift, pages, kv_heads,    \
                      tokens, (bf16*)keys, (bf16*)values, error_flag);                                    \
    else                                                                                                  \
        launch_kernel(read_kernel<float, HD>, grid, dim3(256), 0, stream, true, (const unsigned char*)cache, \
                      positions, token_request, block_table, table_width, page_shift, pages, kv_heads,    \
                      tokens, (float*)keys, (float*)values, error_flag)
    MLXONE_PACKED_DIMS(CALL)
#undef CALL
    MLXONE_LAUNCH_CHECK("read_key_values");
    return 0;
}
MLXONE_BY_WORDS(mlxone_read_key_values)

// Units whose range a block looks for: 256 keys, more where a warp that opens would find more than 128 ranges.
static int units_of_chunk(int blocks, int open_size) {
    return 16 * ceil_div_host((long long)blocks * open_size, 256 * 128);
}

// Floats that mlxone_open_key_values needs as `factors` for half-precision pages.
MLXONE_API long long mlxone_open_factors(int requests, int open_heads, int blocks, int open_size) {
    if (requests <= 0 || open_heads <= 0 || blocks <= 0 || open_size <= 0) return 0;
    return 2LL * requests * open_heads * (1 + ceil_div_host((long long)blocks * open_size, 16 * units_of_chunk(blocks, open_size)));
}

// Requests first_request.. (`requests` of them) and key heads first_head.. (`open_heads` of kv_heads), `blocks`
// pages of `open_size` tokens (a multiple of 16) for each request: opened [2, requests * blocks, open_heads,
// open_size, head_dim], table int32 [requests * blocks + requests + 1]. `window`: as first_visible_key's span; units
// that no token of the step sees by it are zeros (with keep_first > 0, the first positions that stay visible
// behind a window, none are). A key that some token sees and that has no page raises the error flag. factors: null, or (bfloat16) mlxone_open_factors floats: the pages are then
// half-precision, and the first requests * open_heads * 2 of them are what keys and values are to be multiplied by;
// `rows` rows of q (bfloat16, head_dim values) go to `halves` and query_factors [rows] in the same manner.
MLXONE_API int mlxone_open_key_values(const void* cache, const int* block_table, int table_width, int page_size,
                                      int pages, const int* request_start, const int* history, int window,
                                      int keep_first, int first_request, int requests, int kv_heads, int first_head,
                                      int open_heads, int head_dim, int blocks, int open_size, void* opened,
                                      int* table, float* factors, const void* q, long long rows, void* halves,
                                      float* query_factors, int dtype, int* error_flag, cudaStream_t stream) {
    if (requests == 0) return 0;
    if (check_geometry("open_key_values", head_dim, page_size, pages, kv_heads, table_width, cache)) return 1;
    MLXONE_REQUIRE(requests > 0 && requests <= 65535 && first_request >= 0 && blocks > 0 && open_size >= 16 &&
                       open_size % 16 == 0 && first_head >= 0 && open_heads > 0 &&
                       first_head + open_heads <= kv_heads, "open_key_values: bad sizes");
    MLXONE_REQUIRE(factors == nullptr || (dtype == MLXONE_BF16 && requests <= 65535 - 32 && rows >= 0 &&
                                          (((size_t)q | (size_t)halves) & 15) == 0),
                   "open_key_values: half-precision pages take bfloat16 queries that start at a multiple of 16 bytes");
    MLXONE_REQUIRE(((size_t)opened & 15) == 0, "open_key_values: the output starts at a multiple of 16 bytes");
    MLXONE_REQUIRE(keep_first >= 0 && error_flag != nullptr, "open_key_values: bad arguments");
    const int span = keep_first > 0 ? 0 : window;
    const long long half = (long long)requests * blocks * open_heads * open_size * head_dim;
    const int page_shift = 31 - __builtin_clz((unsigned)page_size);
    const int chunk_units = units_of_chunk(blocks, open_size);
    const int chunks = ceil_div_host((long long)blocks * open_size, 16 * chunk_units);
    const unsigned char* held = (const unsigned char*)cache;
    float* largest = nullptr;
    if (factors != nullptr) {
        largest = factors + (size_t)requests * open_heads * 2;
        // layers of the grid for the queries: a row by HD / 8 threads, once around for up to 32 layers
        const long long row_blocks = ceil_div_host(rows, 256 / (head_dim == 96 ? 16 : head_dim / 8));
        const int layers = std::min(ceil_div_host(row_blocks, (long long)chunks * open_heads), 32);
#define CALL(HD)                                                                                          \
    launch_kernel(range_kernel<HD>, dim3(chunks, open_heads, requests + layers), dim3(256), 0, stream, true, \
                  held, block_table, table_width, page_shift, pages, request_start, history, span,        \
                  first_request, requests, first_head, kv_heads, chunk_units, largest, (const bf16*)q,     \
                  rows, (uint4*)halves, query_factors)
        MLXONE_PACKED_DIMS(CALL)
#undef CALL
        MLXONE_LAUNCH_CHECK("open_key_values range");
    }
    // units of a block (8 RUNS = head_dim / 2 threads a unit), whole warps
    const int per = head_dim == 96 ? 4 : 512 / head_dim;
    const dim3 grid(ceil_div_host((long long)blocks * (open_size / 16), per), open_heads, requests);
#define CALL(HD)                                                                                          \
    if (dtype == MLXONE_BF16)                                                                             \
        launch_kernel(open_kernel<bf16, HD>, grid, dim3(per * HD / 2), 0, stream, true, held,             \
                      block_table, table_width, page_shift, pages, request_start, history, span, window,  \
                      keep_first, first_request, first_head, kv_heads, blocks, open_size, half,           \
                      (bf16*)opened, table, (const float*)largest, chunks, factors, error_flag);          \
    else                                                                                                  \
        launch_kernel(open_kernel<float, HD>, grid, dim3(per * HD / 2), 0, stream, true, held,            \
                      block_table, table_width, page_shift, pages, request_start, history, span, window,  \
                      keep_first, first_request, first_head, kv_heads, blocks, open_size, half,           \
                      (float*)opened, table, (const float*)nullptr, chunks, (float*)nullptr, error_flag)
    MLXONE_PACKED_DIMS(CALL)
#undef CALL
    MLXONE_LAUNCH_CHECK("open_key_values");
    return 0;
}
MLXONE_BY_WORDS(mlxone_open_key_values)
