// Beam search: the choice of the best continuations, and the caches brought to the hypotheses that own them next.
//
// Choice. A request has B hypotheses with summed logarithms score_b; candidate (b, v) has score_b + logit_bv -
// log sum_v exp(logit_bv), a hypothesis that has ended one candidate, itself. The B best of a request are
// wanted, best first, ties to the lowest (b, v). Bound by reading the logits once (4 bytes a candidate):
//   beam_parts  a block per (row, part of the vocabulary): the part's maximum and sum of exponentials by a running
//               maximum, and its B best logits. A warp holds its best in its lanes, sorted, and looks at a
//               vector of values only if one of them passes the worst of the B: few do after the first
//               hundreds (about B ln(n / B) of n).
//   beam_choice a block per request: a warp per hypothesis joins the parts (the logarithm in 64 bits), then
//               every candidate counts those ahead of it.
// Within a row logits are compared as they are, between rows sums in 64 bits: no order is lost to rounding. A
// logit that is no number counts as minus infinity; a row whose score or sum of exponentials is not finite
// has no continuation (minus infinity for all of them).
//
// Reordering. In place: hypothesis b takes over what hypothesis parent(b) held, both of the same request. A
// thread owns one place of the state and looks after all hypotheses of the request there: it reads what
// moves, then writes it, so that cycles and several children of one parent need neither scratch nor order.
#include "common.cuh"

namespace {

constexpr int WARPS = 8;
constexpr int MAX_BEAMS = 32;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NOTHING = -1e30f;
constexpr int ERROR_PARENT = 10;       // a parent, slot or page outside its range

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// A value and its place as one number that orders by value, then by the lower place.
__device__ __forceinline__ unsigned long long ranked(float value, int place) {
    const uint32_t bits = __float_as_uint(value);
    const uint32_t order = bits & 0x80000000u ? ~bits : bits | 0x80000000u;
    return (unsigned long long)order << 32 | (uint32_t)~place;
}
__device__ __forceinline__ float value_of(unsigned long long rank) {
    const uint32_t order = (uint32_t)(rank >> 32);
    return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
__device__ __forceinline__ int place_of(unsigned long long rank) { return (int)~(uint32_t)rank; }

// The best `count` of what a warp has met, sorted, one a lane (0: none yet).
struct Best {
    unsigned long long mine = 0, worst = 0;
    __device__ __forceinline__ void offer(unsigned long long rank, int count, int lane) {
        unsigned wanting = __ballot_sync(0xffffffffu, rank > worst);
        while (wanting) {
            const int from = __ffs(wanting) - 1;
            wanting &= wanting - 1;
            const unsigned long long next = __shfl_sync(0xffffffffu, rank, from);
            if (next <= worst) continue;
            const unsigned long long above = __shfl_up_sync(0xffffffffu, mine, 1);
            const int at = __popc(__ballot_sync(0xffffffffu, mine > next));
            mine = lane < at ? mine : lane == at ? next : above;
            worst = __shfl_sync(0xffffffffu, mine, count - 1);
        }
    }
};

// -0 counts as 0 and what is no number as minus infinity
__device__ __forceinline__ float logit_of(float x) { return fmaxf(x, -INFINITY) + 0.f; }

// parts_out [rows, parts, 2]: maximum (of x log2 e) and sum of 2^(x log2 e - maximum); ranks_out [rows, parts, beams]
__global__ void __launch_bounds__(WARPS * 32)
beam_parts_kernel(const float* logits, long long stride, int vocab, int beams, int part_size,
                  const float* scores, const unsigned char* ended,
                  float* parts_out, unsigned long long* ranks_out) {
    __shared__ unsigned long long lists[WARPS][MAX_BEAMS];
    __shared__ float tops[WARPS], sums[WARPS];
    griddep_launch();
    griddep_wait();
    const int row = blockIdx.y, part = blockIdx.x, parts = gridDim.x;
    if ((ended != nullptr && ended[row]) || !isfinite(scores[row])) return;     // nothing of the row is wanted
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* x = logits + (size_t)row * stride;
    const int begin = part * part_size, end = min(begin + part_size, vocab);
    Best best;
    float top = NOTHING, sum = 0.f;
    auto take = [&](const float (&v)[4], int place, int live) {
        const float most = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
        const float scaled = most * LOG2E;
        if (scaled > top) {
            sum *= fast_exp2(top - scaled);
            top = scaled;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += fast_exp2(fmaf(v[i], LOG2E, -top));
        // (equal to the worst still counts here: its place decides)
        if (__any_sync(0xffffffffu, live > 0 && ranked(most, 0) > best.worst)) {
#pragma unroll
            for (int i = 0; i < 4; ++i) best.offer(i < live ? ranked(v[i], place + i) : 0, beams, lane);
        }
    };
    const bool wide = ((size_t)x & 15) == 0 && (begin & 3) == 0;
    if (wide) {
        // four vectors a lane at a time, all asked for before the first is looked at
        constexpr int AHEAD = 4;
        for (int at = begin + warp * AHEAD * 128; at < end; at += WARPS * AHEAD * 128) {
            float v[AHEAD][4];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int place = at + a * 128 + lane * 4;
                if (place + 4 <= end) {
                    const float4 four = __ldcs(reinterpret_cast<const float4*>(x + place));
                    v[a][0] = four.x; v[a][1] = four.y; v[a][2] = four.z; v[a][3] = four.w;
                } else {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[a][i] = place + i < end ? x[place + i] : -INFINITY;
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int place = at + a * 128 + lane * 4;
                if (at + a * 128 >= end) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) v[a][i] = logit_of(v[a][i]);
                take(v[a], place, min(max(end - place, 0), 4));
            }
        }
    } else {
        for (int at = begin + warp * 32; at < end; at += WARPS * 32) {
            const int place = at + lane;
            float v[4] = {place < end ? logit_of(x[place]) : -INFINITY, -INFINITY, -INFINITY, -INFINITY};
            take(v, place, place < end ? 1 : 0);
        }
    }
    // lanes, then warps
    const float warp_top = warp_max(top);
    sum = warp_sum(sum * fast_exp2(top - warp_top));
    if (lane == 0) {
        tops[warp] = warp_top;
        sums[warp] = sum;
    }
    lists[warp][lane] = best.mine;
    __syncthreads();
    if (warp == 0) {
        for (int w = 1; w < WARPS; ++w) best.offer(lane < beams ? lists[w][lane] : 0, beams, lane);
        if (lane < beams) ranks_out[((size_t)row * parts + part) * beams + lane] = best.mine;
        const float all = warp_max(lane < WARPS ? tops[lane] : NOTHING);
        const float total = warp_sum(lane < WARPS ? sums[lane] * fast_exp2(tops[lane] - all) : 0.f);
        if (lane == 0) {
            parts_out[((size_t)row * parts + part) * 2] = all;
            parts_out[((size_t)row * parts + part) * 2 + 1] = total;
        }
    }
}

__global__ void __launch_bounds__(MAX_BEAMS * 32)
beam_choice_kernel(const float* parts_in, const unsigned long long* ranks_in, int parts,
                   int beams, const float* scores, const unsigned char* ended,
                   const int* ends, int end_count, float* scores_out,
                   int* parents_out, int* tokens_out,
                   unsigned char* ended_out) {
    __shared__ double values[MAX_BEAMS * MAX_BEAMS];       // (a NaN: no candidate)
    __shared__ int tokens[MAX_BEAMS * MAX_BEAMS];
    griddep_launch();
    griddep_wait();
    const float* part_sums = settled(parts_in);
    const unsigned long long* part_ranks = settled(ranks_in);
    const int request = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = request * beams + warp;
    const float score = scores[row];
    const bool over = ended != nullptr && ended[row];
    const double minus = -(double)INFINITY;
    double value = (double)NAN;
    int token = lane;
    if (over) {
        if (lane == 0) {
            value = isnan(score) ? minus : (double)score;
            token = ends[0];
        }
    } else {
        double whole = (double)NAN;                        // the logarithm of the row's sum, times log2 e
        Best best;
        if (isfinite(score)) {
            float top = NOTHING;
            for (int i = lane; i < parts; i += 32) top = fmaxf(top, part_sums[((size_t)row * parts + i) * 2]);
            top = warp_max(top);
            float sum = 0.f;
            for (int i = lane; i < parts; i += 32) {
                const float* at = part_sums + ((size_t)row * parts + i) * 2;
                sum += at[1] * fast_exp2(at[0] - top);
            }
            sum = warp_sum(sum);
            whole = (double)top + log2((double)sum);
            const unsigned long long* at = part_ranks + (size_t)row * parts * beams;
            for (int i = 0; i < parts * beams; i += 32)
                best.offer(i + lane < parts * beams ? at[i + lane] : 0, beams, lane);
        }
        if (lane < beams) {
            value = minus;
            if (isfinite(whole)) {
                const float logit = value_of(best.mine);
                token = place_of(best.mine);
                value = (double)score + ((double)logit - whole * 0.6931471805599453094);
            }
        }
    }
    if (lane < beams) {
        values[warp * beams + lane] = value;
        tokens[warp * beams + lane] = token;
    }
    __syncthreads();
    // (a hypothesis' candidates are sorted, so the order of the array is the order of ties)
    for (int i = threadIdx.x; i < beams * beams; i += blockDim.x) {
        const double mine = values[i];
        if (isnan(mine)) continue;
        int ahead = 0;
        for (int k = 0; k < beams * beams; ++k) ahead += values[k] > mine || (values[k] == mine && k < i);
        if (ahead >= beams) continue;
        const int at = request * beams + ahead, parent = i / beams, chosen = tokens[i];
        bool stops = ended != nullptr && ended[request * beams + parent];
        for (int k = 0; k < end_count; ++k) stops = stops || chosen == ends[k];
        scores_out[at] = (float)mine;
        parents_out[at] = parent;
        tokens_out[at] = chosen;
        ended_out[at] = stops ? 1 : 0;
    }
}

// ------------------------------------------------------------------ reordering

// One place of a state for every hypothesis of a request: from[b] < 0: nothing moves.
template <typename V, int MOST>
__device__ __forceinline__ void move_place(unsigned char* base, const long long (&from)[MAX_BEAMS],
                                           const long long (&to)[MAX_BEAMS], int beams, size_t at) {
    V held[MOST];
#pragma unroll
    for (int b = 0; b < MOST; ++b)
        if (b < beams && from[b] >= 0) held[b] = *reinterpret_cast<const V*>(base + from[b] + at);
#pragma unroll
    for (int b = 0; b < MOST; ++b)
        if (b < beams && from[b] >= 0) *reinterpret_cast<V*>(base + to[b] + at) = held[b];
}

// state [entries, slots, bytes]: what hypothesis b's slot holds becomes what its parent's held.
template <typename V, int MOST>
__global__ void __launch_bounds__(256)
reorder_slots_kernel(unsigned char* state, long long slots, long long bytes, const int* slot_of,
                     const int* parents, int beams, int* error_flag) {
    __shared__ long long from[MAX_BEAMS], to[MAX_BEAMS];
    const int request = blockIdx.y;
    if (threadIdx.x < beams) {
        const int b = threadIdx.x, parent = parents[request * beams + b];
        long long source = -1, target = 0;
        if (parent < 0 || parent >= beams) {
            atomicExch(error_flag, ERROR_PARENT);
        } else if (parent != b) {
            source = slot_of[request * beams + parent];
            target = slot_of[request * beams + b];
            if (source < 0 || source >= slots || target < 0 || target >= slots) {
                atomicExch(error_flag, ERROR_PARENT);
                source = -1;
            } else if (source == target) {
                source = -1;
            }
        }
        from[b] = source < 0 ? -1 : source * bytes;
        to[b] = target * bytes;
    }
    __syncthreads();
    unsigned char* base = state + (size_t)blockIdx.z * slots * bytes;
    for (size_t at = ((size_t)blockIdx.x * 256 + threadIdx.x) * sizeof(V); at < (size_t)bytes;
         at += (size_t)gridDim.x * 256 * sizeof(V))
        move_place<V, MOST>(base, from, to, beams, at);
}

// storage [outer, pages, bytes]: the pages of positions starts[request] .. lengths[request] - 1, block by block.
template <typename V, int MOST>
__global__ void __launch_bounds__(256)
reorder_pages_kernel(unsigned char* storage, long long pages, long long bytes, const int* block_table,
                     int table_width, const int* parents, const int* starts,
                     const int* lengths, int page_size, int beams, int* error_flag) {
    __shared__ long long from[MAX_BEAMS], to[MAX_BEAMS];
    const int request = blockIdx.y;
    unsigned char* base = storage + (size_t)blockIdx.z * pages * bytes;
    const int first = max(starts[request], 0) / page_size;
    const int last = min((max(lengths[request], 0) + page_size - 1) / page_size, table_width);
    for (int block = first + blockIdx.x; block < last; block += gridDim.x) {
        __syncthreads();
        if (threadIdx.x < beams) {
            const int b = threadIdx.x, parent = parents[request * beams + b];
            long long source = -1, target = 0;
            if (parent < 0 || parent >= beams) {
                atomicExch(error_flag, ERROR_PARENT);
            } else if (parent != b) {
                source = block_table[(size_t)(request * beams + parent) * table_width + block];
                target = block_table[(size_t)(request * beams + b) * table_width + block];
                // (a page that was given back, on either side: nothing to move)
                if (source >= pages || target >= pages) atomicExch(error_flag, ERROR_PARENT);
                if (source < 0 || target < 0 || source >= pages || target >= pages || source == target) source = -1;
            }
            from[b] = source < 0 ? -1 : source * bytes;
            to[b] = target * bytes;
        }
        __syncthreads();
        for (size_t at = threadIdx.x * sizeof(V); at < (size_t)bytes; at += 256 * sizeof(V))
            move_place<V, MOST>(base, from, to, beams, at);
    }
}

}  // namespace

// Scratch of mlxone_beam_select: into how many parts a row's vocabulary is cut.
MLXONE_API int mlxone_beam_parts(int rows, int vocab) {
    if (rows <= 0 || vocab <= 0) return 1;
    const int wanted = ceil_div_host(148 * 4, rows), most = ceil_div_host(vocab, 1024);
    const int parts = wanted < most ? wanted : most;
    return parts < 1 ? 1 : parts > 64 ? 64 : parts;
}

// logits float32 [requests * beams, vocab], rows `stride` values apart; scores float32 [requests, beams]; ended bytes
// [requests, beams] or null; ends int32 [end_count] (at least one with `ended`). partial: requests * beams * parts * 2
// floats; ranks: requests * beams * parts * beams 64-bit numbers.
MLXONE_API int mlxone_beam_select(const float* logits, long long stride, int requests, int beams, int vocab,
                                  const float* scores, const unsigned char* ended, const int* ends, int end_count,
                                  int parts, float* partial, unsigned long long* ranks, float* scores_out,
                                  int* parents_out, int* tokens_out, unsigned char* ended_out,
                                  cudaStream_t stream) {
    if (requests == 0) return 0;
    MLXONE_REQUIRE(requests > 0 && beams >= 1 && beams <= MAX_BEAMS, "beam_select: 1 to %d hypotheses, not %d",
                   MAX_BEAMS, beams);
    MLXONE_REQUIRE(vocab >= beams, "beam_select: %d tokens are fewer than %d hypotheses", vocab, beams);
    MLXONE_REQUIRE((long long)requests * beams <= 65535, "beam_select: too many rows");
    MLXONE_REQUIRE(parts >= 1 && parts <= 64 && end_count >= 0 && (ended == nullptr || end_count > 0),
                   "beam_select: bad sizes");
    const int part_size = ceil_div_host(ceil_div_host(vocab, parts), 4) * 4;
    launch_kernel(beam_parts_kernel, dim3(parts, requests * beams), dim3(WARPS * 32), 0, stream, true, logits, stride,
                  vocab, beams, part_size, scores, ended, partial, ranks);
    MLXONE_LAUNCH_CHECK("beam_parts");
    launch_kernel(beam_choice_kernel, dim3(requests), dim3(beams * 32), 0, stream, true, (const float*)partial,
                  (const unsigned long long*)ranks, parts, beams, scores, ended, ends, end_count, scores_out,
                  parents_out, tokens_out, ended_out);
    MLXONE_LAUNCH_CHECK("beam_choice");
    return 0;
}

#define MLXONE_MOVE(KERNEL, V, ...)                                                                    \
    do {                                                                                               \
        if (beams <= 4) KERNEL<V, 4><<<grid, 256, 0, stream>>>(__VA_ARGS__);                           \
        else if (beams <= 8) KERNEL<V, 8><<<grid, 256, 0, stream>>>(__VA_ARGS__);                      \
        else if (beams <= 16) KERNEL<V, 16><<<grid, 256, 0, stream>>>(__VA_ARGS__);                    \
        else KERNEL<V, 32><<<grid, 256, 0, stream>>>(__VA_ARGS__);                                     \
    } while (0)
// (the widest pieces that address and size allow)
#define MLXONE_MOVE_ANY(KERNEL, ADDRESS, BYTES, ...)                                                   \
    do {                                                                                               \
        if ((((size_t)(ADDRESS) | (size_t)(BYTES)) & 15) == 0) MLXONE_MOVE(KERNEL, uint4, __VA_ARGS__); \
        else if ((((size_t)(ADDRESS) | (size_t)(BYTES)) & 3) == 0) MLXONE_MOVE(KERNEL, uint32_t, __VA_ARGS__); \
        else MLXONE_MOVE(KERNEL, unsigned char, __VA_ARGS__);                                          \
    } while (0)

// state [entries, slots, bytes] in place; slot_of int32 [requests, beams], every hypothesis a slot of its own;
// parents int32 [requests, beams] within the request.
MLXONE_API int mlxone_reorder_slots(void* state, long long entries, long long slots, long long bytes,
                                    const int* slot_of, const int* parents, int requests, int beams, int* error_flag,
                                    cudaStream_t stream) {
    if (requests == 0 || entries == 0 || bytes == 0) return 0;
    MLXONE_REQUIRE(requests > 0 && requests <= 65535 && beams >= 1 && beams <= MAX_BEAMS,
                   "reorder_slots: 1 to %d hypotheses, not %d", MAX_BEAMS, beams);
    MLXONE_REQUIRE(entries > 0 && entries <= 65535 && slots > 0 && bytes > 0, "reorder_slots: bad sizes");
    const long long pieces = (bytes / 16 + 255) / 256, room = (148LL * 16 + entries * requests - 1) / (entries * requests);
    const dim3 grid((unsigned)(pieces < 1 ? 1 : pieces < room ? pieces : room), requests, (unsigned)entries);
    MLXONE_MOVE_ANY(reorder_slots_kernel, state, bytes, (unsigned char*)state, slots, bytes, slot_of, parents, beams,
                    error_flag);
    MLXONE_LAUNCH_CHECK("reorder_slots");
    return 0;
}

// storage [outer, pages, bytes] in place; block_table int32 [requests * beams, table_width], -1 where there is no page;
// pages of hypotheses of one request that differ in content differ in number, and no page that moves has two owners.
MLXONE_API int mlxone_reorder_pages(void* storage, long long outer, long long pages, long long bytes,
                                    const int* block_table, int table_width, const int* parents, const int* starts,
                                    const int* lengths, int page_size, int requests, int beams, int* error_flag,
                                    cudaStream_t stream) {
    if (requests == 0 || outer == 0 || bytes == 0) return 0;
    MLXONE_REQUIRE(requests > 0 && requests <= 65535 && beams >= 1 && beams <= MAX_BEAMS,
                   "reorder_pages: 1 to %d hypotheses, not %d", MAX_BEAMS, beams);
    MLXONE_REQUIRE(outer > 0 && outer <= 65535 && pages > 0 && bytes > 0 && table_width > 0 && page_size > 0,
                   "reorder_pages: bad sizes");
    const long long room = (148LL * 8 + outer * requests - 1) / (outer * requests);
    const dim3 grid((unsigned)(table_width < room ? table_width : room), requests, (unsigned)outer);
    MLXONE_MOVE_ANY(reorder_pages_kernel, storage, bytes, (unsigned char*)storage, pages, bytes, block_table,
                    table_width, parents, starts, lengths, page_size, beams, error_flag);
    MLXONE_LAUNCH_CHECK("reorder_pages");
    return 0;
}
