// Beam search: the choice of the best continuations, and the caches brought to the hypotheses that own them next.
//
// Choice. A request has B hypotheses with summed logarithms score_b; candidate (b, v) has score_b + logit_bv -
// log sum_v exp(logit_bv), a hypothesis that has ended one candidate, itself. The B best of a request are
// wanted, best first, ties to the lowest (b, v). Bound by reading the logits once (4 bytes a candidate):
//   beam_parts  a block per (row, part of the vocabulary), the part in its registers, 4 to 32 values a thread: the
//               sum of exponentials against the warp's maximum, and the part's B best. The B-th largest of a
//               warp's 32 lane maxima bounds its B best from below; the few values above it go to a list in
//               shared memory, where each counts those ahead of it. A list that runs over (ties) is made again
//               by insertion, value after value.
//   beam_choice a block per request: a warp per hypothesis takes the best of its parts' sorted lists B times (the
//               logarithm in 64 bits), then every candidate counts those ahead of it.
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

// what is no number counts as minus infinity
__device__ __forceinline__ float logit_of(float x) { return fmaxf(x, -INFINITY); }

constexpr int LISTED = 1536;           // candidates of a block's list (32 hypotheses leave about 900)
constexpr int MOST_PARTS = 256;

// parts_out [rows, parts, 2]: maximum (of x log2 e) and sum of 2^(x log2 e - maximum); ranks_out [rows, parts, beams].
// A part is 1,024 V values: V vectors of four a thread.
template <int V>
__global__ void __launch_bounds__(WARPS * 32)
beam_parts_kernel(const float* logits, long long stride, int vocab, int beams, const float* scores,
                  const unsigned char* ended, float* parts_out, unsigned long long* ranks_out) {
    __shared__ unsigned long long list[LISTED];
    __shared__ float tops[WARPS], sums[WARPS];
    __shared__ int listed;
    griddep_launch();
    griddep_wait();
    const int row = blockIdx.y, part = blockIdx.x, parts = gridDim.x;
    if ((ended != nullptr && ended[row]) || !isfinite(scores[row])) return;     // nothing of the row is wanted
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* x = logits + (size_t)row * stride;
    const int begin = part * (V * 1024), end = min(begin + V * 1024, vocab);
    const int first = begin + (int)threadIdx.x * 4;              // of vector v: first + 1024 v
    float value[V][4];
    if (((size_t)x & 15) == 0) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int place = first + v * 1024;
            if (place + 4 <= end) {
                const float4 four = __ldcs(reinterpret_cast<const float4*>(x + place));
                value[v][0] = four.x; value[v][1] = four.y; value[v][2] = four.z; value[v][3] = four.w;
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) value[v][i] = place + i < end ? x[place + i] : -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int place = first + v * 1024 + i;
                value[v][i] = place < end ? x[place] : -INFINITY;
            }
    }
    if (threadIdx.x == 0) listed = 0;
    float most = -INFINITY;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            value[v][i] = logit_of(value[v][i]);
            most = fmaxf(most, value[v][i]);
        }
    // the maximum of the warp, and the B-th largest of its lanes' maxima: no lane's value below that is wanted
    const uint32_t order = (uint32_t)(ranked(most, 0) >> 32);
    uint32_t left = order, bound = 0, top_order = 0;
    for (int k = 0; k < beams; ++k) {
        bound = __reduce_max_sync(0xffffffffu, left);
        if (k == 0) top_order = bound;
        // (one lane of those that have it leaves)
        const unsigned have = __ballot_sync(0xffffffffu, left == bound);
        if (lane == __ffs(have) - 1) left = 0;
    }
    const float top = fmaxf(value_of((unsigned long long)top_order << 32) * LOG2E, NOTHING);
    const float least = value_of((unsigned long long)bound << 32);
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += fast_exp2(fmaf(value[v][i], LOG2E, -top));
    sum = warp_sum(sum);
    if (lane == 0) {
        tops[warp] = top;
        sums[warp] = sum;
    }
    __syncthreads();
    if (most >= least) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int place = first + v * 1024 + i;
                if (value[v][i] >= least && place < end) {
                    const int at = atomicAdd(&listed, 1);
                    if (at < LISTED) list[at] = ranked(value[v][i] + 0.f, place);      // (-0 is 0)
                }
            }
    }
    __syncthreads();
    const int count = listed;
    unsigned long long* out = ranks_out + ((size_t)row * parts + part) * beams;
    if (count <= LISTED) {
        // (at least B unless the part is shorter; all different, so every rank has one owner)
        for (int i = threadIdx.x; i < count; i += WARPS * 32) {
            const unsigned long long mine = list[i];
            int ahead = 0;
            for (int k = 0; k < count; ++k) ahead += list[k] > mine;
            if (ahead < beams) out[ahead] = mine;
        }
        if ((int)threadIdx.x >= count && (int)threadIdx.x < beams) out[threadIdx.x] = 0;
    } else {
        Best best;
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int place = first + v * 1024 + i;
                best.offer(place < end ? ranked(value[v][i] + 0.f, place) : 0, beams, lane);
            }
        __syncthreads();                                         // (the list's room is the warps' now)
        list[warp * MAX_BEAMS + lane] = best.mine;
        __syncthreads();
        if (warp == 0) {
            for (int w = 1; w < WARPS; ++w) best.offer(lane < beams ? list[w * MAX_BEAMS + lane] : 0, beams, lane);
            if (lane < beams) out[lane] = best.mine;
        }
    }
    if (warp == 0) {
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
        unsigned long long best = 0;
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
            // the parts' lists are sorted: a lane looks after every 32nd part's, its first and the one after
            const unsigned long long* at = part_ranks + (size_t)row * parts * beams;
            constexpr int MINE = MOST_PARTS / 32;
            unsigned long long head[MINE], next[MINE];
            int taken[MINE];
#pragma unroll
            for (int i = 0; i < MINE; ++i) {
                const bool there = lane + 32 * i < parts;
                head[i] = there ? at[(size_t)(lane + 32 * i) * beams] : 0;
                next[i] = there && beams > 1 ? at[(size_t)(lane + 32 * i) * beams + 1] : 0;
                taken[i] = 2;
            }
            for (int k = 0; k < beams; ++k) {
                unsigned long long mine = head[0];
#pragma unroll
                for (int i = 1; i < MINE; ++i) mine = head[i] > mine ? head[i] : mine;
                const uint32_t high = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32));
                const uint32_t low = __reduce_max_sync(0xffffffffu, (uint32_t)(mine >> 32) == high ? (uint32_t)mine : 0u);
                const unsigned long long found = (unsigned long long)high << 32 | low;
                if (lane == k) best = found;
#pragma unroll
                for (int i = 0; i < MINE; ++i)
                    if (head[i] == found && found != 0) {
                        head[i] = next[i];
                        next[i] = taken[i] < beams ? at[(size_t)(lane + 32 * i) * beams + taken[i]] : 0;
                        ++taken[i];
                    }
            }
        }
        if (lane < beams) {
            value = minus;
            if (isfinite(whole)) {
                const float logit = value_of(best);
                token = place_of(best);
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

// Vectors of four that a thread takes: as many as leave two blocks an SM and more.
static int beam_vectors(int rows, int vocab) {
    int v = 8;
    while (v > 1 && (long long)rows * ceil_div_host(vocab, 1024 * v) < 2 * 148) v >>= 1;
    while (v < 8 && ceil_div_host(vocab, 1024 * v) > 64) v <<= 1;
    return v;
}

// Scratch of mlxone_beam_select: into how many parts a row's vocabulary is cut.
MLXONE_API int mlxone_beam_parts(int rows, int vocab) {
    if (rows <= 0 || vocab <= 0) return 1;
    return ceil_div_host(vocab, 1024 * beam_vectors(rows, vocab));
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
    MLXONE_REQUIRE(parts == mlxone_beam_parts(requests * beams, vocab) && end_count >= 0 &&
                       (ended == nullptr || end_count > 0), "beam_select: bad sizes");
    MLXONE_REQUIRE(parts <= MOST_PARTS, "beam_select: a vocabulary of %d tokens is too large", vocab);
#define CALL(V)                                                                                               \
    launch_kernel(beam_parts_kernel<V>, dim3(parts, requests * beams), dim3(WARPS * 32), 0, stream, true,     \
                  logits, stride, vocab, beams, scores, ended, partial, ranks)
    switch (beam_vectors(requests * beams, vocab)) {
        case 1: CALL(1); break;
        case 2: CALL(2); break;
        case 4: CALL(4); break;
        default: CALL(8); break;
    }
#undef CALL
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
