// Beam search: the choice of the best continuations, and the caches brought to the hypotheses that own them next.
//
// Choice. A request has B hypotheses with summed logarithms score_b; candidate (b, v) has score_b + logit_bv -
// log sum_v exp(logit_bv), a hypothesis that has ended one candidate, itself. The B best of a request are
// wanted, best first, ties to the lowest (b, v). Bound by reading the logits once (4 bytes a candidate):
//   beam_sums   reads them: a thread takes 32 (eight vectors, all asked for at once) and leaves their maximum, a block
//               of 8,192 the sum of their exponentials. About 5 instructions a value, no exchange but at the end.
//   beam_choice a block per row. With the ceil(B / 8) largest of what each of its 8 warps sees of the row's thread
//               maxima the B-th largest of those bounds the B best from below (B threads have a value of that
//               size at least), so only the values of the few threads whose maximum reaches it are read again;
//               those that reach it are ordered by counting who is ahead. Where they are many the row is walked
//               value by value instead: with ties, and with small vocabularies, for the maxima of p parts of 8,192
//               lie with 2 p of the 8 warps, whose offers are too few for a bound in one part from three hypotheses
//               on, in two from five, in three with 7, 8, 13 to 16 and 19 or more. A request's candidates are ordered in the same way by the first block
//               of its cluster, or (more than eight hypotheses) by its last block to arrive: a counter in the call's
//               own scratch, set to zero by the kernel before.
// Within a row logits are compared as they are, between rows sums in 64 bits: no order is lost to rounding. A
// logit that is no number counts as minus infinity; a row whose score or sum of exponentials is not finite
// has no continuation (minus infinity for all of them).
//
// Measured, us on the GPU: one request of four hypotheses over 65,536 logits 7.7 (two launches; the choice waits
// for the maxima, the chosen logits and its neighbours in turn), 32 of eight (60 MB are wanted) 22.0: 2.7 TB/s, 9.2 at
// the copy rate. About half of that is the sums' reading, half the choice, which waits rather than works. Rows
// that are walked cost more than longer ones with a bound: four hypotheses over 1,000 / 8,192 / 16,384 tokens 19.2 / 22.4 /
// 6.9, eight over 16,384 / 24,576 / 32,000 28.8 / 36.5 / 8.9, 32 requests of eight 57.8 / 72.1 / 15.0. Sorted
// lists by insertion instead of the bound took 47, a part's best kept in registers 31, lists in shared memory 35.
//
// Reordering. In place: hypothesis b takes over what hypothesis parent(b) held, both of the same request. A
// thread owns one place of the state and looks after all hypotheses of the request there: it reads what
// moves, then writes it, so that cycles and several children of one parent need neither scratch nor order.
// Bound by the bytes: matrices of 1 MB (two requests of four, 8 layers, 50 MB read and written) in 11.9 us, 4.2 TB/s;
// pages of 4 bits (eight requests of four, 300 tokens each, 33 MB) in 7.4, 4.5 TB/s.
#include <cooperative_groups.h>

#include "by_words.cuh"
#include "common.cuh"

namespace cg = cooperative_groups;

namespace {

constexpr int WARPS = 8;
constexpr int MAX_BEAMS = 32;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float NOTHING = -3.402823466e38f;      // a maximum of no logits: the lowest number, so that differences stay numbers
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

constexpr int PART = 8192;             // logits of a block, 32 a thread
constexpr int CLUSTER_BEAMS = 8;
constexpr int CHOSEN = 256, LISTED = 512;       // of a row: threads and values that reach the bound

// Where value e (0..31) of thread t of a row lies.
__device__ __forceinline__ int place_in_row(int t, int e) {
    return (t >> 8) * PART + (e >> 2) * 1024 + (t & 255) * 4 + (e & 3);
}

// maxima [rows, parts * 256]; sums [rows, parts, 2]: maximum and sum of exp(x - maximum). The maximum is a logit as it
// is, so that a token that is certain has the logarithm 0.
__global__ void __launch_bounds__(WARPS * 32)
beam_sums_kernel(const float* logits, long long stride, int vocab, int beams, const float* scores,
                 const unsigned char* ended, float* maxima, float* sums_out, int* arrived) {
    __shared__ float tops[WARPS], sums[WARPS];
    griddep_launch();
    griddep_wait();
    const int row = blockIdx.y, part = blockIdx.x, parts = gridDim.x;
    if (part == 0 && row % beams == 0 && threadIdx.x == 0) arrived[row / beams] = 0;
    if ((ended != nullptr && ended[row]) || !isfinite(scores[row])) return;     // nothing of the row is wanted
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float* x = logits + (size_t)row * stride + (size_t)part * PART;
    const int left = vocab - part * PART, first = (int)threadIdx.x * 4;
    float value[8][4];
    if (left >= PART && ((size_t)x & 15) == 0) {
#pragma unroll
        for (int v = 0; v < 8; ++v) {
            const float4 four = __ldcs(reinterpret_cast<const float4*>(x + first + v * 1024));
            value[v][0] = four.x; value[v][1] = four.y; value[v][2] = four.z; value[v][3] = four.w;
        }
    } else {
#pragma unroll
        for (int v = 0; v < 8; ++v)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int place = first + v * 1024 + i;
                value[v][i] = place < left ? x[place] : -INFINITY;
            }
    }
    float most = -INFINITY;
#pragma unroll
    for (int v = 0; v < 8; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            value[v][i] = logit_of(value[v][i]);
            most = fmaxf(most, value[v][i]);
        }
    const float top = fmaxf(most, NOTHING);
    float sum[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < 8; ++v)
#pragma unroll
        for (int i = 0; i < 4; ++i) sum[i & 1] += fast_exp2((value[v][i] - top) * LOG2E);
    maxima[((size_t)row * parts + part) * (WARPS * 32) + threadIdx.x] = most;
    const float warp_top = warp_max(top);
    const float warp_sum_ = warp_sum((sum[0] + sum[1]) * fast_exp2((top - warp_top) * LOG2E));
    if (lane == 0) {
        tops[warp] = warp_top;
        sums[warp] = warp_sum_;
    }
    __syncthreads();
    if (warp == 0) {
        const float all = warp_max(lane < WARPS ? tops[lane] : NOTHING);
        const float total = warp_sum(lane < WARPS ? sums[lane] * fast_exp2((tops[lane] - all) * LOG2E) : 0.f);
        if (lane == 0) {
            sums_out[((size_t)row * parts + part) * 2] = all;
            sums_out[((size_t)row * parts + part) * 2 + 1] = total;
        }
    }
}

// A number that orders as the value does; 0 for none.
__device__ __forceinline__ unsigned long long ordered(double value) {
    const unsigned long long bits = (unsigned long long)__double_as_longlong(value + 0.0);
    return bits >> 63 ? ~bits : bits | 1ull << 63;
}
__device__ __forceinline__ double of_order(unsigned long long order) {
    return __longlong_as_double((long long)(order >> 63 ? order & ~(1ull << 63) : ~order));
}

// CLUSTER: a request's blocks are a cluster and hand their candidates over in shared memory, where the first one
// orders them. Otherwise: keys, tokens [rows, beams], the rows' candidates, best first, as the last block of a
// request finds them.
template <bool CLUSTER>
__global__ void __launch_bounds__(WARPS * 32)
beam_choice_kernel(const float* logits, long long stride, int vocab, const float* maxima_in, const float* sums_in,
                   int parts, int beams, const float* scores, const unsigned char* ended, const int* ends,
                   int end_count, unsigned long long* keys, int* tokens, int* arrived, float* scores_out,
                   int* parents_out, int* tokens_out, unsigned char* ended_out) {
    __shared__ unsigned long long own_keys[CLUSTER ? CLUSTER_BEAMS : 1];
    __shared__ int own_tokens[CLUSTER ? CLUSTER_BEAMS : 1];
    __shared__ unsigned long long list[LISTED];
    __shared__ unsigned long long sorted[MAX_BEAMS];
    __shared__ int chosen[CHOSEN];
    __shared__ uint32_t bounds[MAX_BEAMS];                       // as ranked() orders
    __shared__ double log_of_sum;                                // (the logarithm of the row's sum, less its maximum)
    __shared__ float top_of_row;
    __shared__ int chosen_count, listed, is_last;
    griddep_launch();
    griddep_wait();
    const int row = blockIdx.x, request = row / beams;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float score = scores[row];
    const bool over = ended != nullptr && ended[row];
    // (asked for beside the score; of a row that is not wanted, whatever lies there, looked at no further)
    const float* maxima = settled(maxima_in) + (size_t)row * parts * (WARPS * 32);
    const int threads = parts * WARPS * 32;
    float most = -INFINITY;
#pragma unroll 4
    for (int i = threadIdx.x * 4; i < threads; i += WARPS * 128) {
        const float4 four = *reinterpret_cast<const float4*>(maxima + i);
        most = fmaxf(fmaxf(most, fmaxf(four.x, four.y)), fmaxf(four.z, four.w));
    }
    const double minus = -(double)INFINITY;
    unsigned long long key = 0;                                  // thread k < beams: the row's k-th candidate
    int token = threadIdx.x;
    if (over) {
        if (threadIdx.x == 0) {
            key = ordered(isnan(score) ? minus : (double)score);
            token = ends[0];
        }
    } else if (!isfinite(score)) {
        if ((int)threadIdx.x < beams) key = ordered(minus);
    } else {
        const float* x = logits + (size_t)row * stride;
        if (threadIdx.x == 0) chosen_count = listed = 0;
        if (warp == WARPS - 1) {
            const float* part_sums = settled(sums_in) + (size_t)row * parts * 2;
            float top = NOTHING, sum = 0.f;
            for (int i = lane; i < parts; i += 32) top = fmaxf(top, part_sums[i * 2]);
            top = warp_max(top);
            for (int i = lane; i < parts; i += 32) sum += part_sums[i * 2 + 1] * fast_exp2((part_sums[i * 2] - top) * LOG2E);
            sum = warp_sum(sum);
            // (the logarithm of what is left of the sum without its power of two, in 0..1, is off by 2^-24)
            int power = 0;
            const float rest = frexpf(sum, &power);
            if (lane == 0) {
                top_of_row = top;
                log_of_sum = sum > 0.f ? ((double)(power - 1) + (double)log2f(2.f * rest)) * 0.6931471805599453094
                                       : (double)NAN;
            }
        }
        // the largest maxima that each warp sees, and what they bound
        const int each = (beams + WARPS - 1) / WARPS, offered = each * WARPS;
        uint32_t left = (uint32_t)(ranked(most + 0.f, 0) >> 32);              // (-0 is 0)
        for (int k = 0; k < each; ++k) {
            const uint32_t largest = __reduce_max_sync(0xffffffffu, left);
            if (lane == 0) bounds[warp * each + k] = largest;
            // (one lane of those that have it leaves)
            const unsigned have = __ballot_sync(0xffffffffu, left == largest);
            if (lane == __ffs((int)have) - 1) left = 0;
        }
        __syncthreads();
        const double below = log_of_sum;
        const float top = top_of_row;
        const uint32_t mine = lane < offered ? bounds[lane] : 0u;
        int ahead = 0;
        for (int k = 0; k < offered; ++k) ahead += bounds[k] > mine || (bounds[k] == mine && k < lane);
        const unsigned last = __ballot_sync(0xffffffffu, lane < offered && ahead == beams - 1);
        const float least = value_of((unsigned long long)__shfl_sync(0xffffffffu, mine, __ffs((int)last) - 1) << 32);
        if (most >= least) {
            for (int i = threadIdx.x * 4; i < threads; i += WARPS * 128) {
                const float4 four = *reinterpret_cast<const float4*>(maxima + i);
                const float of[4] = {four.x, four.y, four.z, four.w};
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (of[k] >= least) {
                        const int at = atomicAdd(&chosen_count, 1);
                        if (at < CHOSEN) chosen[at] = i + k;
                    }
            }
        }
        __syncthreads();
        const int chosen_here = chosen_count;
        bool few = chosen_here <= CHOSEN;
        if (few) {
            // (a warp a thread's values, a lane a value)
#pragma unroll 4
            for (int i = warp; i < chosen_here; i += WARPS) {
                const int place = place_in_row(chosen[i], lane);
                const float logit = place < vocab ? logit_of(x[place]) : -INFINITY;
                if (place < vocab && logit >= least) {
                    const int at = atomicAdd(&listed, 1);
                    if (at < LISTED) list[at] = ranked(logit + 0.f, place);
                }
            }
            __syncthreads();
            few = listed <= LISTED;
        }
        if (few) {
            // (all different, so every rank has one owner; at least B of them)
            const int count = listed;
            for (int i = threadIdx.x; i < count; i += WARPS * 32) {
                const unsigned long long rank = list[i];
                int better = 0;
#pragma unroll 8
                for (int k = 0; k < count; ++k) better += list[k] > rank;
                if (better < beams) sorted[better] = rank;
            }
        } else {
            // ties, a small vocabulary, or hardly a logit above minus infinity: eight sorted lists, then one
            __syncthreads();
            Best best;
            for (int from = 0; from < vocab; from += WARPS * 32) {
                const int place = from + threadIdx.x;
                best.offer(place < vocab ? ranked(logit_of(x[place]) + 0.f, place) : 0, beams, lane);
            }
            list[warp * MAX_BEAMS + lane] = best.mine;
            __syncthreads();
            if (warp == 0) {
                for (int w = 1; w < WARPS; ++w) best.offer(lane < beams ? list[w * MAX_BEAMS + lane] : 0, beams, lane);
                if (lane < beams) sorted[lane] = best.mine;
            }
        }
        __syncthreads();
        if ((int)threadIdx.x < beams) {
            key = ordered(minus);
            if (isfinite(below)) {
                const unsigned long long best = sorted[threadIdx.x];
                token = place_of(best);
                key = ordered((double)score + ((double)value_of(best) - (double)top - below));
            }
        }
    }
    if constexpr (CLUSTER) {
        if ((int)threadIdx.x < beams) {
            own_keys[threadIdx.x] = key;
            own_tokens[threadIdx.x] = token;
        }
        cg::cluster_group cluster = cg::this_cluster();
        cluster.sync();
        const int place = threadIdx.x, of = place / beams, first = request * beams;
        unsigned long long own = 0;
        bool stops = false;
        if (cluster.block_rank() == 0 && place < beams * beams) {
            own = cluster.map_shared_rank(own_keys, of)[place % beams];
            token = cluster.map_shared_rank(own_tokens, of)[place % beams];
            stops = ended != nullptr && ended[first + of];
            for (int k = 0; k < end_count; ++k) stops = stops || token == ends[k];
            list[place] = own;
        }
        cluster.sync();                          // (a block's shared memory is read no more: it may leave)
        if (cluster.block_rank() != 0 || place >= beams * beams || own == 0) return;
        // (a row's candidates are sorted, so the order of the list is the order of ties)
        int ahead = 0;
#pragma unroll 8
        for (int k = 0; k < beams * beams; ++k) ahead += list[k] > own || (list[k] == own && k < place);
        if (ahead >= beams) return;
        scores_out[first + ahead] = (float)of_order(own);
        parents_out[first + ahead] = of;
        tokens_out[first + ahead] = token;
        ended_out[first + ahead] = stops ? 1 : 0;
        return;
    }
    if ((int)threadIdx.x < beams) {
        keys[(size_t)row * beams + threadIdx.x] = key;
        tokens[(size_t)row * beams + threadIdx.x] = token;
        __threadfence();
    }
    __syncthreads();
    if (threadIdx.x == 0) is_last = atomicAdd(arrived + request, 1) == beams - 1;
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    // (a row's candidates are sorted, so the order of the array is the order of ties)
    const int among = beams * beams, held = request * beams;
    const unsigned long long* all = settled(keys) + (size_t)held * beams;
    for (int i = threadIdx.x; i < among && i < LISTED; i += WARPS * 32) list[i] = __ldcg(all + i);
    // (thread i's first candidate's token and whether its hypothesis had ended, asked for beside the list)
    int taken = (int)threadIdx.x < among ? __ldcg(tokens + (size_t)held * beams + threadIdx.x) : 0;
    bool stops = ended != nullptr && (int)threadIdx.x < among && ended[held + threadIdx.x / beams];
    const int first_end = end_count > 0 ? ends[0] : -1;
    __syncthreads();
    for (int i = threadIdx.x; i < among; i += WARPS * 32) {
        const unsigned long long own = i < LISTED ? list[i] : __ldcg(all + i);
        int ahead = own == 0 ? beams : 0;
#pragma unroll 8
        for (int k = 0; k < min(among, LISTED); ++k) ahead += list[k] > own || (list[k] == own && k < i);
        for (int k = LISTED; k < among; ++k) {
            const unsigned long long other = __ldcg(all + k);
            ahead += other > own || (other == own && k < i);
        }
        if (ahead >= beams) continue;
        const int at = held + ahead, parent = i / beams;
        if (i >= WARPS * 32) {
            taken = __ldcg(tokens + (size_t)held * beams + i);
            stops = ended != nullptr && ended[held + parent];
        }
        stops = stops || (end_count > 0 && taken == first_end);
        for (int k = 1; k < end_count; ++k) stops = stops || taken == ends[k];
        scores_out[at] = (float)of_order(own);
        parents_out[at] = parent;
        tokens_out[at] = taken;
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

static int beam_part_count(int vocab) { return ceil_div_host(vocab, PART); }

// Bytes of scratch that mlxone_beam_select needs: thread maxima, sums, candidates, counters.
MLXONE_API long long mlxone_beam_scratch(int requests, int beams, int vocab) {
    if (requests <= 0 || beams <= 0 || vocab <= 0) return 0;
    const long long rows = (long long)requests * beams;
    return rows * beam_part_count(vocab) * (WARPS * 32 + 2) * 4 + rows * beams * 12 + requests * 4LL;
}

// logits float32 [requests * beams, vocab], rows `stride` values apart; scores float32 [requests, beams]; ended bytes
// [requests, beams] or null; ends int32 [end_count] (at least one with `ended`). scratch: mlxone_beam_scratch bytes
// of this call's own, at a multiple of 16.
MLXONE_API int mlxone_beam_select(const float* logits, long long stride, int requests, int beams, int vocab,
                                  const float* scores, const unsigned char* ended, const int* ends, int end_count,
                                  void* scratch, float* scores_out, int* parents_out, int* tokens_out,
                                  unsigned char* ended_out, cudaStream_t stream) {
    if (requests == 0) return 0;
    MLXONE_REQUIRE(requests > 0 && beams >= 1 && beams <= MAX_BEAMS, "beam_select: 1 to %d hypotheses, not %d",
                   MAX_BEAMS, beams);
    MLXONE_REQUIRE(vocab >= beams && vocab <= 1 << 30, "beam_select: %d tokens for %d hypotheses", vocab, beams);
    MLXONE_REQUIRE((long long)requests * beams <= 65535, "beam_select: too many rows");
    MLXONE_REQUIRE(end_count >= 0 && (ended == nullptr || end_count > 0) && ((size_t)scratch & 15) == 0,
                   "beam_select: bad sizes");
    const int rows = requests * beams, parts = beam_part_count(vocab);
    float* maxima = static_cast<float*>(scratch);
    float* sums = maxima + (size_t)rows * parts * (WARPS * 32);
    unsigned long long* keys = reinterpret_cast<unsigned long long*>(sums + (size_t)rows * parts * 2);
    int* tokens = reinterpret_cast<int*>(keys + (size_t)rows * beams);
    int* arrived = tokens + (size_t)rows * beams;
    launch_kernel(beam_sums_kernel, dim3(parts, rows), dim3(WARPS * 32), 0, stream, true, logits, stride, vocab, beams,
                  scores, ended, maxima, sums, arrived);
    MLXONE_LAUNCH_CHECK("beam_sums");
    // Up to eight hypotheses (a cluster that every GPU places): handed over in shared memory. Us for the whole call
    // in clusters / by the last block to arrive: one request of four 7.7 / 8.7, 32 of eight 22.0 / 23.0.
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(rows);
    config.blockDim = dim3(WARPS * 32);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim.x = beams;
    attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    const bool cluster = beams <= CLUSTER_BEAMS;
    config.attrs = cluster ? attributes : attributes + 1;
    config.numAttrs = (cluster ? 1 : 0) + (mlxone_pdl_enabled() ? 1 : 0);
    const auto kernel = cluster ? beam_choice_kernel<true> : beam_choice_kernel<false>;
    cudaLaunchKernelEx(&config, kernel, logits, stride, vocab, (const float*)maxima, (const float*)sums, parts, beams,
                       scores, ended, ends, end_count, keys, tokens, arrived, scores_out, parents_out, tokens_out,
                       ended_out);
    MLXONE_LAUNCH_CHECK("beam_choice");
    return 0;
}
MLXONE_BY_WORDS(mlxone_beam_select)

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
MLXONE_BY_WORDS(mlxone_reorder_slots)

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
MLXONE_BY_WORDS(mlxone_reorder_pages)
