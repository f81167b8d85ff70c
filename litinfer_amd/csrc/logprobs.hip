// Log probabilities of given tokens, the entropy of their rows and the likeliest tokens, from rows of float32 logits.
//
// With m the row's maximum, c the number of logits equal to it and R the sum of exp(x - m) over the others:
//     log S = log c + log1p(R / c),  log p(i) = (x_i - m) - log S,  entropy = log S - sum(exp(x - m) (x - m)) / S.
// The maximum's own share is counted, not added up, so that what is small beside it (the entropy of a sure row, the
// log probability of its token) keeps its digits.  All sums are float32 with a fixed order.
//
// Bound by the one read of the logits (2,047 rows of 151,936: 1.24 GB in 212 us, 5.9 TB/s; 64 rows 12 us, of which 5 are the launches and the first trip to
// memory; one row 4.6 us; 20 alternatives of each cost 27, 7.5 and 4 us more).  A wave takes LP_GROUP * U of a row's logits into registers, finds their
// maximum and then adds up against it: no running rescaling, one pass.  It also leaves the maximum of every group of LP_GROUP logits:
// the row's k largest logits, ordered by (value, lower index first), all lie in the k groups whose maxima are first in that
// order (a group in front of them has a logit that is before any of theirs), so the second kernel reads k groups again
// instead of the row.
#include "common.h"

#define LP_GROUP 256              // logits of a group: one float4 a lane
#define LP_MAX_GROUPS 4096
#define LP_MAX_TOP 32
#define LP_WAVES 4
#define LP_JOIN_WAVES 8          // of a block that joins a row

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));        // (rows need not begin on 16 bytes)

struct RowShare { float m, c, r, t; };       // a wave's maximum, how many equal it, sum of the others' exp, sum of exp(d) d

// unsigned integers in the order of the floats; NaN counts as -inf, -0 as 0
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = x != x ? 0xff800000u : __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float float_of(uint32_t o) { return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o); }

// Logits e .. e + 3 of a row of V, -inf behind its end.
__device__ __forceinline__ void load_four(const float* src, int e, int V, float (&v)[4]) {
    if (e + 3 < V) {
        const f32x4u y = *reinterpret_cast<const f32x4u*>(src + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = y[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = e + j < V ? src[e + j] : -INFINITY;
    }
}

template <int U>
__global__ __launch_bounds__(64 * LP_WAVES) void logprob_rows_kernel(const float* __restrict__ x, long stride, int V, int shares,
                                                                     RowShare* __restrict__ out, float* __restrict__ tops, int groups) {
    const int row = blockIdx.y, lane = threadIdx.x & 63, part = blockIdx.x * LP_WAVES + (threadIdx.x >> 6);
    if (part >= shares) return;
    const float* src = x + (size_t)row * stride;
    const int at = part * (LP_GROUP * U);
    float v[U][4];
    float m = -INFINITY;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        load_four(src, at + u * LP_GROUP + 4 * lane, V, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float a = fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3]));
        m = fmaxf(m, a);
        if (tops) {
            const float g = wave_max(a);
            const int k = part * U + u;
            if (lane == 0 && k < groups) tops[(size_t)row * groups + k] = g;
            m = fmaxf(m, g);
        }
    }
    if (!tops) m = wave_max(m);
    const float base = m == -INFINITY ? 0.f : m;
    float c = 0.f, r = 0.f, t = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float d = v[u][j] - base;
            const float e = __builtin_amdgcn_exp2f(d * 1.44269504088896341f);
            const bool same = v[u][j] == m;
            c += same ? 1.f : 0.f;
            r += same ? 0.f : e;
            t += e * fmaxf(d, -1e30f);           // (a logit of -inf has no share; one that is NaN makes the sums NaN)
        }
    c = wave_sum(c);
    r = wave_sum(r);
    t = wave_sum(t);
    if (lane == 0) out[(size_t)row * shares + part] = {m, c, r, t};
}

__device__ __forceinline__ uint64_t wave_max64(uint64_t v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
        const uint64_t w = ((uint64_t)(uint32_t)lane_xor((int)(v >> 32), o) << 32) | (uint32_t)lane_xor((int)(uint32_t)v, o);
        v = w > v ? w : v;
    }
    return v;
}

// The largest of the block's values, in every thread.
__device__ __forceinline__ uint64_t block_max64(uint64_t v, uint64_t* smem) {
    v = wave_max64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = v;
    __syncthreads();
    uint64_t b = smem[0];
#pragma unroll
    for (int w = 1; w < LP_JOIN_WAVES; ++w) b = smem[w] > b ? smem[w] : b;
    return b;
}

// How many of the block's threads' values are counted by f, in every thread; `turn` alternates between calls (one barrier each).
template <typename F>
__device__ __forceinline__ int block_count(int n, int (*smem)[LP_JOIN_WAVES], int turn, F f) {
    int c = 0;
    for (int i = threadIdx.x; i < n; i += 64 * LP_JOIN_WAVES) c += __popcll(__ballot(f(i)));      // (of the lanes that are still in the loop)
    if ((threadIdx.x & 63) == 0) smem[turn & 1][threadIdx.x >> 6] = c;       // (the wave's first lane leaves the loop last)
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < LP_JOIN_WAVES; ++w) c += smem[turn & 1][w];
    return c;
}

// One block a row: joins the waves' shares, then finds the likeliest tokens.  A value that at least k and at most LP_LIST groups' maxima
// reach is found by halving the range between the least and the largest; the logits of these groups that reach it are gathered (at least
// k, seldom many more) and each one's rank counted.  Where many values are equal or likely tokens lie side by side no such value may exist, or more
// logits reach it than there is room for: then the k first are taken one after the other.  So they are in every row of few groups, of which no more are wanted than
// there are (`enough`, 30 for 20 alternatives: up to 7,680 logits; 48 for 32): there all logits reach.  (64 rows with 20 alternatives, us of both kernels: 3,001 logits 32,
// 7,500 42, 8,000 12.)  A chain of short steps with a barrier behind each: eight waves
// take 9.2 us for a row with 20 alternatives (both kernels), four 11.3, sixteen 9.0; at 2,047 rows 242, 242 and 256.
#define LP_LIST 64                // groups that are looked through
#define LP_ROOM 256               // logits that are ranked
__global__ __launch_bounds__(64 * LP_JOIN_WAVES) void logprob_join_kernel(const float* __restrict__ x, long stride, int V, int shares,
                                                                     const RowShare* __restrict__ in, const float* __restrict__ tops, int groups,
                                                                     const int* __restrict__ ids, float* __restrict__ logprob,
                                                                     float* __restrict__ entropy, int top, int* __restrict__ top_ids,
                                                                     float* __restrict__ top_logprob) {
    constexpr int NT = 64 * LP_JOIN_WAVES;
    __shared__ float red[LP_JOIN_WAVES], sums[LP_JOIN_WAVES][3];
    __shared__ uint64_t red64[LP_JOIN_WAVES], list[LP_ROOM];
    __shared__ int chosen[LP_LIST], counts[2][LP_JOIN_WAVES], found;
    extern __shared__ uint32_t keys[];                    // the groups' maxima, in their order (and room for the k first groups' logits)
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const float* src = x + (size_t)row * stride;
    in += (size_t)row * shares;
    // (what is read from memory is asked for before the first of it is waited for)
    const RowShare none = {-INFINITY, 0.f, 0.f, 0.f}, first = tid < shares ? in[tid] : none;
    const int id = ids[row];
    const float given = id >= 0 && id < V ? src[id] : NAN;
    if (top) {
        tops += (size_t)row * groups;
        for (int i = tid; i < groups; i += NT) keys[i] = order_of(tops[i]);
        if (tid == 0) found = 0;
    }
    float m = first.m;
    for (int i = tid + NT; i < shares; i += NT) m = fmaxf(m, in[i].m);
    m = wave_max(m);
    if (lane == 0) red[w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < LP_JOIN_WAVES; ++i) m = fmaxf(m, red[i]);
    float c = 0.f, r = 0.f, t = 0.f;
    for (int i = tid; i < shares; i += NT) {
        const RowShare s = i == tid ? first : in[i];
        if (s.m == m) { c += s.c; r += s.r; t += s.t; continue; }
        const float d = fmaxf(s.m - m, -1e30f), e = expf(s.m - m);
        r += e * (s.c + s.r);
        t += e * (s.t + (s.c + s.r) * d);
    }
    c = wave_sum(c);
    r = wave_sum(r);
    t = wave_sum(t);
    if (lane == 0) { sums[w][0] = c; sums[w][1] = r; sums[w][2] = t; }
    __syncthreads();
    c = r = t = 0.f;
#pragma unroll
    for (int i = 0; i < LP_JOIN_WAVES; ++i) { c += sums[i][0]; r += sums[i][1]; t += sums[i][2]; }
    // (a maximum that is not finite leaves no probabilities)
    const float log_s = fabsf(m) < INFINITY ? logf(c) + log1pf(r / c) : NAN;
    if (tid == 0) {
        logprob[row] = (given - m) - log_s;
        entropy[row] = log_s - t / (c + r);
    }
    if (!top) return;
    // lo is reached by at least `want` groups, hi by fewer (rows of fewer groups than tokens are wanted: by all of them)
    const int want = top < groups ? top : groups;
    uint32_t lo = 0, hi = order_of(m);
    int n = groups, turn = 0;
    if (top == 1) {
        lo = hi;
        n = 1;
    } else {
        // (likely tokens lie a few nats below the first: four tries there, then halves)
        const int enough = min(LP_LIST, want + max(4, want / 2));
        for (float d = 2.f; n > enough && d < 64.f && fabsf(m) < 1e30f; d *= 2.5f) {
            const uint32_t mid = order_of(m - d);
            if (mid <= lo || mid >= hi) break;
            const int reach = block_count(groups, counts, turn++, [&](int i) { return keys[i] >= mid; });
            if (reach >= want) { lo = mid; n = reach; break; }
            hi = mid;
        }
        while (n > enough && hi - lo > 1) {
            const uint32_t mid = lo + (hi - lo) / 2;
            const int reach = block_count(groups, counts, turn++, [&](int i) { return keys[i] >= mid; });
            if (reach >= want) { lo = mid; n = reach; } else hi = mid;
        }
    }
    bool ranked = n <= LP_LIST;
    if (ranked) {
        // the groups in any order, then their logits that reach lo
        for (int i = tid; i < groups; i += NT)
            if (keys[i] >= lo) {
                const int at = atomicAdd(&found, 1);
                if (at < LP_LIST) chosen[at] = i;
            }
        __syncthreads();
        const int held = found;
        ranked = held <= LP_LIST;                         // (one maximum may be many groups')
        __syncthreads();
        if (tid == 0) found = 0;
        __syncthreads();
        if (ranked) {
            constexpr int AT_ONCE = 4;                    // groups of a wave that are on their way together
            for (int g0 = w; g0 < held; g0 += AT_ONCE * LP_JOIN_WAVES) {
                float v[AT_ONCE][4];
                int from[AT_ONCE];
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i) {
                    const int g = g0 + i * LP_JOIN_WAVES;
                    from[i] = g < held ? chosen[g] * LP_GROUP + 4 * lane : V;
                    load_four(src, from[i], V, v[i]);
                }
#pragma unroll
                for (int i = 0; i < AT_ONCE; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t u = order_of(v[i][j]);
                        if (from[i] + j < V && u >= lo) {
                            const int at = atomicAdd(&found, 1);
                            if (at < LP_ROOM) list[at] = ((uint64_t)u << 32) | (uint32_t)~(from[i] + j);
                        }
                    }
            }
            __syncthreads();
            ranked = found <= LP_ROOM;
        }
    }
    if (ranked) {
        const int held = found;
        if (tid < held) {
            const uint64_t mine = list[tid];
            int rank = 0;
            for (int i = 0; i < held; ++i) rank += list[i] > mine ? 1 : 0;
            if (rank < top) {
                const int id = (int)~(uint32_t)mine;
                top_ids[(size_t)row * top + rank] = id;
                top_logprob[(size_t)row * top + rank] = (float_of((uint32_t)(mine >> 32)) - m) - log_s;
            }
        }
        return;
    }
    // the groups with the k first maxima, one after the other, then their logits
    uint64_t before = ~0ull;
    for (int k = 0; k < want; ++k) {
        uint64_t best = 0;
        for (int i = tid; i < groups; i += NT) {
            const uint64_t key = ((uint64_t)keys[i] << 32) | (uint32_t)~i;
            if (key < before && key > best) best = key;
        }
        before = block_max64(best, red64);
        if (tid == 0) chosen[k] = (int)~(uint32_t)before;
    }
    __syncthreads();
    uint32_t* logits = keys + groups;                     // these groups' logits, in their order; 0: behind the row's end
    for (int i = tid; i < want * LP_GROUP; i += NT) {
        const int e = chosen[i / LP_GROUP] * LP_GROUP + i % LP_GROUP;
        logits[i] = e < V ? order_of(src[e]) : 0u;
    }
    before = ~0ull;
    for (int k = 0; k < top; ++k) {
        uint64_t best = 0;
        for (int i = tid; i < want * LP_GROUP; i += NT) {            // (a thread's own)
            const uint64_t key = ((uint64_t)logits[i] << 32) | (uint32_t)~(chosen[i / LP_GROUP] * LP_GROUP + i % LP_GROUP);
            if (logits[i] && key < before && key > best) best = key;
        }
        before = block_max64(best, red64);
        if (tid == 0) {
            const int id = (int)~(uint32_t)before;
            top_ids[(size_t)row * top + k] = id;
            top_logprob[(size_t)row * top + k] = (float_of((uint32_t)(before >> 32)) - m) - log_s;
        }
    }
}

static int row_shares(int V, int u) { return (V + LP_GROUP * u - 1) / (LP_GROUP * u); }
static int groups_of(int V) { return (V + LP_GROUP - 1) / LP_GROUP; }
// Groups of a wave: few where there are few rows, for more waves.  Two and eight, us with 20 alternatives: one row 11.3 and 12.1, 64 rows 21.1 and
// 23.6, 128 rows 26.7 and 31.9, 512 rows 73.3 and 70.2.
static int share_groups(int n) { return n <= 128 ? 2 : 8; }

// Floats of workspace that li_token_logprobs takes for n rows of V logits.
extern "C" long li_token_logprobs_work_floats(int n, int V) {
    if (n <= 0 || V <= 0) return 0;
    return (long)n * (4L * row_shares(V, share_groups(n)) + groups_of(V));
}

// logits [n, V], rows `stride` floats apart; ids [n]; logprob, entropy [n]; top_ids, top_logprob [n, top] (top 0: none).  An id
// outside the row has no probability (NaN).
extern "C" int li_token_logprobs(const float* logits, long stride, const int* ids, int n, int V, int top, float* logprob, float* entropy,
                                 int* top_ids, float* top_logprob, float* work, hipStream_t stream) {
    if (n <= 0 || n > 1 << 30 || V <= 0 || stride < V || groups_of(V) > LP_MAX_GROUPS || top < 0 || top > LP_MAX_TOP || top > V || !work) return LI_ERR_SIZE;
    const int u = share_groups(n), shares = row_shares(V, u), groups = groups_of(V);
    RowShare* share = (RowShare*)work;
    float* tops = work + 4L * n * shares;
    for (int at = 0; at < n; at += 65535) {               // (rows are the first grid's second axis, and a launch has fewer than 2^32 threads)
        const int rows = n - at < 65535 ? n - at : 65535;
        const dim3 grid((shares + LP_WAVES - 1) / LP_WAVES, rows);
        const float* x = logits + (size_t)at * stride;
        RowShare* s = share + (size_t)at * shares;
        float* g = top ? tops + (size_t)at * groups : nullptr;
        if (u == 2) logprob_rows_kernel<2><<<grid, 64 * LP_WAVES, 0, stream>>>(x, stride, V, shares, s, g, groups);
        else logprob_rows_kernel<8><<<grid, 64 * LP_WAVES, 0, stream>>>(x, stride, V, shares, s, g, groups);
        logprob_join_kernel<<<rows, 64 * LP_JOIN_WAVES, top ? 4 * (groups + (top < groups ? top : groups) * LP_GROUP) : 0, stream>>>(
            x, stride, V, shares, s, g, groups, ids + at, logprob + at, entropy + at, top, top ? top_ids + (size_t)at * top : nullptr,
            top ? top_logprob + (size_t)at * top : nullptr);
    }
    return li_launch_status();
}
