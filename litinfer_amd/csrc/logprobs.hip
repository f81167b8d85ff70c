// Log probabilities of given tokens, the entropy of their rows and the likeliest tokens, from rows of float32 logits.
//
// With m the row's maximum, c the number of logits equal to it and R the sum of exp(x - m) over the others:
//     log S = log c + log1p(R / c),  log p(i) = (x_i - m) - log S,  entropy = log S - sum(exp(x - m) (x - m)) / S.
// The maximum's own share is counted, not added up, so that what is small beside it (the entropy of a sure row, the
// log probability of its token) keeps its digits.  All sums are float32 with a fixed order.
//
// Bound by the one read of the logits.  A wave takes LP_GROUP * U of a row's logits into registers, finds their maximum and
// then adds up against it: no running rescaling, one pass.  It also leaves the maximum of every group of LP_GROUP logits:
// the row's k largest logits, ordered by (value, lower index first), all lie in the k groups whose maxima are first in that
// order (a group in front of them has a logit that is before any of theirs), so the second kernel reads k groups again
// instead of the row.
#include "common.h"

#define LP_GROUP 256              // logits of a group: one float4 a lane
#define LP_MAX_GROUPS 4096
#define LP_MAX_TOP 32
#define LP_WAVES 4

typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));        // (rows need not begin on 16 bytes)

struct RowShare { float m, c, r, t; };       // a wave's maximum, how many equal it, sum of the others' exp, sum of exp(d) d

// unsigned integers in the order of the floats; NaN counts as -inf, -0 as 0
__device__ __forceinline__ uint32_t order_of(float x) {
    const uint32_t u = x != x ? 0xff800000u : __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
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
        const int e = at + u * LP_GROUP + 4 * lane;
        if (e + 3 < V) {
            const f32x4u y = *reinterpret_cast<const f32x4u*>(src + e);
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = y[j];
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = e + j < V ? src[e + j] : -INFINITY;
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const float a = fmaxf(fmaxf(v[u][0], v[u][1]), fmaxf(v[u][2], v[u][3]));
        m = fmaxf(m, a);
        if (tops) {
            const float g = wave_max(a);
            const int k = part * U + u;
            if (lane == 0 && k < groups) tops[(size_t)row * groups + k] = g;
        }
    }
    m = wave_max(m);
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
    for (int w = 1; w < LP_WAVES; ++w) b = smem[w] > b ? smem[w] : b;
    return b;
}

// One block a row: joins the waves' shares, then finds the likeliest tokens.
__global__ __launch_bounds__(64 * LP_WAVES) void logprob_join_kernel(const float* __restrict__ x, long stride, int V, int shares,
                                                                     const RowShare* __restrict__ in, const float* __restrict__ tops, int groups,
                                                                     const int* __restrict__ ids, float* __restrict__ logprob,
                                                                     float* __restrict__ entropy, int top, int* __restrict__ top_ids,
                                                                     float* __restrict__ top_logprob) {
    constexpr int NT = 64 * LP_WAVES;
    __shared__ float red[LP_WAVES];
    __shared__ uint64_t red64[LP_WAVES];
    __shared__ int chosen[LP_MAX_TOP];
    const int row = blockIdx.x, tid = threadIdx.x;
    const float* src = x + (size_t)row * stride;
    in += (size_t)row * shares;
    float m = -INFINITY;
    for (int i = tid; i < shares; i += NT) m = fmaxf(m, in[i].m);
    m = wave_max(m);
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    float c = 0.f, r = 0.f, t = 0.f;
    for (int i = tid; i < shares; i += NT) {
        const RowShare s = in[i];
        if (s.m == m) { c += s.c; r += s.r; t += s.t; continue; }
        const float d = fmaxf(s.m - m, -1e30f), e = expf(s.m - m);
        r += e * (s.c + s.r);
        t += e * (s.t + (s.c + s.r) * d);
    }
    c = block_sum<NT>(c, red);
    r = block_sum<NT>(r, red);
    t = block_sum<NT>(t, red);
    // (a maximum that is not finite leaves no probabilities)
    const float log_s = fabsf(m) < INFINITY ? logf(c) + log1pf(r / c) : NAN;
    if (tid == 0) {
        const int id = ids[row];
        logprob[row] = id >= 0 && id < V ? (src[id] - m) - log_s : NAN;
        entropy[row] = log_s - t / (c + r);
    }
    if (!top) return;
    // the groups with the k first maxima, one after the other
    tops += (size_t)row * groups;
    uint64_t before = ~0ull;
    for (int k = 0; k < top && k < groups; ++k) {
        uint64_t best = 0;
        for (int i = tid; i < groups; i += NT) {
            const uint64_t key = ((uint64_t)order_of(tops[i]) << 32) | (uint32_t)~i;
            if (key < before && key > best) best = key;
        }
        before = block_max64(best, red64);
        if (tid == 0) chosen[k] = (int)~(uint32_t)before;
    }
    __syncthreads();
    const int n = (top < groups ? top : groups) * LP_GROUP;
    before = ~0ull;
    for (int k = 0; k < top; ++k) {
        uint64_t best = 0;
        for (int i = tid; i < n; i += NT) {
            const int e = chosen[i / LP_GROUP] * LP_GROUP + i % LP_GROUP;
            if (e >= V) continue;
            const uint64_t key = ((uint64_t)order_of(src[e]) << 32) | (uint32_t)~e;
            if (key < before && key > best) best = key;
        }
        before = block_max64(best, red64);
        if (tid == 0) {
            const int id = (int)~(uint32_t)before;
            top_ids[(size_t)row * top + k] = id;
            top_logprob[(size_t)row * top + k] = (src[id] - m) - log_s;
        }
    }
}

static int row_shares(int V, int u) { return (V + LP_GROUP * u - 1) / (LP_GROUP * u); }
static int groups_of(int V) { return (V + LP_GROUP - 1) / LP_GROUP; }
static int share_groups(int n) { return n <= 16 ? 2 : 8; }

// Floats of workspace that li_token_logprobs takes for n rows of V logits.
extern "C" long li_token_logprobs_work_floats(int n, int V) {
    if (n <= 0 || V <= 0) return 0;
    return (long)n * (4L * row_shares(V, share_groups(n)) + groups_of(V));
}

extern "C" int li_token_logprobs_max_top(void) { return LP_MAX_TOP; }
extern "C" int li_token_logprobs_max_vocab(void) { return LP_MAX_GROUPS * LP_GROUP; }

// logits [n, V], rows `stride` floats apart; ids [n]; logprob, entropy [n]; top_ids, top_logprob [n, top] (top 0: none).  An id
// outside the row has no probability (NaN).
extern "C" int li_token_logprobs(const float* logits, long stride, const int* ids, int n, int V, int top, float* logprob, float* entropy,
                                 int* top_ids, float* top_logprob, float* work, hipStream_t stream) {
    if (n <= 0 || V <= 0 || stride < V || groups_of(V) > LP_MAX_GROUPS || top < 0 || top > LP_MAX_TOP || top > V || !work) return LI_ERR_SIZE;
    const int u = share_groups(n), shares = row_shares(V, u), groups = groups_of(V);
    RowShare* share = (RowShare*)work;
    float* tops = work + 4L * n * shares;
    for (int at = 0; at < n; at += 65535) {               // (rows are the grid's second axis)
        const int rows = n - at < 65535 ? n - at : 65535;
        const dim3 grid((shares + LP_WAVES - 1) / LP_WAVES, rows);
        const float* x = logits + (size_t)at * stride;
        RowShare* s = share + (size_t)at * shares;
        float* g = top ? tops + (size_t)at * groups : nullptr;
        if (u == 2) logprob_rows_kernel<2><<<grid, 64 * LP_WAVES, 0, stream>>>(x, stride, V, shares, s, g, groups);
        else logprob_rows_kernel<8><<<grid, 64 * LP_WAVES, 0, stream>>>(x, stride, V, shares, s, g, groups);
    }
    logprob_join_kernel<<<n, 64 * LP_WAVES, 0, stream>>>(logits, stride, V, shares, share, tops, groups, ids, logprob, entropy, top, top_ids, top_logprob);
    return li_launch_status();
}
