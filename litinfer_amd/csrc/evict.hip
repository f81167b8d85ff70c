// A cache of bounded length: the attention weight that every cached key has drawn, the choice of the keys that stay, and
// their move to the front of the request's pages.
//
//   li_attention_mass   mass[t, g] += sum over the step's queries i that see key t and the query heads h of kv head g of
//                       exp(s_iht - lse_ih), s = scale q_ih . k_tg, lse_ih = log of the sum of exp(s) over the keys that i sees;
//                       a key that this step wrote is set, not added to.
//   li_evict_select     the places of a request that stay: the first, the last, the others by largest mass.
//   li_cache_compact    row j of a request's tensors <- row kept[j].
//
// A page of keys is [kv heads, page size, head size], one of sums [kv heads, page size] float32; a request's block table maps
// place / page size to the page.
#include "common.h"

#include <algorithm>
#include <type_traits>

#define EV_MAX_DH 256
// Places of a request, and rows that a list has room for: loops that step over them in 32 bits end behind the last.
#define EV_MAX_PLACES (1L << 30)

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ attention weight
// Two passes over the scores, since a weight needs the whole row's sum first: the rows' log-sums, then the columns' sums.  Scores
// are held in powers of two (scale times log2 e); a row's statistic is lse = m + log2(sum of 2^(s - m)).
struct MassArgs {
    const int *block_table, *q_start, *q_len, *ctx_len;
    int max_blocks, nh, nkv, dh, page_size, num_pages, q_row_stride;
    uint32_t page_inv;           // 2^32 / page_size, rounded down (page_of)
    float scale;                 // times log2(e)
    int fresh;                   // keys written by this step are set
};

// Segments of the batch that a launch takes, by value: a step's mix is known on the host, and what the workspace was laid out for is what the
// kernels go by.  (A recorded step has single tokens only, all of them, and reads their contexts from the device.)
#define EV_LIST 64
struct Seg {
    int seg, start, q, ctx;
    int off;                     // where the segment's places begin among all; of single tokens, where its scores begin in the workspace
};
struct SegList {
    int n;                       // 0: segment i is the i-th, all of them, lengths from the device
    Seg of[EV_LIST];             // (a segment's numbers side by side: a trip to the launch's arguments takes long)
};

static uint32_t inverse_of(int page_size) { return page_size == 1 ? 0xffffffffu : (uint32_t)((1ull << 32) / (uint32_t)page_size); }
// place / page_size and the rest: the product with the rounded-down inverse is at most one too small
__device__ __forceinline__ int page_of(const MassArgs& a, int t, int& rest) {
    int p = (int)__umulhi((uint32_t)t, a.page_inv);
    rest = t - p * a.page_size;
    if (rest >= a.page_size) { ++p; rest -= a.page_size; }
    return p;
}
// place -> row of [kv heads, page size, *] inside the pool, or -1 where no page holds the place
__device__ __forceinline__ long place_row(const MassArgs& a, const int* table, int kvh, int t) {
    int rest;
    const int page = table[page_of(a, t, rest)];
    if (page < 0 || page >= a.num_pages) return -1;
    return ((long)page * a.nkv + kvh) * a.page_size + rest;
}
// A segment's length on the device, no more than there is room for in the table and where `most` places were laid out (a replay may be told anything).
__device__ __forceinline__ int device_ctx(const MassArgs& a, int seg, int most) { return min(min(a.ctx_len[seg], most), a.max_blocks * a.page_size); }
// the row of a place, some row where there is none (whoever asks does not use it)
__device__ __forceinline__ long some_row(const MassArgs& a, const int* table, int kvh, int t) {
    const long r = place_row(a, table, kvh, t);
    return r < 0 ? (long)kvh * a.page_size : r;
}

// ---- any head size, type and alignment: scores by the vector ALU, computed twice.  Nothing here is made for speed: rows of whole 16 bytes on 16 bytes, which
// models have, go the other ways.  (14 heads on 2 of 36 bfloat16: 8 requests of 2,000 keys 64 us; 512 queries behind 2,048 keys 2.7 ms, where heads of 64 take 29 us.)
template <typename T>
__device__ __forceinline__ float dot_rows(const float* q, const T* k, int dh) {
    float s = 0.f;
    for (int d = 0; d < dh; ++d) s += q[d] * load_as_float(k + d);
    return s;
}

// lse [T, nh]: a wave a (token, head), a key a lane.
template <typename T>
__global__ __launch_bounds__(64) void mass_rows_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, float* __restrict__ lse) {
    __shared__ float qs[EV_MAX_DH];
    const int seg = blockIdx.z, h = blockIdx.y, i = blockIdx.x, lane = threadIdx.x;
    if (i >= a.q_len[seg]) return;
    const int tok = a.q_start[seg] + i, seen = device_ctx(a, seg, 0x7fffffff) - a.q_len[seg] + i + 1;
    const int* table = a.block_table + (size_t)seg * a.max_blocks;
    for (int d = lane; d < a.dh; d += 64) qs[d] = load_as_float(q + (size_t)tok * a.q_row_stride + (size_t)h * a.dh + d);
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    for (int t = lane; t < seen; t += 64) {
        const long row = place_row(a, table, h / (a.nh / a.nkv), t);
        if (row < 0) continue;
        const float s = dot_rows(qs, k + row * a.dh, a.dh) * a.scale;
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;     // (a score of NaN has no part in the maximum, but in the sum)
        l = (m == -INFINITY ? l : l * exp2f(m - base)) + exp2f(s - base);
        m = mn;
    }
    const float mx = wave_max(m);
    l = wave_sum(m == -INFINITY ? l : l * exp2f(m - mx));
    // (a row that sees nothing gives nothing)
    if (lane == 0) lse[(size_t)tok * a.nh + h] = l == 0.f ? INFINITY : (mx == -INFINITY ? 0.f : mx) + log2f(l);
}

// A block takes 64 keys of a (request, kv head); its four waves take the queries in turn and are added up in their order.
template <typename T>
__global__ __launch_bounds__(256) void mass_keys_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, const float* __restrict__ lse,
                                                        float* __restrict__ mass) {
    __shared__ float qs[4][EV_MAX_DH], part[4][64];
    const int seg = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int nq = a.q_len[seg], ctx = device_ctx(a, seg, 0x7fffffff), t = blockIdx.x * 64 + lane, rep = a.nh / a.nkv;
    if ((int)blockIdx.x * 64 >= ctx) return;
    const long row = t < ctx ? place_row(a, a.block_table + (size_t)seg * a.max_blocks, kvh, t) : -1;
    const int base = ctx - nq;                           // place of the step's first token
    const int i0 = max((int)blockIdx.x * 64 - base, 0);  // the first query that sees any of the block's keys
    float sum = 0.f;
    for (int i = i0; i < nq; i += 4) {
        float some = 0.f;                                // (a query's heads first: shorter sums keep their digits)
        for (int r = 0; r < rep; ++r) {
            const int mine = i + w, tok = a.q_start[seg] + mine, h = kvh * rep + r;
            __syncthreads();
            if (mine < nq)
                for (int d = lane; d < a.dh; d += 64) qs[w][d] = load_as_float(q + (size_t)tok * a.q_row_stride + (size_t)h * a.dh + d);
            __syncthreads();
            if (mine < nq && row >= 0 && t <= base + mine)
                some += exp2f(dot_rows(qs[w], k + row * a.dh, a.dh) * a.scale - lse[(size_t)tok * a.nh + h]);
        }
        sum += some;
    }
    part[w][lane] = sum;
    __syncthreads();
    if (w || row < 0) return;
    sum = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
    mass[row] = a.fresh && t >= base ? sum : mass[row] + sum;
}

// ---- on the matrix cores.  A lane's operand is a piece of 16 bytes of a row, as it lies in memory: 8 bfloat16 (one MFMA), or
// 4 float32 (the e-th of four MFMAs takes the e-th; which k a slot stands for is the same on both sides).
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ f32x4_t mma16(const u32x4_t a, const u32x4_t b, f32x4_t c) {        // 16 x 16, rows of a against rows of b
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
}
template <typename T>
__device__ __forceinline__ f32x16_t mma32(const u32x4_t a, const u32x4_t b, f32x16_t c) {      // 32 x 32
    if constexpr (sizeof(T) == 2) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
    } else {
        const f32x4_t x = __builtin_bit_cast(f32x4_t, a), y = __builtin_bit_cast(f32x4_t, b);
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], y[e], c, 0, 0, 0);
        return c;
    }
}

// ---- single tokens.  The scores themselves are kept (4 bytes a query head and key beside the key's dh * 2): reading the keys
// again would cost more.  Bound by the keys' way from memory and, at these sizes, by the launches around it: 64 requests of 100 to 2,001 keys, 12 heads on 2 of 128
// bfloat16 (36 MB), 13.8 us for the scores and 5.3 for the sums; 3 of 20,000 to 32,001 keys, 28 heads on 4 of 128 float32 (162 MB), 39.6 (4.0 TB/s) and 12.1; one
// of 300 keys, 14 heads on 2, 6.2 in one kernel.  A recorded step lays its scores out for the whole tables: 28 heads on 4 of 128 bfloat16, 8 requests of
// 4,000 keys 15.6 in tables of 4,096 places and 22.4 in tables of 32,768 (named, 15.4), 64 of 1,000 in tables of 4,096 57.5 (named, one kernel, 16.6).
#define SG_KEYS 64                // keys of a wave
#define SG_WAVES 4
// Floats of workspace that the requests of a launch take together, unless one takes more by itself: a batch beyond that goes in several launches, one
// after the other, which use it again.  (256 MiB: more work than fills the chip many times over.)
#define SG_ROOM (1L << 26)

// A request's scores [heads, 64 parts] and behind them the statistics (maximum, sum) [heads, parts], a head's in whole lines of 128 bytes.
constexpr int stat_stride(int parts) { return (parts + 15) & ~15; }
static long single_floats(int nh, int parts) { return nh * (parts * (long)SG_KEYS + 2 * stat_stride(parts)); }

// Scores of the 64 keys from k0 on against the heads of a kv head, 16 at a time, by a wave, and the maximum and sum for every head:
// scores [head of the kv head, stride] from key k0 on, stats [head, parts].
template <typename T, int CH>
__device__ __forceinline__ void single_scores(const T* __restrict__ qrow, const T* __restrict__ k, const MassArgs& a, const int* table, int kvh, int k0, int ctx,
                                              int lane, float* scores, long stride, float2* stats, int parts) {
    constexpr int PE = 16 / sizeof(T);                   // elements of a piece
    constexpr int NT = CH * 4 <= 16 ? 4 : CH * 2 <= 16 ? 2 : 1;      // tiles of 16 keys whose pieces are asked for at once
    const int c = lane & 15, g = lane >> 4, rep = a.nh / a.nkv, dh = a.dh;
    long row[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) row[i] = k0 + 16 * i + c < ctx ? place_row(a, table, kvh, k0 + 16 * i + c) : -1;
    const u32x4_t zero = {0, 0, 0, 0};
    for (int h0 = 0; h0 < rep; h0 += 16) {
        u32x4_t qf[CH];
#pragma unroll
        for (int j = 0; j < CH; ++j) {
            const int d = (4 * j + g) * PE;
            qf[j] = h0 + c < rep && d < dh ? *reinterpret_cast<const u32x4_t*>(qrow + (size_t)(h0 + c) * dh + d) : zero;
        }
        f32x4_t s[4];
#pragma unroll
        for (int i0 = 0; i0 < 4; i0 += NT) {
            u32x4_t kf[NT][CH];
#pragma unroll
            for (int i = 0; i < NT; ++i)
#pragma unroll
                for (int j = 0; j < CH; ++j) {
                    const int d = (4 * j + g) * PE;
                    kf[i][j] = row[i0 + i] >= 0 && d < dh ? *reinterpret_cast<const u32x4_t*>(k + row[i0 + i] * dh + d) : zero;
                }
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < CH; ++j) acc = mma16<T>(kf[i][j], qf[j], acc);
                s[i0 + i] = acc;
            }
        }
        // lane (c, g) holds head c's scores of keys 16 i + 4 g + 0..3
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t there = (uint32_t)__ballot(row[i] >= 0) >> (4 * g);       // (lanes 0 .. 15: keys 16 i ..)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                s[i][r] = there >> r & 1 ? s[i][r] * a.scale : -INFINITY;
                m = fmaxf(m, s[i][r]);
            }
        }
        m = lane_xor_max(lane_xor_max(m, 16), 32);
        const float base = m == -INFINITY ? 0.f : m;
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) l += __builtin_amdgcn_exp2f(s[i][r] - base);
        l = lane_xor_add(lane_xor_add(l, 16), 32);
        if (h0 + c < rep) {
            float* out = scores + (size_t)(h0 + c) * stride + k0 + 4 * g;
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<f32x4_t*>(out + 16 * i) = s[i];      // (stride: whole runs of 64)
            if (g == 0) stats[(size_t)(h0 + c) * parts + k0 / SG_KEYS] = make_float2(m, l);
        }
    }
}

// A launch's request `req`: from the list, or the segment `first` + req (then without its row, which only blocks with keys ask for).
__device__ __forceinline__ Seg single_of(const MassArgs& a, const SegList& list, int req, int first, int parts) {
    if (list.n) return list.of[req];
    return {first + req, -1, 1, device_ctx(a, first + req, parts * SG_KEYS), 0};
}
// Where its scores lie: those of listed requests side by side, each as long as it is, of others `parts` runs of 64, `each` floats.
struct Scores {
    int parts;
    float* scores;
    float2* stats;
};
__device__ __forceinline__ Scores scores_of(const MassArgs& a, const SegList& list, const Seg& of, int req, int parts, long each, float* work) {
    Scores s;
    s.parts = list.n ? (of.ctx + SG_KEYS - 1) / SG_KEYS : parts;
    s.scores = work + (list.n ? (long)of.off : req * each);
    s.stats = reinterpret_cast<float2*>(s.scores + (size_t)a.nh * s.parts * SG_KEYS);
    return s;
}

// grid: x runs of 64 keys / 4, y kv heads, z requests.
template <typename T, int CH>
__global__ __launch_bounds__(64 * SG_WAVES) void mass_single_scores_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, SegList list,
                                                                           float* __restrict__ work, long each, int first, int parts) {
    const int req = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 63, rep = a.nh / a.nkv;
    const int k0 = (blockIdx.x * SG_WAVES + (threadIdx.x >> 6)) * SG_KEYS;
    const Seg of = single_of(a, list, req, first, parts);
    if (k0 >= of.ctx) return;
    const Scores s = scores_of(a, list, of, req, parts, each, work);
    const T* qrow = q + (size_t)(list.n ? of.start : a.q_start[of.seg]) * a.q_row_stride + (size_t)kvh * rep * a.dh;
    const size_t head0 = (size_t)kvh * rep;
    const long stride = (long)s.parts * SG_KEYS;
    single_scores<T, CH>(qrow, k, a, a.block_table + (size_t)of.seg * a.max_blocks, kvh, k0, of.ctx, lane, s.scores + head0 * stride, stride, s.stats + head0 * stat_stride(s.parts),
                         stat_stride(s.parts));
}

// lse of a head from the statistics of its `n` parts, by a wave.
__device__ __forceinline__ float join_stats(const float2* st, int n, int lane) {
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < n; i += 64) {
        const float2 v = st[i];
        const float mn = fmaxf(m, v.x), base = mn == -INFINITY ? 0.f : mn;
        l = (m == -INFINITY ? l : l * exp2f(m - base)) + (v.x == -INFINITY ? v.y : v.y * exp2f(v.x - base));
        m = mn;
    }
    const float mx = wave_max(m);
    l = wave_sum(m == -INFINITY ? l : l * exp2f(m - mx));
    return l == 0.f ? INFINITY : (mx == -INFINITY ? 0.f : mx) + log2f(l);
}

// Short contexts: a block takes all of a (request, kv head)'s keys, its scores stay in LDS.  grid: x kv heads, y requests.
// LDS: scores [rep, stride], stats [rep, stride / 64], lse [rep].
constexpr int block_waves(int ch) { return ch >= 8 ? 8 : 16; }          // (as many as have the registers for a run of keys)
template <typename T, int CH>
__global__ __launch_bounds__(64 * block_waves(CH)) void mass_single_block_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, SegList list, int stride,
                                                                          float* __restrict__ mass) {
    constexpr int WAVES = block_waves(CH);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int req = blockIdx.y, seg = list.n ? list.of[req].seg : req, kvh = blockIdx.x, lane = threadIdx.x & 63, w = threadIdx.x >> 6, rep = a.nh / a.nkv;
    const int ctx = list.n ? list.of[req].ctx : device_ctx(a, seg, stride), parts = stride / SG_KEYS;
    float* scores = reinterpret_cast<float*>(lds);
    float2* stats = reinterpret_cast<float2*>(scores + (size_t)rep * stride);
    float* lse = reinterpret_cast<float*>(stats + rep * parts);
    const int* table = a.block_table + (size_t)seg * a.max_blocks;
    const T* qrow = q + (size_t)(list.n ? list.of[req].start : a.q_start[seg]) * a.q_row_stride + (size_t)kvh * rep * a.dh;
    for (int k0 = w * SG_KEYS; k0 < ctx; k0 += WAVES * SG_KEYS)
        single_scores<T, CH>(qrow, k, a, table, kvh, k0, ctx, lane, scores, stride, stats, parts);
    __syncthreads();
    const int n = (ctx + SG_KEYS - 1) / SG_KEYS;
    for (int h = w; h < rep; h += WAVES) {
        const float v = join_stats(stats + h * parts, n, lane);
        if (lane == 0) lse[h] = v;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < ctx; t += 64 * WAVES) {
        const long row = place_row(a, table, kvh, t);
        if (row < 0) continue;
        const float before = a.fresh && t == ctx - 1 ? 0.f : mass[row];
        float sum = 0.f;
        for (int h = 0; h < rep; ++h) sum += __builtin_amdgcn_exp2f(scores[h * stride + t] - lse[h]);
        mass[row] = before + sum;
    }
}

#define SG_LSE 64                 // heads of a kv head whose lse a block holds at a time
__global__ __launch_bounds__(256) void mass_single_add_kernel(MassArgs a, SegList list, float* __restrict__ work, long each, int first, int parts, float* __restrict__ mass) {
    __shared__ float lse[SG_LSE];
    const int req = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6, t = blockIdx.x * 256 + threadIdx.x, rep = a.nh / a.nkv;
    const Seg of = single_of(a, list, req, first, parts);
    const int ctx = of.ctx;
    if ((int)blockIdx.x * 256 >= ctx) return;
    const Scores s = scores_of(a, list, of, req, parts, each, work);
    const int n = (ctx + SG_KEYS - 1) / SG_KEYS;
    const long row = t < ctx ? place_row(a, a.block_table + (size_t)of.seg * a.max_blocks, kvh, t) : -1;
    const float before = row >= 0 && !(a.fresh && t == ctx - 1) ? mass[row] : 0.f;
    const size_t head0 = (size_t)kvh * rep;
    const long stride = (long)s.parts * SG_KEYS;
    float sum = 0.f;
    for (int h0 = 0; h0 < rep; h0 += SG_LSE) {
        const int heads = min(rep - h0, SG_LSE);
        __syncthreads();
        for (int h = w; h < heads; h += 4) {
            const float v = join_stats(s.stats + (head0 + h0 + h) * stat_stride(s.parts), n, lane);
            if (lane == 0) lse[h] = v;
        }
        __syncthreads();
        if (row >= 0)
            for (int h = 0; h < heads; ++h) sum += __builtin_amdgcn_exp2f(s.scores[(head0 + h0 + h) * stride + t] - lse[h]);
    }
    if (row >= 0) mass[row] = before + sum;
}

// ---- portions: tiles of 32 x 32 scores.  One side's rows stay in a wave's registers (ST tiles of 32 rows a wave), the other's go
// through LDS in stages of 64 rows (32 where three of 64 do not fit).  Loads go straight into LDS.  The columns' pass asks for a stage while the one before
// the last is worked on; the rows' pass asks for it then too, but waits for it at once: the table's entry for the stage behind it (look_up) is a load
// like any other, asked for last and wanted first, and loads arrive in order.  So its third stage in LDS gains it nothing, and the rows' pass takes
// a sixth longer than the columns' for the same products.  A row's pieces are swizzled (place p of row r holds piece p ^ (r & 15)), so that rows' pieces of one column lie
// in different banks.
//
// A step is one tile of 32 staged rows: its products, beside them the exponentials of the tile before (MFMAs and the vector ALU work side by
// side), and the first pieces of the next tile's rows, which then wait in registers.  What bounds a step is both together: of two tiles of bfloat16 rows of 128, 16
// MFMAs alone take 262 ns, the 32 exponentials 120, the 64 other vector instructions 115, interleaved 329.  1,999 queries of 40 heads on 8 behind 16,000
// keys: rows' statistics 417 to 448 us, columns' sums 354 to 374 (up to 830 and 980 TFLOP/s of products; matrix cores busy 38 and 47 %, the vector ALU 64 and 59; the log of a
// row's sum is wanted before the first weight can be added, so that all products are made twice).
#define PT_WAVES 4
#define PT_BUFS 3
#define PT_RING 4                 // pieces of a row that are read ahead
constexpr int stage_tiles(int row_bytes) { return PT_BUFS * 64 * row_bytes <= 159 * 1024 ? 2 : 1; }

// 16 bytes a lane from `src`, to `at` (an offset in LDS, the same in all lanes) + 16 * lane; nobody but s_waitcnt vmcnt knows when they have arrived.
__device__ __forceinline__ void load_to_lds(const void* src, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(src) : "memory", "m0");
}
// The same from `base`, the same in all lanes, and `offset` bytes.
__device__ __forceinline__ void load_to_lds(const void* base, uint32_t offset, uint32_t at) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(__builtin_amdgcn_readfirstlane(at)), "v"(offset), "s"(base) : "memory", "m0");
}
__device__ __forceinline__ uint32_t lds_offset(const void* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p; }

// The wave's loads but the `LATER` youngest have arrived, and with them, behind the barrier, all waves' (a wave's loads retire in order).
template <int LATER>
__device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
    __syncthreads();
}
template <int PPR>
__device__ __forceinline__ int swizzle(int r) { return r & (PPR < 16 ? PPR - 1 : 15); }

// All waves bring ROWS rows, PPR places a row: load(i, row, piece, offset in LDS of the lanes' first place) for a lane's i-th place.
template <int PPR, int ROWS, typename Load>
__device__ __forceinline__ void stage_rows(uint32_t at, int w, int lane, Load load) {
    constexpr int LOADS = ROWS * PPR / (64 * PT_WAVES);
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int first = (w * LOADS + i) * 64, slot = first + lane, r = slot / PPR;
        load(i, r, (slot % PPR) ^ swizzle<PPR>(r), at + 16 * first);
    }
}
// Where a lane's pieces of its row lie in a tile.
template <int PPR>
__device__ __forceinline__ void staged_at(int c, int half, int (&at)[PPR / 2]) {
#pragma unroll
    for (int j = 0; j < PPR / 2; ++j) at[j] = 16 * (c * PPR + ((2 * j + half) ^ swizzle<PPR>(c)));
}
__device__ __forceinline__ u32x4_t staged_piece(const char* rows, int at) { return *reinterpret_cast<const u32x4_t*>(rows + at); }

// The tile `rows` against the ST tiles that are held.  ring holds the tile's first pieces; each that has been used makes room for the piece
// PT_RING further on, behind the last for the first ones of the tile `next`.  beside(j) is the share of other work between piece j's
// products and the next's: the order is kept as it is written.
template <int CH, int ST, typename Mma, typename Beside>
__device__ __forceinline__ void multiply_rows(const char* rows, const char* next, const int (&at)[CH], u32x4_t (&ring)[PT_RING], const u32x4_t (&held)[ST][CH],
                                              f32x16_t (&acc)[ST], Mma mma, Beside beside) {
    const f32x16_t zero = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    static_assert(CH % PT_RING == 0, "a tile begins at the ring's beginning");
#pragma unroll
    for (int j = 0; j < CH; ++j) {
#pragma unroll
        for (int x = 0; x < ST; ++x) acc[x] = mma(ring[j % PT_RING], held[x][j], j ? acc[x] : zero);
        ring[j % PT_RING] = j + PT_RING < CH ? staged_piece(rows, at[j + PT_RING]) : staged_piece(next, at[j + PT_RING - CH]);
        beside(j);
        __builtin_amdgcn_sched_barrier(0);
    }
}
template <int ST>
__device__ __forceinline__ void nothing(f32x16_t (&acc)[ST]) {
#pragma unroll
    for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[x][r] = -INFINITY;
}
// Calls step(constant i, t) for t = 0 .. n - 1 with i = t modulo 6: buffers, tiles of a stage and accumulators are constants of the code.
template <typename Step>
__device__ __forceinline__ void in_steps(int n, Step step) {
    for (int t = 0; t < n; t += 6) {
        step(std::integral_constant<int, 0>{}, t);
        if (t + 1 < n) step(std::integral_constant<int, 1>{}, t + 1);
        if (t + 2 < n) step(std::integral_constant<int, 2>{}, t + 2);
        if (t + 3 < n) step(std::integral_constant<int, 3>{}, t + 3);
        if (t + 4 < n) step(std::integral_constant<int, 4>{}, t + 4);
        if (t + 5 < n) step(std::integral_constant<int, 5>{}, t + 5);
    }
}

// The rows' statistics: a wave holds ST * 32 queries of one head, the block streams keys.  Wave tiles of a kv head are numbered from the
// last queries, whose rows are the longest, to the first, a tile's heads side by side: the four that a block takes see about the same keys.
// grid: x kv heads times wave tiles / 4 (of the longest segment), z segments * splits; a split is `share` stages of keys.  The kv head goes fastest,
// here and below: blocks go round the XCDs, so an XCD's second-level cache holds one kv head's rows, or a few.
// stats [splits, nh, T], or, where there is one split, lse [nh, T] itself.
template <typename T, int DHP, int ST>
__global__ __launch_bounds__(64 * PT_WAVES) void mass_rows_tile_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, SegList list,
                                                                       float2* __restrict__ stats, float* __restrict__ lse, int splits, int share,
                                                                       int tokens) {
    constexpr int PE = 16 / sizeof(T), PPR = DHP / PE, CH = PPR / 2, TPS = stage_tiles(16 * PPR), ROWS = 32 * TPS, STAGE_BYTES = ROWS * PPR * 16;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int which = blockIdx.z / splits, seg = list.of[which].seg, split = blockIdx.z % splits, kvh = blockIdx.x % a.nkv, tok0 = list.of[which].start;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, half = lane >> 5;
    const int nq = list.of[which].q, base = list.of[which].ctx - nq, rep = a.nh / a.nkv, pieces = a.dh / PE;
    const int tiles = (nq + 32 * ST - 1) / (32 * ST), wt0 = blockIdx.x / a.nkv * PT_WAVES;
    if (wt0 >= tiles * rep) return;
    const int* table = a.block_table + (size_t)seg * a.max_blocks;
    const int wt = min(wt0 + w, tiles * rep - 1);        // (a wave without a tile repeats the last one and stores nothing)
    const bool mine = wt0 + w < tiles * rep;
    const int h = kvh * rep + wt % rep, i0 = (tiles - 1 - wt / rep) * (32 * ST);
    // the block's keys: up to the last that its first wave sees, this split's share of the stages
    const int last = base + min((tiles - wt0 / rep) * (32 * ST), nq) - 1;
    const int s0 = split * share, s1 = min(last / ROWS + 1, s0 + share);
    if (s0 >= s1) {                                      // none (and there is another split): nothing is what its rows add
        for (int i = i0 + lane; mine && i < min(i0 + 32 * ST, nq); i += 64)
            stats[((size_t)split * a.nh + h) * tokens + tok0 + i] = make_float2(-INFINITY, 0.f);
        return;
    }
    if (pieces < PPR) {
        for (int i = tid; i < PT_BUFS * STAGE_BYTES / 16; i += 64 * PT_WAVES) reinterpret_cast<u32x4_t*>(lds)[i] = u32x4_t{0, 0, 0, 0};
        __syncthreads();
    }
    u32x4_t qf[ST][CH];
    int pos[ST];
#pragma unroll
    for (int x = 0; x < ST; ++x) {
        const int i = min(i0 + 32 * x + c, nq - 1);
        pos[x] = base + i;
        const T* src = q + (size_t)(tok0 + i) * a.q_row_stride + (size_t)h * a.dh;
#pragma unroll
        for (int j = 0; j < CH; ++j) qf[x][j] = 2 * j + half < pieces ? *reinterpret_cast<const u32x4_t*>(src + (2 * j + half) * PE) : u32x4_t{0, 0, 0, 0};
    }
    const int seen_all = base + i0, seen_any = base + min(i0 + 32 * ST, nq) - 1;      // the wave's first and last query's places
    float m[ST], l[ST];
#pragma unroll
    for (int x = 0; x < ST; ++x) { m[x] = -INFINITY; l[x] = 0.f; }
    // (the rows of a stage are looked up in the table a stage before they are asked for, one a lane)
    constexpr int LOADS = ROWS * PPR / (64 * PT_WAVES);
    const uint32_t lds0 = lds_offset(lds);
    uint32_t row = 0;                                    // in pieces
    uint64_t next_there = 0, there[PT_BUFS];             // which of a stage's keys have a page
    auto look_up = [&](int s) __attribute__((always_inline)) {
        const long r = place_row(a, table, kvh, min(s * ROWS + lane % ROWS, last));
        next_there = __ballot(r >= 0);
        row = (uint32_t)(r < 0 ? (long)kvh * a.page_size : r) * pieces;
    };
    auto load = [&](auto which_buf) __attribute__((always_inline)) {
        constexpr int buf = decltype(which_buf)::value;
        there[buf] = next_there;
        if (pieces == PPR)                               // (whole rows need no mask, whose branches cost more than the loads)
            stage_rows<PPR, ROWS>(lds0 + buf * STAGE_BYTES, w, lane, [&](int, int r, int p, uint32_t to) __attribute__((always_inline)) {
                load_to_lds((const u32x4_t*)k + ((uint32_t)__shfl((int)row, r, LI_WAVE) + p), to);
            });
        else
            stage_rows<PPR, ROWS>(lds0 + buf * STAGE_BYTES, w, lane, [&](int, int r, int p, uint32_t to) __attribute__((always_inline)) {
                const uint32_t piece = (uint32_t)__shfl((int)row, r, LI_WAVE) + p;
                if (p < pieces) load_to_lds((const u32x4_t*)k + piece, to);
            });
    };
    int at[CH];
    staged_at<PPR>(c, half, at);
    u32x4_t ring[PT_RING];
    // lane (c, half) gets query c's scores of keys 8 (r / 4) + 4 half + r % 4
    // A tile joins the rows' statistics in CH shares: the first quarter finds the maxima, the others add up.
    float b[ST], sum[ST][4];                             // (four sums: one would wait for itself)
    constexpr int LEAD = CH / 4, EACH = CH - LEAD;
    auto add_up = [&](const f32x16_t (&acc)[ST], int j) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < ST; ++x) {
            if (j == x * LEAD / ST) {
                float mx = acc[x][0];
#pragma unroll
                for (int r = 1; r < 16; ++r) mx = fmaxf(mx, acc[x][r]);
                const float mn = fmaxf(m[x], mx * a.scale);
                b[x] = fmaxf(mn, -1e30f);                // (nothing seen yet: 2^(-inf + 1e30) is nothing)
                l[x] *= __builtin_amdgcn_exp2f(fmaxf(m[x], -1e30f) - b[x]);
                m[x] = mn;
                sum[x][0] = sum[x][1] = sum[x][2] = sum[x][3] = 0.f;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (j >= LEAD && (16 * x + r) * EACH / (16 * ST) == j - LEAD) sum[x][r & 3] += __builtin_amdgcn_exp2f(fmaf(acc[x][r], a.scale, -b[x]));
            if (j == CH - 1) l[x] += (sum[x][0] + sum[x][1]) + (sum[x][2] + sum[x][3]);
        }
    };
    // keys that a query does not see, if there may be any among these 32
    auto hide = [&](f32x16_t (&acc)[ST], int k0, uint32_t there) __attribute__((always_inline)) {
        if (there == ~0u && k0 + 31 <= seen_all) return;
#pragma unroll
        for (int x = 0; x < ST; ++x) {
            const int last_seen = pos[x] - k0;           // (a mask in bits: the compiler makes branches of two conditions)
            const uint32_t seen = (there & (last_seen < 0 ? 0u : 0xffffffffu >> (31 - min(last_seen, 31)))) >> (4 * half);
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[x][r] = seen >> (8 * (r >> 2) + (r & 3)) & 1 ? acc[x][r] : -INFINITY;
        }
    };
    auto stay = [&]() __attribute__((always_inline)) {   // (the compiler would move the exponentials behind the branch that follows)
#pragma unroll
        for (int x = 0; x < ST; ++x) asm volatile("" : "+v"(m[x]), "+v"(l[x]));
    };
    f32x16_t acc[2][ST];
    nothing<ST>(acc[0]);
    nothing<ST>(acc[1]);
    int pending = 0;
    look_up(s0);
    load(std::integral_constant<int, 0>{});
    look_up(s0 + 1);
    if (s0 + 1 < s1) {
        load(std::integral_constant<int, 1>{});
        look_up(s0 + 2);
        arrived<LOADS>();
    } else {
        arrived<0>();
    }
#pragma unroll
    for (int j = 0; j < PT_RING; ++j) ring[j] = staged_piece(lds, at[j]);
    in_steps((s1 - s0) * TPS, [&](auto index, int t) __attribute__((always_inline)) {
        constexpr int I = decltype(index)::value, buf = I / TPS % PT_BUFS, y = I % TPS, nbuf = (I + 1) / TPS % PT_BUFS, ny = (I + 1) % TPS, now = I & 1;
        const int s = s0 + t / TPS, k0 = s * ROWS + 32 * y;
        if (y == TPS - 1 && s + 1 < s1) {                // the next stage is there, and nobody reads the one before this any more
            arrived<0>();
            if (s + 2 < s1) { load(std::integral_constant<int, (buf + 2) % PT_BUFS>{}); look_up(s + 3); }
        }
        if (k0 > seen_any) return;
        multiply_rows<CH, ST>(lds + buf * STAGE_BYTES + 32 * y * PPR * 16, lds + nbuf * STAGE_BYTES + 32 * ny * PPR * 16, at, ring, qf, acc[now],
                              [](const u32x4_t staged, const u32x4_t held, f32x16_t v) { return mma32<T>(staged, held, v); },
                              [&](int j) __attribute__((always_inline)) { add_up(acc[now ^ 1], j); });
        stay();
        hide(acc[now], k0, (uint32_t)(there[buf] >> (32 * y)));
        pending = now;
    });
#pragma unroll
    for (int j = 0; j < CH; ++j) {                       // the last tile's
        if (pending == 0) add_up(acc[0], j);
        else add_up(acc[1], j);
    }
#pragma unroll
    for (int x = 0; x < ST; ++x) {
        const float mx = lane_xor_max(m[x], 32), b = fmaxf(mx, -1e30f);
        const float sum = lane_xor_add(l[x] * __builtin_amdgcn_exp2f(fmaxf(m[x], -1e30f) - b), 32);
        const int i = i0 + 32 * x + c;
        if (!mine || half != 0 || i >= nq) continue;
        const size_t at = (size_t)h * tokens + tok0 + i;
        if (splits > 1) stats[(size_t)split * tokens * a.nh + at] = make_float2(mx, sum);
        else lse[at] = sum == 0.f ? INFINITY : (mx == -INFINITY ? 0.f : mx) + log2f(sum);
    }
}

// lse [nh, T] from the splits' statistics (rows of other segments hold what they hold and are not asked for).
__global__ __launch_bounds__(256) void mass_lse_kernel(const float2* __restrict__ stats, int splits, long rows, float* __restrict__ lse) {
    const long i = blockIdx.x * 256L + threadIdx.x;
    if (i >= rows) return;
    float m = -INFINITY, l = 0.f;
    for (int s = 0; s < splits; ++s) {
        const float2 v = stats[s * rows + i];
        const float mn = fmaxf(m, v.x), b = fmaxf(mn, -1e30f);
        l = l * exp2f(fmaxf(m, -1e30f) - b) + v.y * exp2f(fmaxf(v.x, -1e30f) - b);
        m = mn;
    }
    lse[i] = l == 0.f ? INFINITY : (m == -INFINITY ? 0.f : m) + log2f(l);
}

// The columns' sums: a wave holds ST * 32 keys, the block streams the queries that see any of them, head by head.
// grid: x kv heads times blocks of keys (of the longest segment), y splits of the (head, stage of queries) pairs, z segments.  A block of keys has
// as many splits as make about `share` pairs each: late keys are seen by few queries.
// part [splits, kv heads, places]; a segment's places begin at its `off`.
// The pairs of the block of keys from b0 on: its first stage of queries, stages a head, splits.
struct Pairs { int first, n, splits; };
__device__ __forceinline__ Pairs pairs_of(int b0, int base, int nq, int rep, int rows, int share) {
    const int first = max(b0 - base, 0) / rows, n = (nq + rows - 1) / rows - first;
    return {first, n, (rep * n + share - 1) / share};
}

template <typename T, int DHP, int ST>
__global__ __launch_bounds__(64 * PT_WAVES, DHP * sizeof(T) <= 256 ? 2 : 1) void mass_keys_tile_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, SegList list,
                                                                       const float* __restrict__ lse, float* __restrict__ part, int share, int tokens, long places) {
    constexpr int PE = 16 / sizeof(T), PPR = DHP / PE, CH = PPR / 2, TPS = stage_tiles(16 * PPR), ROWS = 32 * TPS, STAGE_BYTES = ROWS * PPR * 16, KEYS = 32 * ST;
    constexpr int LOADS = ROWS * PPR / (64 * PT_WAVES);
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int which = blockIdx.z, seg = list.of[which].seg, kvh = blockIdx.x % a.nkv, split = blockIdx.y;
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, half = lane >> 5;
    const int nq = list.of[which].q, ctx = list.of[which].ctx, base = ctx - nq, rep = a.nh / a.nkv, pieces = a.dh / PE, tok0 = list.of[which].start;
    const int b0 = blockIdx.x / a.nkv * KEYS * PT_WAVES, k0 = b0 + w * KEYS;
    if (b0 >= ctx) return;
    const Pairs pairs = pairs_of(b0, base, nq, rep, ROWS, share);
    if (split >= pairs.splits) return;
    const int* table = a.block_table + (size_t)seg * a.max_blocks;
    if (pieces < PPR) {
        for (int i = tid; i < PT_BUFS * STAGE_BYTES / 16; i += 64 * PT_WAVES) reinterpret_cast<u32x4_t*>(lds)[i] = u32x4_t{0, 0, 0, 0};
        __syncthreads();
    }
    u32x4_t kf[ST][CH];
#pragma unroll
    for (int x = 0; x < ST; ++x) {
        const T* src = k + some_row(a, table, kvh, min(k0 + 32 * x + c, ctx - 1)) * a.dh;
#pragma unroll
        for (int j = 0; j < CH; ++j) kf[x][j] = 2 * j + half < pieces ? *reinterpret_cast<const u32x4_t*>(src + (2 * j + half) * PE) : u32x4_t{0, 0, 0, 0};
    }
    f32x16_t sums[ST];
#pragma unroll
    for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) sums[x][r] = 0.f;
    // pairs (head, stage of queries), numbered head by head; this split's share of them
    const int first = pairs.first, n = pairs.n;
    const int u0 = (int)((long)rep * n * split / pairs.splits), u1 = (int)((long)rep * n * (split + 1) / pairs.splits);
    int lh = u0 / n, ls = first + u0 % n;                // the pair that is loaded next
    const uint32_t lds0 = lds_offset(lds), q_bytes = (uint32_t)a.q_row_stride * sizeof(T);
    uint32_t offset[LOADS];                              // of a lane's pieces from the stage's first row
    stage_rows<PPR, ROWS>(0, w, lane, [&](int i, int r, int p, uint32_t) __attribute__((always_inline)) { offset[i] = r * q_bytes + 16 * p; });
    float lq[PT_BUFS][TPS];                              // the queries' lse of the stages on their way, and where these begin
    int from[PT_BUFS];
    auto load = [&](auto which_buf) __attribute__((always_inline)) {
        constexpr int buf = decltype(which_buf)::value;
        const int i0 = ls * ROWS;
        const T* rows = q + (size_t)(tok0 + i0) * a.q_row_stride + (size_t)(kvh * rep + lh) * a.dh;
        const float* row_lse = lse + (size_t)(kvh * rep + lh) * tokens + tok0 + i0;
        from[buf] = i0;
        if (pieces == PPR && i0 + ROWS <= nq) {          // (whole rows, all of them there: no masks, whose branches cost more than the loads)
#pragma unroll
            for (int y = 0; y < TPS; ++y) lq[buf][y] = row_lse[32 * y + c];
            stage_rows<PPR, ROWS>(lds0 + buf * STAGE_BYTES, w, lane,
                                  [&](int i, int, int, uint32_t to) __attribute__((always_inline)) { load_to_lds(rows, offset[i], to); });
        } else {
#pragma unroll
            for (int y = 0; y < TPS; ++y) lq[buf][y] = i0 + 32 * y + c < nq ? row_lse[32 * y + c] : INFINITY;
            stage_rows<PPR, ROWS>(lds0 + buf * STAGE_BYTES, w, lane, [&](int, int r, int p, uint32_t to) __attribute__((always_inline)) {
                if (p < pieces) load_to_lds(rows, min(r, nq - 1 - i0) * q_bytes + 16 * p, to);
            });
        }
        if (++ls == first + n) { ls = first; ++lh; }
    };
    int at[CH];
    staged_at<PPR>(c, half, at);
    u32x4_t ring[PT_RING];
    auto add_up = [&](const f32x16_t (&acc)[ST], float lq, int j) __attribute__((always_inline)) {       // a tile's sums, in CH shares
#pragma unroll
        for (int x = 0; x < ST; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if ((16 * x + r) * CH / (16 * ST) == j) sums[x][r] += __builtin_amdgcn_exp2f(fmaf(acc[x][r], a.scale, -lq));
    };
    // a tile whose queries do not all see all the wave's keys is added up at once, and leaves nothing for later
    auto hide = [&](f32x16_t (&acc)[ST], float& lq, int q0) __attribute__((always_inline)) {
        if (base + q0 >= k0 + KEYS - 1 && q0 < nq) return;
        const int pos = base + q0 + c;
        if (q0 < nq && base + q0 + 31 >= k0)
#pragma unroll
            for (int x = 0; x < ST; ++x)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float e = __builtin_amdgcn_exp2f(fmaf(acc[x][r], a.scale, -lq));
                    sums[x][r] += k0 + 32 * x + 4 * half + 8 * (r >> 2) + (r & 3) <= pos ? e : 0.f;
                }
        nothing<ST>(acc);
        lq = 0.f;
    };
    auto stay = [&]() __attribute__((always_inline)) {   // (the compiler would move the exponentials behind the branch that follows)
#pragma unroll
        for (int x = 0; x < ST; ++x) asm volatile("" : "+v"(sums[x]));
    };
    f32x16_t acc[2][ST];
    float lacc[2] = {0.f, 0.f};
    nothing<ST>(acc[0]);
    nothing<ST>(acc[1]);
    if (u0 < u1) {
        load(std::integral_constant<int, 0>{});
        if (u0 + 1 < u1) {
            load(std::integral_constant<int, 1>{});
            arrived<LOADS>();
        } else {
            arrived<0>();
        }
#pragma unroll
        for (int j = 0; j < PT_RING; ++j) ring[j] = staged_piece(lds, at[j]);
    }
    const int steps = (u1 - u0) * TPS;
    in_steps(steps, [&](auto index, int t) __attribute__((always_inline)) {
        constexpr int I = decltype(index)::value, buf = I / TPS % PT_BUFS, y = I % TPS, nbuf = (I + 1) / TPS % PT_BUFS, ny = (I + 1) % TPS, now = I & 1;
        const int u = u0 + t / TPS;
        if (y == TPS - 1 && u + 1 < u1) {                // the next stage is there, and nobody reads the one before this any more
            arrived<0>();
            if (u + 2 < u1) load(std::integral_constant<int, (buf + 2) % PT_BUFS>{});
        }
        multiply_rows<CH, ST>(lds + buf * STAGE_BYTES + 32 * y * PPR * 16, lds + nbuf * STAGE_BYTES + 32 * ny * PPR * 16, at, ring, kf, acc[now],
                              [](const u32x4_t staged, const u32x4_t held, f32x16_t v) { return mma32<T>(held, staged, v); },
                              [&](int j) __attribute__((always_inline)) { add_up(acc[now ^ 1], lacc[now ^ 1], j); });
        stay();
        lacc[now] = lq[buf][y];
        hide(acc[now], lacc[now], from[buf] + 32 * y);
    });
#pragma unroll
    for (int j = 0; j < CH; ++j) {                       // the last tile's
        if (steps & 1) add_up(acc[0], lacc[0], j);
        else add_up(acc[1], lacc[1], j);
    }
    float* out = part + ((size_t)split * a.nkv + kvh) * places + list.of[blockIdx.z].off;
#pragma unroll
    for (int x = 0; x < ST; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            float v = sums[x][r];
            v = lane_xor_add(lane_xor_add(lane_xor_add(lane_xor_add(lane_xor_add(v, 16), 8), 4), 2), 1);
            const int t = k0 + 32 * x + 4 * half + 8 * (r >> 2) + (r & 3);
            if (c == 0 && t < ctx) out[t] = v;
        }
}

// The splits' sums, in their order, join the keys'.
__global__ __launch_bounds__(256) void mass_join_kernel(MassArgs a, SegList list, const float* __restrict__ part, int keys, int rows, int share, long places,
                                                        float* __restrict__ mass) {
    const int seg = list.of[blockIdx.z].seg, kvh = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x, ctx = list.of[blockIdx.z].ctx;
    if (t >= ctx) return;
    const long row = place_row(a, a.block_table + (size_t)seg * a.max_blocks, kvh, t);
    if (row < 0) return;
    const int nq = list.of[blockIdx.z].q, splits = pairs_of(t / keys * keys, ctx - nq, nq, a.nh / a.nkv, rows, share).splits;
    const float* src = part + (size_t)kvh * places + list.of[blockIdx.z].off + t;
    float sum = 0.f;
    for (int s = 0; s < splits; s += 4) {                // (four on their way at a time)
        float v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = s + i < splits ? src[(size_t)(s + i) * a.nkv * places] : 0.f;
        sum += (v[0] + v[1]) + (v[2] + v[3]);
    }
    mass[row] = a.fresh && t >= ctx - nq ? sum : mass[row] + sum;
}

// ---- the plan of a batch, from its segments in host memory: which kernels, how many splits, where things lie in the workspace
struct MassPlan {
    int single = 0, multi = 0;           // segments of one token, of more
    int device_ctx = 0, multi_ctx = 0, multi_q = 0;
    int parts = 0, block_lds = 0;        // runs of 64 keys of the longest of them
    bool one_block = false;              // short contexts of single tokens: one kernel
    bool listed = false;                 // single tokens are named in the launch, with their lengths
    int row_splits = 1, key_splits = 1, row_st = 1, key_st = 1, row_share = 1, key_share = 1, stage = 64;      // (shares: stages, pairs)
    long places = 0;                     // of the longer segments' sums, all together
    long rows = 0, lse = 0, sums = 0, floats = 0;                              // offsets, and the whole (single tokens' scores lie first)
    bool tiled = false, valid = false;
};

struct Batch { const int *q_start, *q_len, *ctx_len; };      // in host memory

// (the tiles' loads count pieces of 16 bytes in 32 bits, and bytes of 64 rows)
static bool tiled_takes(int dtype, int dh, int q_row_stride, const void* q, const void* k, float scale, long tokens, long nh, long rows) {
    const int es = dtype == LI_BF16 ? 2 : 4;
    return tokens * (q_row_stride * (long)es / 16) < 1L << 32 && 64L * q_row_stride * es < 1L << 32 && rows * (dh * es / 16) < 1L << 32 && tokens * nh < 1L << 31 && dh * es % 16 == 0 && q_row_stride * (long)es % 16 == 0 && ((uintptr_t)q | (uintptr_t)k) % 16 == 0 && scale > 0.f && scale < INFINITY;
}

// Places of a segment's sums: whole blocks of keys.
static long places_of(int ctx) { return (ctx + 64 * PT_WAVES - 1) / (64 * PT_WAVES) * (64L * PT_WAVES); }

// The requests of the next launch of single tokens, from segment i on (which moves behind them): as many as a list and SG_ROOM hold.
struct Singles { int n, parts; long floats; };
static Singles next_singles(const int* q_len, const int* ctx_len, int nseg, int nh, int& i, SegList* list = nullptr, const int* q_start = nullptr) {
    Singles s = {0, 0, 0};
    for (; i < nseg && s.n < EV_LIST; ++i) {
        if (q_len[i] != 1) continue;
        const int parts = (ctx_len[i] + SG_KEYS - 1) / SG_KEYS;
        const long mine = single_floats(nh, parts);
        if (s.n && s.floats + mine > SG_ROOM) break;
        if (list) list->of[s.n] = {i, q_start[i], 1, ctx_len[i], (int)s.floats};
        s.parts = std::max(s.parts, parts);
        s.floats += mine;
        ++s.n;
    }
    if (list) list->n = s.n;
    return s;
}
// The same where the lengths are read on the device: up to `left` requests of `parts` runs each.
static Singles next_singles(int left, int parts, int nh) {
    const long mine = single_floats(nh, parts);
    const int n = (int)std::min((long)left, std::max(SG_ROOM / mine, 1L));
    return {n, parts, n * mine};
}

static MassPlan mass_plan(const int* q_len, const int* ctx_len, int nseg, int tokens, int padded_ctx, int nh, int nkv, int dh, bool f32, bool tiled) {
    MassPlan p;
    long total = 0;
    for (int i = 0; i < nseg; ++i) {
        const int ctx = padded_ctx > 0 ? padded_ctx : ctx_len[i];
        if (q_len[i] <= 0 || ctx < q_len[i]) return p;
        total += q_len[i];
        if (q_len[i] == 1 && tiled) {
            ++p.single;
            p.device_ctx = ctx > p.device_ctx ? ctx : p.device_ctx;
        } else {
            ++p.multi;
            p.multi_ctx = ctx > p.multi_ctx ? ctx : p.multi_ctx;
            p.multi_q = q_len[i] > p.multi_q ? q_len[i] : p.multi_q;
            p.places += places_of(ctx);
        }
    }
    if (total != tokens || p.places >= 1L << 31) return p;
    p.valid = true;
    p.tiled = tiled;
    const int rep = nh / nkv;
    if (!tiled) { p.floats = (long)tokens * nh; return p; }
    if (p.single) {
        p.parts = (p.device_ctx + SG_KEYS - 1) / SG_KEYS;
        const long lds = 4 * (rep * (SG_KEYS + 2L) * p.parts + rep);
        // One kernel where a block has few keys, or where the blocks fill the compute units, us: bfloat16, 28 heads on 4 of 128, one request of 300 keys 9.0
        // (two kernels) and 6.8, 64 requests 13.3 and 7.1, of 1,000 20.0 and 14.8, of 2,000 32.5 and 25.6; 8 requests of 1,000 9.4 and 12.8, 64
        // of 2,000 on 2 kv heads 20.3 and 23.5.  Recorded steps are asked about the tables' room, not the contexts; one kernel and two, us: 28 heads on 4, one
        // request of 500 in 512 places 8.7 and 9.6, of 1,000 in 1,024 13.0 and 9.6, 64 of 1,000 in 1,024 16.5 and 23.1, of 2,000 in 2,048 32.4 and 41.5; 8 of 1,000 in 1,024 14.0
        // and 10.8; 12 heads on 2 (128 blocks: two kernels), 64 of 1,100 in 2,048 15.8 and 20.0, of 2,000 25.1 and 22.0.
        p.one_block = lds <= 150 * 1024 && (p.device_ctx <= 512 || ((long)p.single * nkv >= 192 && p.device_ctx <= 2048));
        p.block_lds = (int)lds;
        // a mix, or few: they are named, and their lengths need no trip to memory
        p.listed = padded_ctx <= 0 && (p.single < nseg || nseg <= EV_LIST);
        if (!p.one_block && !p.listed) p.floats = next_singles(p.single, p.parts, nh).floats;
        if (!p.one_block && p.listed)
            for (int i = 0; i < nseg;) p.floats = std::max(p.floats, next_singles(q_len, ctx_len, nseg, nh, i).floats);
    }
    if (p.multi) {
        // Blocks of about equal length: as many as the compute units hold at a time, each with no less than 8 stages of keys (4 pairs of a head and a stage
        // of queries), or, where there is work for many rounds, 96 stages (40 or 80 pairs) each.  A wave holds two tiles where that leaves blocks of
        // some length, else one, and there are more of them.  Rows: two from 16 stages a block on.  Keys: two from 20 pairs a block on; one and two, us of both
        // passes: a prompt of 2,048 of 28 heads on 4 79 and 87, of 512 of 14 heads on 2 21 and 26, 990 of 12 heads on 2 behind 500 33 and 36, 4 x 512 of 28
        // heads behind 1,000 68 and 78 (8 to 14 pairs); 2,048 behind 2,000 149 and 149 (21); a prompt of 4,000 of 28 heads 195 and 191 (28), 2,048 behind
        // 8,000 375 and 334, 1,999 of 40 heads on 8 behind 16,000 850 and 788 (166).  float32, whose rows take twice the registers: one tile always; one and two, us of both
        // passes: a prompt of 2,048 of 28 heads on 4 of 128 379 and 470, 512 of 14 heads on 2 of 64 behind 2,048 73 and 98, 2,048 of the same behind 8,192 691 and 736, but 512 of 28
        // heads behind 4,096 377 and 312.
        const int rows = 32 * stage_tiles((dh <= 64 ? 64 : dh <= 128 ? 128 : 256) * (f32 ? 4 : 2));
        for (p.row_st = f32 ? 1 : 2;; p.row_st = 1) {
            long stages = 0, most = 0, all = 0;
            for (int i = 0; i < nseg; ++i) {
                if (q_len[i] < 2) continue;
                const long tiles = (q_len[i] + 32 * p.row_st - 1) / (32 * p.row_st), blocks = (tiles * rep + PT_WAVES - 1) / PT_WAVES;
                all += blocks * nkv;
                stages += blocks * nkv * ((ctx_len[i] - q_len[i] / 2 + rows - 1) / rows);
                most = std::max(most, (long)(ctx_len[i] + rows - 1) / rows);
            }
            const long one = p.row_st == 2 || f32 ? 512 : 768;
            // (a block's last share is half a share on average)
            const long fit = 2 * one > all ? (2 * stages + 2 * one - all - 1) / (2 * one - all) : 96;
            p.row_share = (int)std::min(std::max(fit, 8L), 96L);
            p.row_share = (int)std::max((long)p.row_share, (most + 511) / 512);
            p.row_splits = (int)((most + p.row_share - 1) / p.row_share);
            if (p.row_st == 1 || stages >= one * 16) break;
        }
        for (p.key_st = f32 ? 1 : 2;; p.key_st = 1) {
            const int keys = 32 * PT_WAVES * p.key_st;
            const long one = p.key_st == 2 || f32 ? 512 : 768;
            long units = 0;
            for (int i = 0; i < nseg; ++i) {
                if (q_len[i] < 2) continue;
                const long n = (q_len[i] + rows - 1) / rows, base = ctx_len[i] - q_len[i];
                units += (long)nkv * rep * (base / keys * n + ((ctx_len[i] + keys - 1) / keys - base / keys) * (n + 1) / 2);
            }
            p.key_share = (int)std::min(std::max((units + one - 1) / one, 4L), p.key_st == 2 || f32 ? 40L : 80L);
            if (p.key_st == 1 || units >= one * 20) break;
        }
        const long longest = (long)rep * ((p.multi_q + rows - 1) / rows);
        p.key_share = (int)std::max((long)p.key_share, (longest + 32767) / 32768);
        p.key_splits = (int)((longest + p.key_share - 1) / p.key_share);
        p.stage = rows;
        p.rows = p.floats;
        p.lse = p.rows + 2L * p.row_splits * tokens * nh;
        p.sums = p.lse + (long)tokens * nh;
        p.floats = p.sums + (long)p.key_splits * nkv * p.places;
    }
    return p;
}

// Floats of workspace for a batch (its segments in host memory); -1: not a batch.  padded_ctx > 0: a batch that is recorded and replayed
// for any contexts up to that.  q, k: the addresses, whose alignment decides on the kernel; rows: pages * nkv * page_size.
extern "C" long li_attention_mass_work_floats(const int* q_len, const int* ctx_len, int nseg, int tokens, int padded_ctx, int nh, int nkv, int dh, int dtype,
                                              int q_row_stride, const void* q, const void* k, float scale, long rows) {
    if (nseg <= 0 || tokens <= 0 || nh <= 0 || nkv <= 0 || nh % nkv || !q_len || !ctx_len) return -1;
    const MassPlan p = mass_plan(q_len, ctx_len, nseg, tokens, padded_ctx, nh, nkv, dh, dtype == LI_F32, tiled_takes(dtype, dh, q_row_stride, q, k, scale, tokens, nh, rows));
    return p.valid ? (p.floats > 0 ? p.floats : 1) : -1;
}

template <typename K>
static bool allow_lds(K kernel, int bytes) {
    return bytes <= 64 * 1024 || hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes) == hipSuccess;
}

template <typename T, int DHP>
static int launch_mass_tiled(const T* q, const T* k, float* mass, const MassArgs& a, const MassPlan& p, const Batch& b,
                             int nseg, int tokens, float* work, hipStream_t stream) {
    constexpr int PE = 16 / sizeof(T), CH16 = DHP / (4 * PE), ST = sizeof(T) == 2 ? 2 : 1;
    constexpr int LDS_BYTES = PT_BUFS * 32 * stage_tiles(DHP * (int)sizeof(T)) * DHP * (int)sizeof(T);
    if (p.single) {
        for (int at = 0, i = 0; at < p.single;) {
            SegList list;
            list.n = 0;
            const Singles now = p.listed ? next_singles(b.q_len, b.ctx_len, nseg, a.nh, i, &list, b.q_start)
                                : p.one_block ? Singles{p.single, p.parts, 0} : next_singles(p.single - at, p.parts, a.nh);
            if (p.one_block) {
                const auto block = mass_single_block_kernel<T, CH16>;
                if (!allow_lds(block, p.block_lds)) return LI_ERR_LAUNCH;
                block<<<dim3(a.nkv, now.n), 64 * block_waves(CH16), p.block_lds, stream>>>(q, k, a, list, p.parts * SG_KEYS, mass);
            } else {
                mass_single_scores_kernel<T, CH16><<<dim3((now.parts + SG_WAVES - 1) / SG_WAVES, a.nkv, now.n), 64 * SG_WAVES, 0, stream>>>(
                    q, k, a, list, work, single_floats(a.nh, now.parts), at, now.parts);
                mass_single_add_kernel<<<dim3((now.parts + 3) / 4, a.nkv, now.n), 256, 0, stream>>>(a, list, work, single_floats(a.nh, now.parts), at, now.parts, mass);
            }
            at += now.n;
        }
    }
    if (p.multi) {
        const auto rows = p.row_st == ST ? mass_rows_tile_kernel<T, DHP, ST> : mass_rows_tile_kernel<T, DHP, 1>;
        const auto keys = p.key_st == ST ? mass_keys_tile_kernel<T, DHP, ST> : mass_keys_tile_kernel<T, DHP, 1>;
        const int keys_block = 32 * PT_WAVES * p.key_st;
        if (!allow_lds(rows, LDS_BYTES) || !allow_lds(keys, LDS_BYTES)) return LI_ERR_LAUNCH;
        const int rep = a.nh / a.nkv, tiles = (p.multi_q + 32 * p.row_st - 1) / (32 * p.row_st);
        float2* stats = (float2*)(work + p.rows);
        float *lse = work + p.lse, *sums = work + p.sums;
        const long rows_n = (long)tokens * a.nh;
        for (int pass = 0; pass < 2; ++pass) {
            long off = 0;
            for (int at = 0, i = 0; at < p.multi;) {
                SegList list;
                int n = 0;
                for (; i < nseg && n < EV_LIST; ++i)
                    if (b.q_len[i] > 1) {
                        list.of[n++] = {i, b.q_start[i], b.q_len[i], b.ctx_len[i], (int)off};
                        off += places_of(b.ctx_len[i]);
                    }
                list.n = n;
                at += n;
                if (pass == 0) {
                    rows<<<dim3((tiles * rep + PT_WAVES - 1) / PT_WAVES * a.nkv, 1, n * p.row_splits), 64 * PT_WAVES, LDS_BYTES, stream>>>(
                        q, k, a, list, stats, lse, p.row_splits, p.row_share, tokens);
                } else {
                    keys<<<dim3((p.multi_ctx + keys_block - 1) / keys_block * a.nkv, p.key_splits, n), 64 * PT_WAVES, LDS_BYTES, stream>>>(
                        q, k, a, list, lse, sums, p.key_share, tokens, p.places);
                    mass_join_kernel<<<dim3((p.multi_ctx + 255) / 256, a.nkv, n), 256, 0, stream>>>(a, list, sums, keys_block, p.stage, p.key_share, p.places, mass);
                }
            }
            if (pass == 0 && p.row_splits > 1) mass_lse_kernel<<<(unsigned)((rows_n + 255) / 256), 256, 0, stream>>>(stats, p.row_splits, rows_n, lse);
        }
    }
    return li_launch_status();
}

template <typename T>
static int launch_mass(const T* q, const T* k, float* mass, const MassArgs& a, const MassPlan& p, const Batch& b, int nseg, int tokens,
                       float* work, hipStream_t stream) {
    if (p.tiled && a.dh <= 64) return launch_mass_tiled<T, 64>(q, k, mass, a, p, b, nseg, tokens, work, stream);
    if (p.tiled && a.dh <= 128) return launch_mass_tiled<T, 128>(q, k, mass, a, p, b, nseg, tokens, work, stream);
    if (p.tiled) return launch_mass_tiled<T, 256>(q, k, mass, a, p, b, nseg, tokens, work, stream);
    mass_rows_kernel<T><<<dim3(p.multi_q, a.nh, nseg), 64, 0, stream>>>(q, k, a, work);
    mass_keys_kernel<T><<<dim3((p.multi_ctx + 63) / 64, a.nkv, nseg), 256, 0, stream>>>(q, k, a, work, mass);
    return li_launch_status();
}

// q_start, q_len, ctx_len: the batch's segments on the device; those with h_ the same in host memory.  padded_ctx > 0: the contexts may be others
// when a recording is replayed, up to that; then every segment brings one token.  work: li_attention_mass_work_floats of the same batch
// (no fewer than are found to be wanted: a batch that was changed since is refused).
extern "C" int li_attention_mass(const void* q, int q_row_stride, const void* kc, float* mass, int dtype, const int* block_table, int max_blocks,
                                 const int* q_start, const int* q_len, const int* ctx_len, const int* h_q_start, const int* h_q_len,
                                 const int* h_ctx_len, int nseg, int tokens,
                                 int padded_ctx, int nh, int nkv, int dh, int page_size, int num_pages, float scale, int fresh, float* work,
                                 long work_floats, hipStream_t stream) {
    if (nseg <= 0 || nseg > 65535 || tokens <= 0 || nh <= 0 || nh > 65535 || nkv <= 0 || nkv > 4095 || nh % nkv || dh <= 0 || dh > EV_MAX_DH || page_size <= 0 ||
        max_blocks <= 0 || (long)max_blocks * page_size > EV_MAX_PLACES || num_pages <= 0 ||
        (long)num_pages * nkv * page_size >= 1L << 31 || !h_q_start || !h_q_len || !h_ctx_len || !work)
        return LI_ERR_SIZE;
    const long room = (long)max_blocks * page_size;
    for (int i = 0; i < nseg; ++i)
        if (h_ctx_len[i] > room || h_q_start[i] < 0 || (long)h_q_start[i] + h_q_len[i] > tokens || (padded_ctx > 0 && (h_q_len[i] != 1 || padded_ctx > room))) return LI_ERR_SIZE;
    if (dtype != LI_F32 && dtype != LI_BF16) return LI_ERR_DTYPE;
    const MassArgs a = {block_table, q_start, q_len, ctx_len, max_blocks, nh, nkv, dh, page_size, num_pages, q_row_stride,
                        inverse_of(page_size), scale * 1.44269504088896341f, fresh};
    const MassPlan p = mass_plan(h_q_len, h_ctx_len, nseg, tokens, padded_ctx, nh, nkv, dh, dtype == LI_F32, tiled_takes(dtype, dh, q_row_stride, q, kc, scale, tokens, nh, (long)num_pages * nkv * page_size));
    if (!p.valid || p.floats > work_floats) return LI_ERR_SIZE;
    const Batch b = {h_q_start, h_q_len, h_ctx_len};
    if (dtype == LI_F32) return launch_mass((const float*)q, (const float*)kc, mass, a, p, b, nseg, tokens, work, stream);
    return launch_mass((const bf16_t*)q, (const bf16_t*)kc, mass, a, p, b, nseg, tokens, work, stream);
}

// ------------------------------------------------------------------ which keys stay
// unsigned integers in the order of the floats; -0 counts as 0, NaN as less than everything
__device__ __forceinline__ uint32_t mass_order(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

struct SelectArgs {
    const float* mass;
    const int *block_table, *lens, *keeps;
    int max_blocks, first, recent, K, nkv, page_size, num_pages;
    uint32_t page_inv;
    int* out;
    int fours;                   // four places side by side lie in one page, on 16 bytes
};

// Places lo .. hi - 1 of a request compete for `want` of its places; the others of its `len` stay anyway.
struct Contest { int len, lo, hi, want; };
__device__ __forceinline__ Contest contest_of(const SelectArgs& a, int req) {
    const int len = (int)min((long)max(a.lens[req], 0), (long)a.max_blocks * a.page_size);
    const int keep = min(min(max(a.keeps[req], 0), len), a.K), recent = min(a.recent, keep), first = min(a.first, keep - recent);
    return {len, first, len - recent, keep - recent - first};
}
// A place's sum in the order of the floats; 0, as little as there is, where no page holds it.
__device__ __forceinline__ int page_of(const SelectArgs& a, int t) {
    const int p = (int)__umulhi((uint32_t)t, a.page_inv);
    return p + (t - p * a.page_size >= a.page_size ? 1 : 0);
}
__device__ __forceinline__ uint32_t place_key(const SelectArgs& a, const float* pool, const int* table, int kvh, int t) {
    const int p = page_of(a, t), page = table[p];
    return page < 0 || page >= a.num_pages ? 0u : mass_order(pool[((size_t)page * a.nkv + kvh) * a.page_size + t - p * a.page_size]);
}

// The sum of the threads' v before this one, and of all of them.  NT threads; smem has a place a wave.
template <int NT>
__device__ __forceinline__ int block_before(int v, int* smem, int& all) {
    constexpr int W = NT / 64;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int up = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(up, o, 64);
        if (lane >= o) up += x;
    }
    __syncthreads();
    if (lane == 63) smem[w] = up;
    __syncthreads();
    int before = up - v;
    all = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) {
        const int x = smem[i];
        if (i < w) before += x;
        all += x;
    }
    return before;
}

// A block a (entry, request, kv head), a thread VPT places side by side, whose sums it keeps.  The least sum that is taken is found digit by
// digit: 256 equal parts of the range between the contest's least and its largest are counted in LDS, then those of the part in which the least
// taken sum lies, and so on, until all of a part is taken or it is a single value, of whose places the lowest are taken.  (Equal parts of
// the floats' order, not their leading bits: sums lie within a few octaves, and would meet in a few counters.)
// Bound by that chain, two trips to memory and eight to twelve barriers, not by the 4 bytes a place: 8 requests of 2,500 to 4,096 places x 28 entries x 4 kv heads (19 MB)
// 16.2 us, 8 entries x 8 kv heads of 32,000 (9 MB) 26.6.  (Halving by ballots of a bit a time took 35 and 56.)
template <int NT, int VPT>
__global__ __launch_bounds__(NT) void evict_select_kernel(SelectArgs a) {
    constexpr int W = NT / 64;
    // Counters are kept apart for every CP-th lane, where there are many sums: those of one part wait for each other.  (1,024 x 32 places with 1, 2, 4 and 8
    // copies 29.5, 27.8, 26.7 and 26.8 us; 512 x 8 with 1, 2 and 8 16.6, 16.4 and 21.1.)
    constexpr int CP = VPT >= 32 ? 4 : 1;
    __shared__ __attribute__((aligned(16))) int counts[256 * CP];
    __shared__ int waves[W], part[3];
    __shared__ uint32_t ends[2][W];
    const int kvh = blockIdx.x, req = blockIdx.y, entry = blockIdx.z, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int* table = a.block_table + (size_t)req * a.max_blocks;
    const float* pool = a.mass + (size_t)entry * a.num_pages * a.nkv * a.page_size;
    int* dst = a.out + (((size_t)entry * gridDim.y + req) * a.nkv + kvh) * a.K;
    const Contest c = contest_of(a, req);
    const bool choose = c.want > 0 && c.want < c.hi - c.lo;
    const int t0 = tid * VPT;
    uint32_t taken = 0;                                   // bit j: place t0 + j stays
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
        const int t = t0 + j;
        if (t < c.len && (t < c.lo || t >= c.hi || (!choose && c.want > 0))) taken |= 1u << j;
    }
    if (choose) {
        uint32_t key[VPT];                                // 1 + the order of the sums that compete, 0 for the other places
        float sum[VPT];
        const int last = c.len - 1;
        if (a.fours) {
            int at[VPT / 4];
#pragma unroll
            for (int j = 0; j < VPT / 4; ++j) at[j] = table[page_of(a, min(t0 + 4 * j, last))];
#pragma unroll
            for (int j = 0; j < VPT / 4; ++j) {
                const int t = min(t0 + 4 * j, last) & ~3;
                const bool there = at[j] >= 0 && at[j] < a.num_pages;
                const f32x4_t v = *reinterpret_cast<const f32x4_t*>(pool + ((size_t)(there ? at[j] : 0) * a.nkv + kvh) * a.page_size + t - page_of(a, t) * a.page_size);
#pragma unroll
                for (int i = 0; i < 4; ++i) sum[4 * j + i] = there ? v[i] : NAN;
            }
        } else {
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const int t = min(t0 + j, last), p = page_of(a, t), page = table[p];
                const bool there = page >= 0 && page < a.num_pages;
                const float v = pool[((size_t)(there ? page : 0) * a.nkv + kvh) * a.page_size + t - p * a.page_size];
                sum[j] = there ? v : NAN;
            }
        }
        uint32_t least = ~0u, most = 0;
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const int t = t0 + j;
            const bool competes = t >= c.lo && t < c.hi;
            key[j] = competes ? mass_order(sum[j]) + 1 : 0u;         // (the order's largest, a NaN of the other sign, does not occur)
            least = min(least, competes ? key[j] : ~0u);
            most = max(most, key[j]);
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) {
            least = min(least, (uint32_t)lane_xor((int)least, o));
            most = max(most, (uint32_t)lane_xor((int)most, o));
        }
        if (lane == 0) { ends[0][w] = least; ends[1][w] = most; }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < W; ++i) { least = min(least, ends[0][i]); most = max(most, ends[1][i]); }
        uint32_t from = least, span = most - least;       // keys from .. from + span are looked at: all before are not taken, all behind are
        int left = c.want, held = 0;                      // how many of these are taken; how many they are
        for (;;) {
            const int shift = max(24 - __clz(span | 1), 0);
            for (int i = tid; i < 256 * CP; i += NT) counts[i] = 0;
            __syncthreads();
#pragma unroll
            for (int j = 0; j < VPT; ++j) {
                const uint32_t d = key[j] - from;         // (a key of 0 lies far behind)
                if (d <= span) atomicAdd(&counts[(d >> shift) * CP + lane % CP], 1);
            }
            __syncthreads();
            if (w == 0) {                                 // from the last part down: the first at which `left` are reached
                int n4[4] = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int y = 0; y < CP; ++y) n4[i] += counts[(255 - i - 4 * lane) * CP + y];
                const int four = (n4[0] + n4[1]) + (n4[2] + n4[3]);
                int up = four;
#pragma unroll
                for (int o = 1; o < 64; o <<= 1) {
                    const int x = __shfl_up(up, o, 64);
                    if (lane >= o) up += x;
                }
                int above = up - four;                    // in the parts before the lane's own
                if (above < left && left <= up) {
                    int p = 255 - 4 * lane, n = n4[0];
#pragma unroll
                    for (int i = 1; i < 4; ++i)
                        if (above + n < left) { above += n; --p; n = n4[i]; }
                    part[0] = p; part[1] = above; part[2] = n;
                }
            }
            __syncthreads();
            left -= part[1];
            held = part[2];
            from += (uint32_t)part[0] << shift;
            span = min((1u << shift) - 1, most - from);   // (no further than the largest: a key of 0 would be among the next)
            if (left == held || shift == 0) break;
        }
        // all above the part, and of the part all, or, where it is one value, the lowest `left` places
        int rank = 0, all;
        if (left != held) {
            int mine = 0;
#pragma unroll
            for (int j = 0; j < VPT; ++j) mine += key[j] == from ? 1 : 0;
            rank = block_before<NT>(mine, waves, all);
        }
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            const bool part_of = key[j] >= from && key[j] - from <= span;
            if (key[j] > from && !part_of) taken |= 1u << j;
            if (part_of && (left == held || rank++ < left)) taken |= 1u << j;
        }
    }
    int all;
    int rank = block_before<NT>(__popc(taken), waves, all);
#pragma unroll
    for (int j = 0; j < VPT; ++j)
        if (taken >> j & 1) {
            if (rank < a.K) dst[rank] = t0 + j;
            ++rank;
        }
    for (int r = all + tid; r < a.K; r += NT) dst[r] = -1;
}

#define SEL_NT 1024

// Requests that are longer than a block's registers: the sums are read again for every digit, eight bits of them, the digits counted in LDS.  (The digits are
// the leading bits of the floats' order, of which sums within a few octaves share most: many lanes add to one counter.)  Bound by that and by five
// passes of one block over the list: one request of 40,000 places, 8 entries x 8 kv heads 156 us, of 130,000 599; 28 x 4 208 and 601.
__global__ __launch_bounds__(SEL_NT) void evict_select_long_kernel(SelectArgs a) {
    __shared__ int hist[256], wsum[SEL_NT / 64], pick[2];
    const int kvh = blockIdx.x, req = blockIdx.y, entry = blockIdx.z, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int* table = a.block_table + (size_t)req * a.max_blocks;
    const float* pool = a.mass + (size_t)entry * a.num_pages * a.nkv * a.page_size;
    int* dst = a.out + (((size_t)entry * gridDim.y + req) * a.nkv + kvh) * a.K;
    const Contest c = contest_of(a, req);
    uint32_t prefix = 0, known = 0;
    int left = c.want;                                   // how many are still to be taken among those with the prefix
    const bool all = c.want >= c.hi - c.lo;
    if (c.want > 0 && !all)
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int t = c.lo + tid; t < c.hi; t += SEL_NT) {
                const uint32_t u = place_key(a, pool, table, kvh, t);
                if ((u & known) == prefix) atomicAdd(&hist[(u >> shift) & 255], 1);
            }
            __syncthreads();
            if (tid == 0) {
                int b = 255, n = left;
                for (; b > 0 && hist[b] < n; --b) n -= hist[b];
                pick[0] = b;
                pick[1] = n;
            }
            __syncthreads();
            prefix |= (uint32_t)pick[0] << shift;
            known |= 255u << shift;
            left = pick[1];
        }
    int at = 0, ties = 0;                                // places written, places equal to the last one taken
    for (int t0 = 0; t0 < c.len; t0 += SEL_NT) {
        const int t = t0 + tid;
        bool in = false, tie = false;
        if (t < c.len) {
            if (t < c.lo || t >= c.hi || all) in = true;
            else if (c.want > 0) {
                const uint32_t u = place_key(a, pool, table, kvh, t);
                in = u > prefix;
                tie = u == prefix;
            }
        }
        const uint64_t tb = __ballot(tie), below = (1ull << lane) - 1;
        __syncthreads();
        if (lane == 0) wsum[w] = __popcll(tb);
        __syncthreads();
        int rank = ties + __popcll(tb & below);
        for (int i = 0; i < SEL_NT / 64; ++i) {
            if (i < w) rank += wsum[i];
            ties += wsum[i];
        }
        if (tie && rank < left) in = true;
        const uint64_t ib = __ballot(in);
        __syncthreads();
        if (lane == 0) wsum[w] = __popcll(ib);
        __syncthreads();
        int pos = at + __popcll(ib & below);
        for (int i = 0; i < SEL_NT / 64; ++i) {
            if (i < w) pos += wsum[i];
            at += wsum[i];
        }
        if (in && pos < a.K) dst[pos] = t;
    }
    for (int j = at + tid; j < a.K; j += SEL_NT) dst[j] = -1;
}

// mass [entries, num_pages, nkv, page_size]; lens, keeps [n]; out [entries, n, nkv, K], ascending, -1 behind the last.
extern "C" int li_evict_select(const float* mass, const int* block_table, int max_blocks, const int* lens, const int* keeps, int n, int first, int recent,
                               int* out, int K, int entries, int nkv, int page_size, int num_pages, hipStream_t stream) {
    if (n <= 0 || n > 65535 || entries <= 0 || entries > 65535 || nkv <= 0 || K <= 0 || K > EV_MAX_PLACES || first < 0 || recent < 0 || max_blocks <= 0 || num_pages <= 0 || page_size <= 0 ||
        (long)max_blocks * page_size > EV_MAX_PLACES)
        return LI_ERR_SIZE;
    const SelectArgs a = {mass, block_table, lens, keeps, max_blocks, first, recent, K, nkv, page_size, num_pages, inverse_of(page_size), out,
                          page_size % 4 == 0 && (uintptr_t)mass % 16 == 0};
    const long room = (long)max_blocks * page_size;      // (as long as any request can be; the tables say no more)
    const dim3 grid(nkv, n, entries);
    // (More threads with fewer places each until their barriers cost more; us: 8 requests of 4,000 x 28 entries x 4 heads with 256, 512 and 1,024 threads
    // 18.8, 16.5 and 24.5, of 1,000 8.3, 13.8 and 20.8; of 16,000 with 512 and 1,024 63 and 79, but 19.0 and 17.3 where each has a compute unit to itself.)
    if (room <= 1024) evict_select_kernel<256, 4><<<grid, 256, 0, stream>>>(a);
    else if (room <= 4096) evict_select_kernel<512, 8><<<grid, 512, 0, stream>>>(a);
    else if (room <= 16384 && (long)entries * n * nkv > 256) evict_select_kernel<512, 32><<<grid, 512, 0, stream>>>(a);
    else if (room <= 16384) evict_select_kernel<1024, 16><<<grid, 1024, 0, stream>>>(a);
    else if (room <= 32768) evict_select_kernel<1024, 32><<<grid, 1024, 0, stream>>>(a);
    else evict_select_long_kernel<<<grid, SEL_NT, 0, stream>>>(a);
    return li_launch_status();
}

// ------------------------------------------------------------------ the kept rows move to the front
#define CMP_NT 256
#define CMP_U 4                   // pieces of a thread that move at a time
#define CMP_LIST 2048             // rows whose addresses lie in LDS
#define CMP_MAX_TENSORS 4

struct CompactTensors {
    void* data[CMP_MAX_TENSORS];
    int pieces[CMP_MAX_TENSORS];         // pieces of a row
    int wide[CMP_MAX_TENSORS];           // a piece is 16 bytes, else 4
    uint32_t inv[CMP_MAX_TENSORS];       // 2^32 / pieces
};

// kept is ascending, so kept[j] >= j: rows that are read lie at or behind those that are written, and rows of a later chunk behind
// all that an earlier one writes.  So a chunk's rows may be asked for any time before, and have to have arrived, for all threads, before it is
// written: the chunk behind is on its way while one waits at the barrier and is written.  Where a row stays, or has no page, nothing is written.
// Bound by memory: 8 requests of 2,500 to 4,096 cut to 2,048, 28 entries, 4 kv heads, keys and values of 128 bfloat16 and the sums (1.9 GB read and written) 394 to 431 us,
// 4.4 to 4.8 TB/s where a large copy gets 4.7.
template <typename V>
__device__ __forceinline__ void compact_rows(V* __restrict__ data, int pieces, uint32_t inv, const int* __restrict__ kept, int K, const int* __restrict__ table,
                                             int max_blocks, int kvh, int nkv, int page_size, uint32_t page_inv, int num_pages,
                                             int* from, int* to) {
    const int tid = threadIdx.x;
    const long room = (long)max_blocks * page_size;
    auto row_of = [&](int t) -> int {
        int p = (int)__umulhi((uint32_t)t, page_inv), rest = t - p * page_size;
        if (rest >= page_size) { ++p; rest -= page_size; }
        const int page = table[p];
        return page < 0 || page >= num_pages ? -1 : (page * nkv + kvh) * page_size + rest;
    };
    // a thread's pieces of a chunk of whole rows: row and piece of the row are the same in every chunk
    const int rows = max(CMP_NT * CMP_U / pieces, 1), spread = rows * pieces;
    int row[CMP_U], piece[CMP_U];
#pragma unroll
    for (int u = 0; u < CMP_U; ++u) {
        const int p = tid + CMP_NT * u;
        int r = (int)__umulhi((uint32_t)p, inv);
        if (p - r * pieces >= pieces) ++r;
        row[u] = p < spread ? r : CMP_LIST;               // (none)
        piece[u] = p - r * pieces;
    }
    for (int j0 = 0; j0 < K; j0 += CMP_LIST) {
        const int n = min(K - j0, CMP_LIST);
        __syncthreads();
        bool any = false;
        for (int j = tid; j < n; j += CMP_NT) {
            const int src = kept[j0 + j];
            any |= src >= 0;
            int a = -1, b = -1;
            if (src > j0 + j && src < room) {             // (not the list's end, nor a row that stays)
                a = row_of(src);
                b = row_of(j0 + j);
            }
            from[j] = a < 0 || b < 0 ? -1 : a;
            to[j] = b;
        }
        if (!__syncthreads_or(any)) return;
        V v[2][CMP_U];
        auto load = [&](V (&x)[CMP_U], int first) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < CMP_U; ++u) {
                const int r = first + row[u], a = r < n ? from[r] : -1;
                x[u] = data[(size_t)max(a, 0) * pieces + piece[u]];
            }
        };
        auto store = [&](V (&x)[CMP_U], int first) __attribute__((always_inline)) {
#pragma unroll
            for (int u = 0; u < CMP_U; ++u) asm volatile("" : "+v"(x[u]));       // what was asked for has arrived ...
            __syncthreads();                                                     // ... for all threads
#pragma unroll
            for (int u = 0; u < CMP_U; ++u) {
                const int r = first + row[u];
                if (r < n && from[r] >= 0) data[(size_t)to[r] * pieces + piece[u]] = x[u];
            }
        };
        load(v[0], 0);
        for (int first = 0; first < n; first += 2 * rows) {
            load(v[1], first + rows);
            store(v[0], first);
            load(v[0], first + 2 * rows);
            store(v[1], first + rows);
        }
    }
}

__global__ __launch_bounds__(CMP_NT, 6) void cache_compact_kernel(CompactTensors ts, const int* __restrict__ kept, int K, const int* __restrict__ block_table,
                                                               int max_blocks, int n, int nkv, int page_size, uint32_t page_inv, int num_pages) {
    __shared__ int from[CMP_LIST], to[CMP_LIST];
    const int kvh = blockIdx.x % nkv, which = blockIdx.x / nkv, req = blockIdx.y, entry = blockIdx.z;
    const int* list = kept + (((size_t)entry * n + req) * nkv + kvh) * K;
    const int* table = block_table + (size_t)req * max_blocks;
    const int pieces = ts.pieces[which];
    const size_t base = (size_t)entry * num_pages * nkv * page_size * pieces;
    if (ts.wide[which]) compact_rows((f32x4_t*)ts.data[which] + base, pieces, ts.inv[which], list, K, table, max_blocks, kvh, nkv, page_size, page_inv, num_pages, from, to);
    else compact_rows((float*)ts.data[which] + base, pieces, ts.inv[which], list, K, table, max_blocks, kvh, nkv, page_size, page_inv, num_pages, from, to);
}

// tensors: `count` pointers to [entries, num_pages, nkv, page_size, row] with rows of row_bytes[i] (multiples of 4); kept
// [entries, n, nkv, K] as li_evict_select leaves it.
extern "C" int li_cache_compact(void* const* tensors, const int* row_bytes, int count, const int* block_table, int max_blocks, const int* kept, int K, int n,
                                int entries, int nkv, int page_size, int num_pages, hipStream_t stream) {
    if (n <= 0 || n > 65535 || entries <= 0 || entries > 65535 || nkv <= 0 || K <= 0 || K > EV_MAX_PLACES || count <= 0 || count > CMP_MAX_TENSORS || max_blocks <= 0 ||
        num_pages <= 0 || page_size <= 0 || (long)max_blocks * page_size > EV_MAX_PLACES)
        return LI_ERR_SIZE;
    CompactTensors ts = {};
    for (int i = 0; i < count; ++i) {
        if (row_bytes[i] <= 0 || row_bytes[i] % 4) return LI_ERR_SIZE;
        ts.data[i] = tensors[i];
        ts.wide[i] = row_bytes[i] % 16 == 0 && (uintptr_t)tensors[i] % 16 == 0;
        ts.pieces[i] = row_bytes[i] / (ts.wide[i] ? 16 : 4);
        if (ts.pieces[i] > CMP_NT * CMP_U || (long)num_pages * nkv * page_size >= 1L << 31) return LI_ERR_SIZE;
        ts.inv[i] = inverse_of(ts.pieces[i]);
    }
    cache_compact_kernel<<<dim3(nkv * count, n, entries), CMP_NT, 0, stream>>>(ts, kept, K, block_table, max_blocks, n, nkv, page_size, inverse_of(page_size), num_pages);
    return li_launch_status();
}
