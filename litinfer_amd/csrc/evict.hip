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

#define EV_MAX_DH 256

typedef float f32x4_t __attribute__((ext_vector_type(4)));

// ------------------------------------------------------------------ attention weight, any head size
struct MassArgs {
    const int *block_table, *q_start, *q_len, *ctx_len;
    int max_blocks, nseg, nh, nkv, dh, page_size, num_pages, q_row_stride;
    float scale;                 // times log2(e): scores are held in powers of two
    int fresh;                   // keys written by this step are set
};

// place -> row of [kv heads, page size, *] inside the pool, or -1 where no page holds the place
__device__ __forceinline__ long place_row(const MassArgs& a, int seg, int kvh, int t) {
    const int page = a.block_table[(size_t)seg * a.max_blocks + t / a.page_size];
    if (page < 0 || page >= a.num_pages) return -1;
    return ((long)page * a.nkv + kvh) * a.page_size + t % a.page_size;
}

template <typename T>
__device__ __forceinline__ float dot_rows(const float* q, const T* k, int dh) {
    float s = 0.f;
    for (int d = 0; d < dh; ++d) s += q[d] * load_as_float(k + d);
    return s;
}

// lse [T, nh] (powers of two): a wave a (token, head), a key a lane.
template <typename T>
__global__ __launch_bounds__(64) void mass_rows_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, float* __restrict__ lse) {
    __shared__ float qs[EV_MAX_DH];
    const int seg = blockIdx.z, h = blockIdx.y, i = blockIdx.x, lane = threadIdx.x;
    if (i >= a.q_len[seg]) return;
    const int tok = a.q_start[seg] + i, seen = a.ctx_len[seg] - a.q_len[seg] + i + 1;
    for (int d = lane; d < a.dh; d += 64) qs[d] = load_as_float(q + (size_t)tok * a.q_row_stride + (size_t)h * a.dh + d);
    __syncthreads();
    float m = -INFINITY, l = 0.f;
    for (int t = lane; t < seen; t += 64) {
        const long row = place_row(a, seg, h / (a.nh / a.nkv), t);
        if (row < 0) continue;
        const float s = dot_rows(qs, k + row * a.dh, a.dh) * a.scale;
        const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;     // (a score of NaN has no part in the maximum, but in the sum)
        l = (m == -INFINITY ? l : l * exp2f(m - base)) + exp2f(s - base);
        m = mn;
    }
    const float mx = wave_max(m);
    l = wave_sum(m == -INFINITY ? l : l * exp2f(m - mx));
    if (lane == 0) lse[(size_t)tok * a.nh + h] = l == 0.f ? INFINITY : (mx == -INFINITY ? 0.f : mx) + log2f(l);     // (a row that sees nothing gives nothing)
}

// A block takes 64 keys of a (request, kv head); its four waves take the queries in turn and are added up in their order.
template <typename T>
__global__ __launch_bounds__(256) void mass_keys_kernel(const T* __restrict__ q, const T* __restrict__ k, MassArgs a, const float* __restrict__ lse,
                                                        float* __restrict__ mass) {
    __shared__ float qs[4][EV_MAX_DH], part[4][64];
    const int seg = blockIdx.z, kvh = blockIdx.y, lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int nq = a.q_len[seg], ctx = a.ctx_len[seg], t = blockIdx.x * 64 + lane, rep = a.nh / a.nkv;
    if ((int)blockIdx.x * 64 >= ctx) return;
    const long row = t < ctx ? place_row(a, seg, kvh, t) : -1;
    const int base = ctx - nq;                           // place of the step's first token
    const int i0 = max((int)blockIdx.x * 64 - base, 0);  // the first query that sees any of the block's keys
    float sum = 0.f;
    for (int i = i0; i < nq; i += 4)
        for (int r = 0; r < rep; ++r) {
            const int mine = i + w, tok = a.q_start[seg] + mine, h = kvh * rep + r;
            __syncthreads();
            if (mine < nq)
                for (int d = lane; d < a.dh; d += 64) qs[w][d] = load_as_float(q + (size_t)tok * a.q_row_stride + (size_t)h * a.dh + d);
            __syncthreads();
            if (mine < nq && row >= 0 && t <= base + mine)
                sum += exp2f(dot_rows(qs[w], k + row * a.dh, a.dh) * a.scale - lse[(size_t)tok * a.nh + h]);
        }
    part[w][lane] = sum;
    __syncthreads();
    if (w || row < 0) return;
    sum = ((part[0][lane] + part[1][lane]) + part[2][lane]) + part[3][lane];
    mass[row] = a.fresh && t >= base ? sum : mass[row] + sum;
}

extern "C" long li_attention_mass_work_floats(int tokens, int nh) { return (long)tokens * nh; }

extern "C" int li_attention_mass(const void* q, int q_row_stride, const void* kc, float* mass, int dtype, const int* block_table, int max_blocks,
                                 const int* q_start, const int* q_len, const int* ctx_len, int nseg, int max_q_len, int max_ctx_len,
                                 int nh, int nkv, int dh, int page_size, int num_pages, float scale, int fresh, float* work, hipStream_t stream) {
    if (nseg <= 0 || nseg > 65535 || nh <= 0 || nh > 65535 || nkv <= 0 || nh % nkv || dh <= 0 || dh > EV_MAX_DH || page_size <= 0 || max_blocks <= 0 ||
        max_q_len <= 0 || max_ctx_len < max_q_len || (long)max_ctx_len > (long)max_blocks * page_size || !work)
        return LI_ERR_SIZE;
    const MassArgs a = {block_table, q_start, q_len, ctx_len, max_blocks, nseg, nh, nkv, dh, page_size, num_pages, q_row_stride,
                        scale * 1.44269504088896341f, fresh};
    const dim3 rows(max_q_len, nh, nseg), keys((max_ctx_len + 63) / 64, nkv, nseg);
    if (dtype == LI_F32) {
        mass_rows_kernel<float><<<rows, 64, 0, stream>>>((const float*)q, (const float*)kc, a, work);
        mass_keys_kernel<float><<<keys, 256, 0, stream>>>((const float*)q, (const float*)kc, a, work, mass);
    } else if (dtype == LI_BF16) {
        mass_rows_kernel<bf16_t><<<rows, 64, 0, stream>>>((const bf16_t*)q, (const bf16_t*)kc, a, work);
        mass_keys_kernel<bf16_t><<<keys, 256, 0, stream>>>((const bf16_t*)q, (const bf16_t*)kc, a, work, mass);
    } else {
        return LI_ERR_DTYPE;
    }
    return li_launch_status();
}

// ------------------------------------------------------------------ which keys stay
// unsigned integers in the order of the floats; -0 counts as 0, NaN as less than everything
__device__ __forceinline__ uint32_t mass_order(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x + 0.f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

#define SEL_NT 256

// A block a (entry, request, kv head).  The m-th largest sum of the places between the first and the last ones is found digit by
// digit, eight bits a pass, by counting; then one pass in order writes the places.
__global__ __launch_bounds__(SEL_NT) void evict_select_kernel(const float* __restrict__ mass, const int* __restrict__ block_table, int max_blocks,
                                                              const int* __restrict__ lens, const int* __restrict__ keeps, int first_n, int recent_n,
                                                              int* __restrict__ out, int K, int nkv, int page_size, int num_pages) {
    __shared__ int hist[256], wsum[SEL_NT / 64], pick[2];
    const int kvh = blockIdx.x, req = blockIdx.y, entry = blockIdx.z, nreq = gridDim.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int* table = block_table + (size_t)req * max_blocks;
    const float* pool = mass + (size_t)entry * num_pages * nkv * page_size;
    int* dst = out + (((size_t)entry * nreq + req) * nkv + kvh) * K;
    const long room = (long)max_blocks * page_size;
    const int len = (int)min((long)max(lens[req], 0), room);
    const int keep = min(min(max(keeps[req], 0), len), K);
    const int recent = min(recent_n, keep), first = min(first_n, keep - recent), lo = first, hi = len - recent;
    const int want = keep - recent - first;              // places chosen by their sums among lo .. hi - 1
    auto key = [&](int t) {
        const int page = table[t / page_size];
        return page < 0 || page >= num_pages ? 0u : mass_order(pool[((size_t)page * nkv + kvh) * page_size + t % page_size]);
    };
    uint32_t prefix = 0, known = 0;
    int left = want;                                     // how many are still to be taken among those with the prefix
    if (want > 0 && want < hi - lo)
        for (int shift = 24; shift >= 0; shift -= 8) {
            __syncthreads();
            hist[tid] = 0;
            __syncthreads();
            for (int t = lo + tid; t < hi; t += SEL_NT) {
                const uint32_t u = key(t);
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
    const bool all = want >= hi - lo;
    int at = 0, ties = 0;                                // places written, places equal to the last one taken
    for (int t0 = 0; t0 < len; t0 += SEL_NT) {
        const int t = t0 + tid;
        bool in = false, tie = false;
        if (t < len) {
            if (t < lo || t >= hi || all) in = true;
            else if (want > 0) {
                const uint32_t u = key(t);
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
        if (in && pos < K) dst[pos] = t;
    }
    for (int j = at + tid; j < K; j += SEL_NT) dst[j] = -1;
}

// mass [entries, num_pages, nkv, page_size]; lens, keeps [n]; out [entries, n, nkv, K], ascending, -1 behind the last.
extern "C" int li_evict_select(const float* mass, const int* block_table, int max_blocks, const int* lens, const int* keeps, int n, int first, int recent,
                               int* out, int K, int entries, int nkv, int page_size, int num_pages, hipStream_t stream) {
    if (n <= 0 || n > 65535 || entries <= 0 || entries > 65535 || nkv <= 0 || K <= 0 || first < 0 || recent < 0 || max_blocks <= 0 || page_size <= 0 ||
        (long)max_blocks * page_size >= 1L << 31)
        return LI_ERR_SIZE;
    evict_select_kernel<<<dim3(nkv, n, entries), SEL_NT, 0, stream>>>(mass, block_table, max_blocks, lens, keeps, first, recent, out, K, nkv, page_size, num_pages);
    return li_launch_status();
}

// ------------------------------------------------------------------ the kept rows move to the front
#define CMP_NT 256
#define CMP_U 8
#define CMP_MAX_TENSORS 4

struct CompactTensors {
    void* data[CMP_MAX_TENSORS];
    int pieces[CMP_MAX_TENSORS];         // pieces of a row
    int wide[CMP_MAX_TENSORS];           // a piece is 16 bytes, else 4
    int count;
};

// kept is ascending, so kept[j] >= j: rows that are read lie at or behind those that are written, and rows of a later chunk behind
// all that an earlier one writes.  A chunk is read whole, then written.
template <typename V>
__device__ __forceinline__ void compact_rows(V* __restrict__ data, int pieces, const int* __restrict__ kept, int K, const int* __restrict__ table,
                                             int max_blocks, int kvh, int nkv, int page_size, int num_pages) {
    const long room = (long)max_blocks * page_size;
    const long total = (long)K * pieces;
    auto row_of = [&](int t) -> long {
        const int page = table[t / page_size];
        return page < 0 || page >= num_pages ? -1 : ((long)page * nkv + kvh) * page_size + t % page_size;
    };
    for (long p0 = 0; p0 < total; p0 += CMP_NT * CMP_U) {
        if (kept[p0 / pieces] < 0) break;                // (the list has ended: the same answer in every thread)
        V v[CMP_U];
        long to[CMP_U];
#pragma unroll
        for (int u = 0; u < CMP_U; ++u) {
            const long p = p0 + threadIdx.x + (long)CMP_NT * u;
            to[u] = -1;
            if (p >= total) continue;
            const int j = (int)(p / pieces), c = (int)(p % pieces), src = kept[j];
            if (src <= j || src >= room) continue;       // the list's end, or a row that stays
            const long a = row_of(src), b = row_of(j);
            if (a < 0 || b < 0) continue;
            v[u] = data[a * pieces + c];
            to[u] = b * pieces + c;
        }
        __builtin_amdgcn_s_waitcnt(0);                   // what was asked for has arrived
        __syncthreads();
#pragma unroll
        for (int u = 0; u < CMP_U; ++u)
            if (to[u] >= 0) data[to[u]] = v[u];
        __syncthreads();
    }
}

__global__ __launch_bounds__(CMP_NT) void cache_compact_kernel(CompactTensors ts, const int* __restrict__ kept, int K, const int* __restrict__ block_table,
                                                               int max_blocks, int n, int nkv, int page_size, int num_pages) {
    const int kvh = blockIdx.x % nkv, which = blockIdx.x / nkv, req = blockIdx.y, entry = blockIdx.z;
    const int* list = kept + (((size_t)entry * n + req) * nkv + kvh) * K;
    const int* table = block_table + (size_t)req * max_blocks;
    const int pieces = ts.pieces[which];
    const size_t base = (size_t)entry * num_pages * nkv * page_size * pieces;
    if (ts.wide[which]) compact_rows((f32x4_t*)ts.data[which] + base, pieces, list, K, table, max_blocks, kvh, nkv, page_size, num_pages);
    else compact_rows((float*)ts.data[which] + base, pieces, list, K, table, max_blocks, kvh, nkv, page_size, num_pages);
}

// tensors: `count` pointers to [entries, num_pages, nkv, page_size, row] with rows of row_bytes[i] (multiples of 4); kept
// [entries, n, nkv, K] as li_evict_select leaves it.
extern "C" int li_cache_compact(void* const* tensors, const int* row_bytes, int count, const int* block_table, int max_blocks, const int* kept, int K, int n,
                                int entries, int nkv, int page_size, int num_pages, hipStream_t stream) {
    if (n <= 0 || n > 65535 || entries <= 0 || entries > 65535 || nkv <= 0 || K <= 0 || count <= 0 || count > CMP_MAX_TENSORS || max_blocks <= 0 ||
        page_size <= 0 || (long)max_blocks * page_size >= 1L << 31)
        return LI_ERR_SIZE;
    CompactTensors ts = {};
    ts.count = count;
    for (int i = 0; i < count; ++i) {
        if (row_bytes[i] <= 0 || row_bytes[i] % 4) return LI_ERR_SIZE;
        ts.data[i] = tensors[i];
        ts.wide[i] = row_bytes[i] % 16 == 0 && (uintptr_t)tensors[i] % 16 == 0;
        ts.pieces[i] = row_bytes[i] / (ts.wide[i] ? 16 : 4);
    }
    cache_compact_kernel<<<dim3(nkv * count, n, entries), CMP_NT, 0, stream>>>(ts, kept, K, block_table, max_blocks, n, nkv, page_size, num_pages);
    return li_launch_status();
}
