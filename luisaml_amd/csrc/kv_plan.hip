// kv_plan.hip -- a step's pages, lengths and row indexes from the tokens that
// each request brings (gfx950).
//
//   old = ended ? 0 : held,  kv = old + n,  cu = exclusive sums of n
//   a stack of free pages: pages of sequences that ended go onto it, then every
//   column ceil(old / T) .. ceil(kv / T) - 1 takes one from its top, both in
//   order of (sequence, column); so the page of the r-th new column is known
//   from sums alone and nothing is handed out by an atomic.
//
// Bound by latency: a few dependent round trips to memory and the sums' barriers.
// One workgroup does it all where there is little to write; else it leaves the
// sums, and a second launch writes the new columns and the rows, each finding
// its sequence by bisection in LDS.
#include "kv_cache.hpp"
#include "lcml_internal.hpp"

namespace lcml {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
constexpr int kLdsSeqs = 2048;    // sequences whose sums fit a workgroup's LDS
constexpr int kEmitThreads = 256;

// inclusive sum over the lanes of a wavefront
__device__ inline int64_t wave_scan(int64_t v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const int64_t u = __shfl_up((long long)v, m);
        v += (threadIdx.x & 63) >= (unsigned)m ? u : 0;
    }
    return v;
}
// exclusive sum over the workgroup; *total: of all
__device__ inline int64_t block_scan(int64_t v, int64_t *red, int64_t *total) {
    const int wave = threadIdx.x >> 6;
    const int64_t in = wave_scan(v);
    if ((threadIdx.x & 63) == 63) red[wave] = in;
    __syncthreads();
    int64_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kPlanWaves; ++w) {
        const int64_t u = red[w];
        before += w < wave ? u : 0;
        all += u;
    }
    __syncthreads();
    *total = all;
    return before + in - v;
}

// the last of at[0 .. n] (rising, at[0] <= i < at[n]) that is not above i
template <class T>
__device__ inline int32_t find(const T *at, int32_t n, int64_t i) {
    int32_t lo = 0, hi = n;
    while (hi - lo > 1) {
        const int32_t m = (lo + hi) >> 1;
        if ((int64_t)at[m] <= i)
            lo = m;
        else
            hi = m;
    }
    return lo;
}

__device__ inline int32_t clamp32(int64_t v) { return (int32_t)(v < 0x7fffffff ? v : 0x7fffffff); }

// columns of n tokens, as far as the table goes
__device__ inline int32_t columns(const KvPlan &p, int32_t n) {
    const int32_t c = (int32_t)(((int64_t)n + (1 << p.tshift) - 1) >> p.tshift);
    return c < p.table_cols ? c : p.table_cols;
}

// a sequence before and after
struct Seq {
    int32_t old, kv;
};
__device__ inline Seq seq_of(const KvPlan &p, int32_t b) {
    const int32_t held = p.kv_len_in[b], n = p.new_tokens[b];
    Seq s;
    s.old = (p.ended && p.ended[b] != 0) || held < 0 ? 0 : held;
    s.kv = clamp32((int64_t)s.old + (n > 0 ? n : 0));
    return s;
}

// What is left to write once the sums are there: the new columns' pages, and
// the rows' positions and slots.  cu: row offsets; need: new columns before
// each sequence; both [seqs + 1].
template <class Need>
__device__ inline void emit(const KvPlan &p, const int32_t *cu, const Need *need, int32_t top, int64_t first, int64_t step) {
    const int64_t pages = (int64_t)need[p.seqs];
    for (int64_t i = first; i < pages; i += step) {
        const int32_t b = find(need, p.seqs, i), kv = p.kv_len[b];
        const int64_t at = top - 1 - i;
        // the last of a sequence's new columns is its last column
        const int32_t c = columns(p, kv) - (int32_t)((int64_t)need[b + 1] - i);
        p.table[(int64_t)b * p.table_stride + c] = at >= 0 ? p.free_pages[at] : -1;
    }
    if (!p.positions && !p.slots) return;
    for (int64_t r = first; r < p.tokens; r += step) {
        int32_t pos = -1;
        int64_t slot = -1;
        if (r < cu[p.seqs]) {
            const int32_t b = find(cu, p.seqs, r), kv = p.kv_len[b];
            pos = kv - (cu[b + 1] - (int32_t)r);
            const int32_t c = pos >> p.tshift, fresh = columns(p, kv) - (int32_t)((int64_t)need[b + 1] - (int64_t)need[b]);
            if (p.slots && c < p.table_cols) {
                const int64_t at = top - 1 - ((int64_t)need[b] + c - fresh);
                const int32_t page = c < fresh ? p.table[(int64_t)b * p.table_stride + c] : at >= 0 ? p.free_pages[at] : -1;
                if (page >= 0 && page < p.pages) slot = ((int64_t)page << p.tshift) + (pos & ((1 << p.tshift) - 1));
            }
        }
        if (p.positions) p.positions[r] = pos;
        if (p.slots) p.slots[r] = slot;
    }
}

// One workgroup: returned pages, lengths and sums; ALL: and the rest.  (Every
// input that an output may be the same array as is read before the barrier
// that the output is written after.)
template <bool ALL>
__global__ __launch_bounds__(kPlanThreads) void k_kv_plan(KvPlan p) {
    __shared__ int64_t red[kPlanWaves];
    __shared__ int64_t lens[kPlanThreads + 1];
    __shared__ int32_t s_cu[ALL ? kPlanThreads + 1 : 1];
    const int tid = threadIdx.x;
    int32_t top = p.free_in[0];
    top = top < 0 ? 0 : top > p.pages ? p.pages : top;
    __syncthreads();  // `left` may be the same word
    if (p.ended) {
        for (int32_t b0 = 0; b0 < p.seqs; b0 += kPlanThreads) {
            const int32_t b = b0 + tid;
            int32_t from = 0, n = 0;
            if (b < p.seqs && p.ended[b] != 0) {
                const int32_t held = p.kv_len_in[b];
                from = p.first_own ? p.first_own[b] : 0;
                from = from > 0 ? from : 0;
                n = columns(p, held > 0 ? held : 0) - from;
            }
            int64_t total, got;
            const int64_t at = block_scan(n > 0 ? n : 0, red, &total);
            lens[tid] = at;
            if (tid == 0) lens[kPlanThreads] = total;
            __syncthreads();
            for (int64_t i0 = 0; i0 < total; i0 += kPlanThreads) {
                const int64_t i = i0 + tid;
                int32_t page = -1;
                if (i < total) {
                    const int32_t k = find(lens, kPlanThreads, i), bb = b0 + k;
                    int32_t c = p.first_own ? p.first_own[bb] : 0;
                    c = (c > 0 ? c : 0) + (int32_t)(i - lens[k]);
                    page = p.table[(int64_t)bb * p.table_stride + c];
                }
                const bool back = page >= 0 && page < p.pages;
                const int64_t place = top + block_scan(back, red, &got);
                if (back && place < p.pages) p.free_pages[place] = page;
                top = clamp32(top + got < p.pages ? top + got : p.pages);
            }
            __syncthreads();
        }
    }
    int64_t rows = 0, fresh = 0;
    for (int32_t b0 = 0; b0 < p.seqs; b0 += kPlanThreads) {
        const int32_t b = b0 + tid;
        Seq s{0, 0};
        if (b < p.seqs) s = seq_of(p, b);
        int64_t n, f;
        const int32_t want = columns(p, s.kv) - columns(p, s.old);
        const int64_t row = rows + block_scan(s.kv - s.old, red, &n);
        const int64_t need = fresh + block_scan(want, red, &f);
        if (b < p.seqs) {
            p.kv_len[b] = s.kv;
            p.cu_q[b] = clamp32(row);
            if (ALL)
                lens[tid] = need, s_cu[tid] = clamp32(row);
            else
                p.work[b] = need;
        }
        rows += n, fresh += f;
    }
    if (tid == 0) {
        p.cu_q[p.seqs] = clamp32(rows);
        p.left[0] = (int32_t)(top - fresh > -0x7fffffff ? top - fresh : -0x7fffffff);
        if (ALL)
            lens[p.seqs] = fresh, s_cu[p.seqs] = clamp32(rows);
        else
            p.work[p.seqs] = fresh, p.work[p.seqs + 1] = top;
    }
    if constexpr (ALL) {
        __syncthreads();  // and the returned pages, and kv_len
        emit(p, s_cu, lens, top, tid, kPlanThreads);
    }
}

template <bool LDS>
__global__ __launch_bounds__(kEmitThreads) void k_kv_plan_emit(KvPlan p) {
    __shared__ int32_t cu[LDS ? kLdsSeqs + 1 : 1];
    __shared__ int64_t need[LDS ? kLdsSeqs + 1 : 1];
    const int32_t top = (int32_t)p.work[p.seqs + 1];
    const int64_t first = (int64_t)blockIdx.x * kEmitThreads + threadIdx.x, step = (int64_t)gridDim.x * kEmitThreads;
    if constexpr (LDS) {
        for (int32_t b = threadIdx.x; b <= p.seqs; b += kEmitThreads) cu[b] = p.cu_q[b], need[b] = p.work[b];
        __syncthreads();
        emit(p, cu, need, top, first, step);
    } else {
        emit(p, p.cu_q, p.work, top, first, step);
    }
}

bool at_once(int64_t seqs, int64_t tokens) { return seqs <= kPlanThreads && tokens <= 2048; }

}  // namespace

int64_t kv_plan_workspace(int64_t seqs, int64_t tokens) { return at_once(seqs, tokens) ? 0 : (seqs + 2) * 8; }

hipError_t launch_kv_plan(const KvPlan &p, hipStream_t s, const char **kernel) {
    if (at_once(p.seqs, p.tokens)) {
        *kernel = "kv_plan";
        hipLaunchKernelGGL(k_kv_plan<true>, dim3(1), dim3(kPlanThreads), 0, s, p);
        return hipGetLastError();
    }
    *kernel = "kv_plan, kv_plan_emit";
    hipLaunchKernelGGL(k_kv_plan<false>, dim3(1), dim3(kPlanThreads), 0, s, p);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess) return err;
    const int64_t most = p.tokens > p.seqs ? p.tokens : p.seqs, groups = (most + kEmitThreads - 1) / kEmitThreads;
    const dim3 grid((unsigned)(groups < 4096 ? groups : 4096));
    if (p.seqs <= kLdsSeqs)
        hipLaunchKernelGGL(k_kv_plan_emit<true>, grid, dim3(kEmitThreads), 0, s, p);
    else
        hipLaunchKernelGGL(k_kv_plan_emit<false>, grid, dim3(kEmitThreads), 0, s, p);
    return hipGetLastError();
}

}  // namespace lcml
