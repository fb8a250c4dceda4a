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
//
// Measured: 64 sequences of a decode step 4.0 us in a graph, 5.4 where pages
// come back (one round trip more), 256 4.3 and 6.5, 1024 6.5 and 9.9, 4096 17 and
// 33; 48 prompts, 196 000 rows, 7.7 in two launches, 13 with 4400 pages that come
// back.
#include "kv_cache.hpp"
#include "lcml_internal.hpp"

namespace lcml {
namespace {

constexpr int kMostThreads = 1024;
constexpr int kLdsSeqs = 2048;  // sequences whose sums fit a workgroup's LDS
constexpr int kEmitThreads = 256;

// v plus the value that the DPP control brings, where it brings one
template <int CTRL, int ROWS>
__device__ inline int64_t add_dpp(int64_t v) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xf, false);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xf, false);
    return v + (int64_t)((uint64_t)hi << 32 | lo);
}
// inclusive sum over the lanes of a wavefront: 1, 2, 4, 8 to the right within
// sixteen lanes, then each sixteen's last lane to the next, then 32's
__device__ inline int64_t wave_scan(int64_t v) {
    v = add_dpp<0x111, 0xf>(v);
    v = add_dpp<0x112, 0xf>(v);
    v = add_dpp<0x114, 0xf>(v);
    v = add_dpp<0x118, 0xf>(v);
    v = add_dpp<0x142, 0xa>(v);
    return add_dpp<0x143, 0xc>(v);
}
// v[x]: exclusive sum over the workgroup, total[x]: of all; red alternates
// between two calls, so that one barrier does
template <int NT, int N>
__device__ inline void block_scan(int64_t (&v)[N], int64_t (&total)[N], int64_t (*red)[NT / 64]) {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int x = 0; x < N; ++x) {
        const int64_t in = wave_scan(v[x]);
        if ((threadIdx.x & 63) == 63) red[x][wave] = in;
        v[x] = in - v[x];
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < N; ++x) {
        total[x] = 0;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            const int64_t u = red[x][w];
            v[x] += w < wave ? u : 0;
            total[x] += u;
        }
    }
}

// the last of at[0 .. n] (rising, at[0] <= i < at[n], n <= 2^30) that is not above i
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

constexpr int32_t kMostRows = 0x7fffffff;  // of all sequences, and tokens of one: as far as int32 goes
__device__ inline int32_t clamp32(int64_t v) { return (int32_t)(v < kMostRows ? v : kMostRows); }

// columns of n tokens, as far as the table goes
__device__ inline int32_t columns(const KvPlan &p, int32_t n) {
    const int32_t c = (int32_t)(((int64_t)n + (1 << p.tshift) - 1) >> p.tshift);
    return c < p.table_cols ? c : p.table_cols;
}

// What is left to write once the sums are there: the new columns' pages, and
// the rows' positions and slots.  cu: row offsets; need: new columns before
// each sequence; both [seqs + 1]; kv: lengths; cut: the first position of the
// sequence whose rows end at kMostRows, where its offsets may not say it.
__device__ inline void emit(const KvPlan &p, const int32_t *cu, const int64_t *need, const int32_t *kv, int32_t top,
                            int32_t cut, int64_t first, int64_t step) {
    const int64_t fresh = need[p.seqs], rows = p.positions || p.slots ? p.tokens : 0;
    const int64_t most = fresh > rows ? fresh : rows;
    for (int64_t i = first; i < most; i += step) {
        // loads of both before the stores
        int32_t page = -1, pos = -1, of = -1;
        int64_t column = -1;
        if (i < fresh) {
            const int32_t b = find(need, p.seqs, i);
            // the last of a sequence's new columns is its last column
            column = (int64_t)b * p.table_stride + (columns(p, kv[b]) - (int32_t)(need[b + 1] - i));
            if (top - 1 - i >= 0) page = p.free_pages[top - 1 - i];
        }
        if (i < rows && i < cu[p.seqs]) {
            const int32_t b = find(cu, p.seqs, i);
            pos = cu[b + 1] < kMostRows ? kv[b] - (cu[b + 1] - (int32_t)i) : cut + ((int32_t)i - cu[b]);
            const int32_t c = pos >> p.tshift, old = columns(p, kv[b]) - (int32_t)(need[b + 1] - need[b]);
            if (p.slots && c < p.table_cols) {
                const int64_t at = top - 1 - (need[b] + c - old);
                if (c < old)
                    of = p.table[(int64_t)b * p.table_stride + c];
                else if (at >= 0)
                    of = p.free_pages[at];
            }
        }
        if (column >= 0) p.table[column] = page;
        if (i >= rows) continue;
        if (p.positions) p.positions[i] = pos;
        if (p.slots)
            p.slots[i] = of >= 0 && of < p.pages ? ((int64_t)of << p.tshift) + (pos & ((1 << p.tshift) - 1)) : -1;
    }
}

// One workgroup: returned pages, lengths and sums; ALL (seqs <= NT): and the
// rest.  Each input that an output may share memory with is read by the thread
// that writes there, or before a barrier.
template <int NT, bool ALL>
__global__ __launch_bounds__(NT) void k_kv_plan(KvPlan p) {
    // table entries of a thread at a time; one count for each of them and each
    // wavefront, a lane of which scans them
    constexpr int kEach = 4, kCounts = kEach * NT / 64;
    static_assert(kCounts <= 64, "one lane each");
    __shared__ int64_t red[2][3][NT / 64];
    __shared__ int64_t lens[NT + 1];
    __shared__ int32_t firsts[NT], counts[2][kCounts];
    __shared__ int64_t s_need[ALL ? NT + 1 : 1];
    __shared__ int32_t s_cu[ALL ? NT + 1 : 1], s_kv[ALL ? NT : 1], s_cut;
    // work's last element: the stack's height, and `cut`
    int32_t *const last = ALL ? nullptr : reinterpret_cast<int32_t *>(p.work + p.seqs + 1);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int turn = 0;
    int32_t top = p.free_in[0];
    int64_t rows = 0, fresh = 0;
    for (int32_t b0 = 0; b0 < p.seqs; b0 += NT) {
        const int32_t b = b0 + tid;
        const bool in = b < p.seqs;
        const int32_t held0 = in ? p.kv_len_in[b] : 0, n = in ? p.new_tokens[b] : 0;
        const bool ended = p.ended && in && p.ended[b] != 0;
        int32_t own = p.first_own && in ? p.first_own[b] : 0;
        own = own > 0 ? own : 0;
        const int32_t held = held0 > 0 ? held0 : 0, old = ended ? 0 : held, kv = clamp32((int64_t)old + (n > 0 ? n : 0));
        const int32_t back = ended ? columns(p, held) - own : 0;
        // rows, new columns, returned columns
        int64_t at[3] = {kv - old, columns(p, kv) - columns(p, old), back > 0 ? back : 0}, total[3];
        block_scan<NT>(at, total, red[turn]);
        turn ^= 1;
        if (b0 == 0) top = top < 0 ? 0 : top > p.pages ? p.pages : top;
        if (total[2] > 0) {
            const int32_t there = p.seqs - b0 < NT ? p.seqs - b0 : NT;
            lens[tid] = at[2], firsts[tid] = own;
            if (tid == 0) lens[NT] = total[2];
            __syncthreads();
            for (int64_t i0 = 0; i0 < total[2]; i0 += (int64_t)NT * kEach) {
                int32_t page[kEach];
                uint64_t back[kEach];
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int64_t i = i0 + e * NT + tid;
                    page[e] = -1;
                    if (i < total[2]) {
                        const int32_t k = find(lens, there, i);
                        page[e] = p.table[(int64_t)(b0 + k) * p.table_stride + firsts[k] + (int32_t)(i - lens[k])];
                    }
                }
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    back[e] = __builtin_amdgcn_ballot_w64(page[e] >= 0 && page[e] < p.pages);
                    if (lane == 0) counts[turn][e * (NT / 64) + wave] = __builtin_popcountll(back[e]);
                }
                __syncthreads();
                const int64_t mine = lane < kCounts ? counts[turn][lane] : 0, sums = wave_scan(mine);
                turn ^= 1;
#pragma unroll
                for (int e = 0; e < kEach; ++e) {
                    const int32_t before = __builtin_amdgcn_readlane((int32_t)(sums - mine), e * (NT / 64) + wave);
                    const int64_t place = top + before + (int32_t)__builtin_popcountll(back[e] & ((1ull << lane) - 1));
                    if ((back[e] >> lane & 1) && place < p.pages) p.free_pages[place] = page[e];
                }
                const int64_t all = top + (int64_t)__builtin_amdgcn_readlane((int32_t)sums, 63);
                top = (int32_t)(all < p.pages ? all : p.pages);
            }
            if (b0 + NT < p.seqs) __syncthreads();  // lens is written again
        }
        if (in) {
            const int32_t row = clamp32(rows + at[0]);
            p.kv_len[b] = kv;
            p.cu_q[b] = row;
            if (ALL)
                s_need[tid] = at[1], s_cu[tid] = row, s_kv[tid] = kv;
            else
                p.work[b] = fresh + at[1];
            if (row < kMostRows && rows + at[0] + (kv - old) >= kMostRows) (ALL ? &s_cut : last + 1)[0] = old;
        }
        rows += total[0], fresh += total[1];
    }
    if (p.seqs == 0) {
        __syncthreads();  // `left` may be free_in
        top = top < 0 ? 0 : top > p.pages ? p.pages : top;
    }
    if (tid == 0) {
        p.cu_q[p.seqs] = clamp32(rows);
        p.left[0] = (int32_t)(top - fresh > -0x7fffffff ? top - fresh : -0x7fffffff);
        if (ALL)
            s_need[p.seqs] = fresh, s_cu[p.seqs] = clamp32(rows);
        else
            p.work[p.seqs] = fresh, last[0] = top;
    }
    if constexpr (ALL) {
        __syncthreads();  // and the returned pages
        emit(p, s_cu, s_need, s_kv, top, s_cut, tid, NT);
    }
}

template <bool LDS>
__global__ __launch_bounds__(kEmitThreads) void k_kv_plan_emit(KvPlan p) {
    __shared__ int32_t cu[LDS ? kLdsSeqs + 1 : 1], kv[LDS ? kLdsSeqs : 1];
    __shared__ int64_t need[LDS ? kLdsSeqs + 1 : 1];
    const int32_t *const last = reinterpret_cast<const int32_t *>(p.work + p.seqs + 1);
    const int32_t top = last[0], cut = last[1];
    const int64_t first = (int64_t)blockIdx.x * kEmitThreads + threadIdx.x, step = (int64_t)gridDim.x * kEmitThreads;
    if constexpr (LDS) {
        for (int32_t b = threadIdx.x; b <= p.seqs; b += kEmitThreads) {
            cu[b] = p.cu_q[b], need[b] = p.work[b];
            if (b < p.seqs) kv[b] = p.kv_len[b];
        }
        __syncthreads();
        emit(p, cu, need, kv, top, cut, first, step);
    } else {
        emit(p, p.cu_q, p.work, p.kv_len, top, cut, first, step);
    }
}

// One launch or two, in us in a graph: 64 sequences of 512 rows in all 5.1 and 6.7,
// 1024 5.1 and 6.9, 2048 6.3 and 6.8, 4096 8.5 and 6.9; 1000 of 2000 7.9 and 9.5; 8
// of 2048 5.6 and 6.7, of 4096 7.3 and 6.5.
bool at_once(int64_t seqs, int64_t tokens) { return seqs <= kMostThreads && tokens <= 2 * kMostThreads; }

}  // namespace

int64_t kv_plan_workspace(int64_t seqs, int64_t tokens) { return at_once(seqs, tokens) ? 0 : (seqs + 2) * 8; }

hipError_t launch_kv_plan(const KvPlan &p, hipStream_t s, const char **kernel) {
    if (at_once(p.seqs, p.tokens)) {
        *kernel = "kv_plan";
        // 64 sequences, 64 rows: 4.0 us with 256 threads, 5.1 with 1024; 256 and 256 4.3
        // and 5.5, 200 and 400 5.5 both, 256 and 512 5.5 both (where pages come back
        // 5.4 and 7.3, 6.5 and 7.8, 7.1 and 7.8, 7.7 and 7.9)
        if (p.seqs <= 256 && p.tokens <= 256)
            hipLaunchKernelGGL((k_kv_plan<256, true>), dim3(1), dim3(256), 0, s, p);
        else
            hipLaunchKernelGGL((k_kv_plan<kMostThreads, true>), dim3(1), dim3(kMostThreads), 0, s, p);
        return hipGetLastError();
    }
    *kernel = "kv_plan, kv_plan_emit";
    hipLaunchKernelGGL((k_kv_plan<kMostThreads, false>), dim3(1), dim3(kMostThreads), 0, s, p);
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
