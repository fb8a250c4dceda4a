// attention.hip -- attention over the E4M3 KV cache (gfx950).
//
//   o = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - max)
// over the tokens j that a query sees: j < kv_len, j <= its own position
// (causal), j > its position - window.  A query that sees none, or only scores
// of -inf, gives 0.
#include "kv_cache.hpp"
#include "lcml_internal.hpp"

namespace lcml {
namespace {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

constexpr int kThreads = 256;

// One query row and head for each workgroup: scores of 256 tokens at a time,
// one token a thread, then the columns of V, one a thread.
__global__ __launch_bounds__(kThreads) void k_attention_rows(AttentionArgs a) {
    __shared__ float q[256], p[kThreads];
    const KvTokens &t = a.t;
    const int32_t row = blockIdx.x / a.q_heads, h = blockIdx.x % a.q_heads, D = t.dim;
    const int32_t kvh = h / (a.q_heads / t.heads);
    int32_t b = 0;  // the row's sequence: the first with cu[b + 1] > row
    for (int32_t lo = 0, hi = t.seqs; lo < hi;) {
        b = (lo + hi) >> 1;
        if (t.cu[b + 1] > row)
            hi = b;
        else
            lo = b = b + 1;
    }
    if (b >= t.seqs) return;
    const SeqRows s = seq_rows(t, b);
    if (row < s.row0 || row >= s.row0 + s.n) return;
    const int32_t pos = s.pos0 + (row - s.row0);
    if ((int32_t)threadIdx.x < D) {
        const int64_t i = row * a.q_token + h * a.q_head + threadIdx.x;
        q[threadIdx.x] = a.q_bf16 ? bits_f32((uint32_t)static_cast<const uint16_t *>(a.q)[i] << 16)
                                  : static_cast<const float *>(a.q)[i];
    }
    __syncthreads();
    int64_t first = a.window > 0 ? (int64_t)pos - a.window + 1 : 0;
    if (first < 0) first = 0;
    const int64_t end = a.causal && pos + 1 < s.len ? pos + 1 : s.len;
    float m = -__builtin_inff(), l = 0.0f, o = 0.0f;
    for (int64_t j0 = first & ~(int64_t)15; j0 < end; j0 += kThreads) {
        const int64_t j = j0 + threadIdx.x;
        float x = -__builtin_inff();
        const int32_t page = j < end ? page_of(t, b, (int32_t)(j >> t.tshift)) : -1;
        if (j >= first && page >= 0) {
            const int64_t at = (int64_t)page * t.heads + kvh;
            const uint8_t *blk = a.k + (at << t.tshift) * D;
            const int32_t slot = (int32_t)j & ((1 << t.tshift) - 1);
            float acc = 0.0f;
            for (int32_t e = 0; e < D; e += 16) {
                const u4 w = *reinterpret_cast<const u4 *>(blk + k_place(slot, e, D));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const f2 u = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[c], false);
                    const f2 v = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[c], true);
                    acc = fmaf(u[0], q[e + 4 * c], acc);
                    acc = fmaf(u[1], q[e + 4 * c + 1], acc);
                    acc = fmaf(v[0], q[e + 4 * c + 2], acc);
                    acc = fmaf(v[1], q[e + 4 * c + 3], acc);
                }
            }
            x = acc * a.ks[at] * a.scale;
        }
        float top = -__builtin_inff();
        p[threadIdx.x] = x;
        __syncthreads();
        for (int w = 0; w < kThreads; ++w) top = fmaxf(top, p[w]);
        __syncthreads();
        const float m1 = fmaxf(m, top), base = m1 == -__builtin_inff() ? 0.0f : m1;
        const float e = expf(x - base);
        p[threadIdx.x] = e;
        __syncthreads();
        const float keep = m == -__builtin_inff() ? 0.0f : expf(m - base);
        o *= keep;
        l *= keep;
        for (int w = 0; w < kThreads; ++w) l += p[w];
        if ((int32_t)threadIdx.x < D) {
            for (int w = 0; w < kThreads && j0 + w < end; ++w) {
                if (j0 + w < first) continue;
                const int32_t pg = page_of(t, b, (int32_t)((j0 + w) >> t.tshift));
                if (pg < 0) continue;
                const int64_t at = (int64_t)pg * t.heads + kvh;
                const int32_t slot = (int32_t)(j0 + w) & ((1 << t.tshift) - 1);
                const uint8_t c = a.v[(at << t.tshift) * D + v_place(slot, threadIdx.x, D)];
                o = fmaf(p[w] * a.vs[at], __builtin_amdgcn_cvt_f32_fp8((int)c, 0), o);
            }
        }
        m = m1;
        __syncthreads();
    }
    if ((int32_t)threadIdx.x < D) {
        const int64_t i = row * a.o_token + h * a.o_head + threadIdx.x;
        const float y = l == 0.0f ? 0.0f : o / l;
        if (a.o_bf16)
            static_cast<uint16_t *>(a.o)[i] = bf16_rne(y);
        else
            static_cast<float *>(a.o)[i] = y;
    }
}

}  // namespace

int64_t attention_workspace(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t) { return 0; }

hipError_t launch_attention(const AttentionArgs &a, void *, hipStream_t s, const char **kernel) {
    *kernel = "attention_rows";
    hipLaunchKernelGGL(k_attention_rows, dim3((unsigned)((int64_t)a.t.tokens * a.q_heads)), dim3(kThreads), 0, s, a);
    return hipGetLastError();
}

}  // namespace lcml
