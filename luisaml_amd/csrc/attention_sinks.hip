// attention_sinks.hip -- attention through a sliding window beside which the
// first positions stay visible (attention_kernels.hpp, kSinks).
#include "attention_kernels.hpp"

namespace lcml {
namespace {

// Few rows in one workgroup of eight wavefronts each, instead of parts of four
// and a join: a window bounds the steps, so that a join is seldom worth its
// launch and its bytes.
constexpr int kLoneWaves = 8;

template <int DC, int NQ, int NP>
void start_lone(const AttentionArgs &a, const Plan &p, hipStream_t s) {
    hipLaunchKernelGGL((k_attention_few<DC, NQ, NP, kLoneWaves, kSinks>), dim3((unsigned)p.groups), dim3(kLoneWaves * 64), 0, s, a,
                       p.sp);
}
template <int NQ, int NP>
hipError_t launch_lone(const AttentionArgs &a, const Plan &p, hipStream_t s) {
    a.t.dim <= 64 ? start_lone<1, NQ, NP>(a, p, s) : start_lone<2, NQ, NP>(a, p, s);
    return hipGetLastError();
}

// By measurement, in us, parts and a join against eight wavefronts (heads of
// 128 in bf16 unless said, one query a sequence, 8 KV heads): 64 workgroups and
// 10 steps 12.0 / 10.2, 17 13.6 / 13.0, 25 14.1 / 15.3; 128 and 32 steps 19.4 /
// 19.1, 47 23.3 / 24.7; 192 and 47 steps 35.8 / 27.1, 125 54 / 55; 256 and 32
// steps 34 / 25, 125 70 / 63; 512 and 47 steps 78 / 64, 125 128 / 119; heads of
// 64, 256 and 47 steps 29 / 20; fp32, 256 and 47 steps 44 / 34.  Heads of more
// than 128 elements have no registers for a second wavefront a SIMD.
bool lone(const AttentionArgs &a, const Plan &p) {
    const int64_t groups = p.groups / p.sp.splits, steps = ((int64_t)p.sp.chunk * p.sp.splits) >> 6;
    const int64_t most = groups < 128 ? 20 : groups < 192 ? 40 : 128;
    return p.few && p.sp.splits > 1 && a.t.dim <= 128 && groups <= 512 && steps <= most;
}

}  // namespace

hipError_t launch_attention_sinks(const AttentionArgs &a, void *work, hipStream_t s, const char **kernel) {
    Plan p = make_plan(a.t.seqs, a.q_heads, a.t.heads, a.t.dim, a.max_q, a.max_kv, a.window, a.sinks);
    if (!lone(a, p)) return launch_form<kSinks>(a, p, work, s, kernel);
    p.groups /= p.sp.splits, p.sp.chunk *= p.sp.splits, p.sp.splits = 1;
    set_divisors(p.sp, a);
    *kernel = "attention_few";
    if (a.q_bf16) return a.o_bf16 ? launch_lone<1, 1>(a, p, s) : launch_lone<1, 2>(a, p, s);
    return a.o_bf16 ? launch_lone<2, 1>(a, p, s) : launch_lone<2, 2>(a, p, s);
}

}  // namespace lcml
