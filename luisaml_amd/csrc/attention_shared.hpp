// attention_shared.hpp -- attention for groups of sequences that share their
// first tokens (attention_kernels.hpp, kPrefix and kOwn), built for bf16 queries
// by attention_shared.hip and for fp32 ones by attention_shared_f32.hip.
//
// What a group shares is read once, for the rows of all its sequences
// together, which then also fill the matrix instructions' columns; each
// sequence's own tokens as ever.  Both leave parts (results divided by their
// sums, and the sums' logarithms), and one join puts a row's together:
//   o = sum_p o_p 2^(L_p) / sum_p 2^(L_p),   L_p = log2 sum_(j in p) w_j
#pragma once

#include "attention_kernels.hpp"

namespace lcml {
namespace {

constexpr int kMostParts = kMostSplits / 2;  // of the prefix, and of the own tokens

// The prefix's workgroups, and then the own tokens' where few rows have them,
// in one launch: the former wait for the matrix cores and the latter for
// memory, and short calls save a launch.
template <int DP, bool EXACT, int NQ, int NP, bool MANY>
__global__ __launch_bounds__(256, DP <= 128 ? 2 : 1) void k_attention_shared(AttentionArgs prefix, Split psp,
                                                                             AttentionArgs own, Split osp, uint32_t first) {
    constexpr int DC = (DP + 63) / 64;
    using Few = FewLds<DC, kFewWaves>;
    using Prefix = std::conditional_t<MANY, ManyLds<DP>, Few>;
    __shared__ __attribute__((aligned(16))) char lds[sizeof(Prefix) > sizeof(Few) ? sizeof(Prefix) : sizeof(Few)];
    if (blockIdx.x < first) {
        if constexpr (MANY)
            many_rows<DP, EXACT, NQ, NP, kPrefix>(prefix, psp, blockIdx.x, *reinterpret_cast<ManyLds<DP> *>(lds));
        else
            few_rows<DC, NQ, NP, kFewWaves, kPrefix>(prefix, psp, blockIdx.x, *reinterpret_cast<Few *>(lds));
    } else {
        few_rows<DC, NQ, NP, kFewWaves, kOwn>(own, osp, blockIdx.x - first, *reinterpret_cast<Few *>(lds));
    }
}
static_assert(kManyWaves == 4 && kFewWaves == 4, "both in workgroups of 256");

// fewer parts where there are too many for the join
inline void cap_parts(Plan &p) {
    if (p.sp.splits <= kMostParts) return;
    p.groups = p.groups / p.sp.splits * kMostParts;
    p.sp.chunk = (int32_t)((((int64_t)p.sp.chunk * p.sp.splits + kMostParts - 1) / kMostParts + 63) & ~63);
    p.sp.splits = kMostParts;
}

// The parts of a prefix that many rows read: as many as make the least of, in
// us by measurement (heads of 128, others by their columns),
//   a step, 1.8 for a workgroup alone on its CU and 1.15 for each of several;
//   a start and an end for every two of a CU's, which overlap;
//   what the parts write and the join reads back, at 3.5 TB/s;
//   the own tokens' workgroups of few rows, which run beside one workgroup a CU
//   but after several.
// 64 queries behind 16384 tokens (16 row tiles): 16 parts 51 us, 17 (272
// workgroups) 56, 24 55, 32 62; 560 rows of 3 groups behind 6000 (74 tiles): 3
// parts 70 us, 6 53, 8 64; 8 x 100 rows behind 8192 (200 tiles): 3 parts 201 us,
// 5 174.  Other heads enter by a factor alone, and the model misses more there.
// What it takes and the best of 1 to 48 parts, in us: 64 queries of 32 heads over
// 8 behind 16384, heads of 64 40.5 and 36.3 (32 parts), 96 45.2 and 45.0, 128 50.0
// both, 256 (16 over 4) 71.3 and 62.3 (24); 8 x 100 behind 8192 64 136 and 115 (5),
// 96 162 and 148 (5), 256 241 both; 3 groups of 5 x 40 behind 6000 (16 over 2) 64
// 47.1 and 44.8 (6), 96 60.8 and 58.5 (5), 256 172 and 163 (3), 128 in fp32 90.6
// and 87.8 (6).
inline void divide_prefix(Plan &p, const Plan &own, int64_t dim, int64_t span) {
    const int64_t groups = p.groups / p.sp.splits, steps = (span + 63) / 64;
    const int64_t most = steps / 4 > kMostParts ? kMostParts : steps / 4;  // four steps at least
    const double width = many_width_of(dim), scale = width < 96 ? 0.67 : width / 128;
    const double own_us = own.few ? 3.5 + 2.5 * ((own.sp.chunk / 64 + kFewWaves - 1) / kFewWaves) : 0.0;
    const auto length = [&](int64_t n) { return (steps + n - 1) / n; };
    int64_t best = 1;
    double least = 0.0;
    for (int64_t n = 1; n <= most || n == 1; ++n) {
        const int64_t each = (groups * n + 255) / 256;  // workgroups of a CU
        const double us = length(n) * scale * (each == 1 ? 1.8 : 1.15 * each) + 8.0 * ((each + 1) / 2) +
                          groups * n * (kManyRows * 8.0 / 3.5e6) * dim + (each == 1 ? 0.0 : own_us);
        if (n == 1 || us < least) best = n, least = us;
    }
    p.sp.splits = (int32_t)best, p.sp.chunk = (int32_t)(length(best) * 64), p.groups = groups * best;
}

struct SharedPlan {
    Plan prefix, own;
};
inline SharedPlan make_shared_plan(int64_t tokens, int64_t seqs, int64_t groups, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_q, int64_t max_own, int64_t max_prefix) {
    SharedPlan s{};
    s.own = make_plan(seqs, q_heads, kv_heads, dim, max_q, max_own + 63, 0, 0);  // from a multiple of 64 on
    cap_parts(s.own);
    s.own.sp.parts = s.own.sp.splits;
    if (groups == 0) return s;
    // the tiles of all groups' rows, and one more for each group that ends inside a tile
    const int64_t rows = tokens * (q_heads / kv_heads);
    s.prefix = divide(s.own.few && few_rows(kv_heads, dim, rows, max_prefix), kv_heads, rows, max_prefix);
    if (!s.prefix.few) divide_prefix(s.prefix, s.own, dim, max_prefix);
    cap_parts(s.prefix);
    s.prefix.sp.tiles += (int32_t)(groups - 1);
    s.prefix.groups = kv_heads * s.prefix.sp.tiles * s.prefix.sp.splits;
    s.own.sp.first = s.prefix.sp.splits;
    s.prefix.sp.parts = s.own.sp.parts = s.prefix.sp.splits + s.own.sp.splits;
    return s;
}

// (own tokens that many rows have: none of their workgroups)
template <int DP, int NQ, int NP>
void start_shared(const AttentionArgs &prefix, const AttentionArgs &own, const SharedPlan &p, hipStream_t s) {
    const dim3 grid((unsigned)(p.prefix.groups + (p.own.few ? p.own.groups : 0))), block(256);
    const uint32_t first = (uint32_t)p.prefix.groups;
    if (p.prefix.few)
        hipLaunchKernelGGL((k_attention_shared<(DP == 96 ? 128 : DP), false, NQ, NP, false>), grid, block, 0, s, prefix, p.prefix.sp, own, p.own.sp, first);
    else if (own.t.dim == DP)
        hipLaunchKernelGGL((k_attention_shared<DP, true, NQ, NP, true>), grid, block, 0, s, prefix, p.prefix.sp, own, p.own.sp, first);
    else
        hipLaunchKernelGGL((k_attention_shared<DP, false, NQ, NP, true>), grid, block, 0, s, prefix, p.prefix.sp, own, p.own.sp, first);
}

template <int NQ, int NP>
hipError_t launch_shared_t(const AttentionArgs &prefix, const AttentionArgs &own, const SharedPlan &p, hipStream_t s) {
    hipError_t err = hipSuccess;
    if (p.own.few || p.prefix.groups) {
        const int width = many_width_of(own.t.dim);
        width == 64    ? start_shared<64, NQ, NP>(prefix, own, p, s)
        : width == 96  ? start_shared<96, NQ, NP>(prefix, own, p, s)
        : width == 128 ? start_shared<128, NQ, NP>(prefix, own, p, s)
                       : start_shared<256, NQ, NP>(prefix, own, p, s);
        err = hipGetLastError();
    }
    if (!p.own.few && err == hipSuccess) err = start_attention_many<kOwn, NQ, NP>(own, p.own, s);
    return err == hipSuccess ? start_join<kOwn, NP>(own, p.own.sp, p.own.sp.parts, s) : err;
}

// NQ = 1: the queries are bf16
template <int NQ>
hipError_t launch_shared(const AttentionArgs &own, const int32_t *prefix_table, int64_t prefix_stride, int64_t prefix_cols,
                         int64_t max_prefix, void *work, hipStream_t s, const char **kernel) {
    AttentionArgs prefix = own;
    prefix.t.table = prefix_table, prefix.t.table_stride = prefix_stride, prefix.t.table_cols = (int32_t)prefix_cols;
    prefix.max_q = own.t.tokens, prefix.max_kv = max_prefix, prefix.causal = 0;  // all rows lie behind it
    SharedPlan p = make_shared_plan(own.t.tokens, own.t.seqs, own.groups, own.q_heads, own.t.heads, own.t.dim, own.max_q,
                                    own.max_kv, max_prefix);
    if (p.prefix.groups)
        set_divisors(p.prefix.sp, prefix);
    else
        p.prefix.few = true;
    set_divisors(p.own.sp, own);
    p.prefix.sp.o = p.own.sp.o = static_cast<float *>(work);
    p.prefix.sp.lse = p.own.sp.lse = p.own.sp.o + (int64_t)own.t.tokens * own.q_heads * p.own.sp.parts * own.t.dim;
    *kernel = !p.own.few ? (p.prefix.groups ? "attention_shared_many, attention_many, attention_join" : "attention_many, attention_join")
              : !p.prefix.few && p.prefix.groups ? "attention_shared_many, attention_join"
                                                 : "attention_shared_few, attention_join";
    return own.o_bf16 ? launch_shared_t<NQ, 1>(prefix, own, p, s) : launch_shared_t<NQ, 2>(prefix, own, p, s);
}

}  // namespace
}  // namespace lcml
