// qk_norm_rope.hip -- RMS norms of the heads of queries and keys, and the
// rotation by position, in one pass (gfx950).
//
//   v = x / sqrt(mean(x^2) + eps) * gamma                       (a head's D elements)
//   (v_a, v_b) -> (v_a cos - v_b sin, v_b cos + v_a sin)        for the pairs below rot
// with pairs (i, i + rot / 2), or neighbours (2 i, 2 i + 1).  Everything is
// fp32 between the load and the one rounding of the result.
//
// HBM-bound: a lane holds eight pairs of a head, so that a rotation never
// crosses lanes and a norm is a sum over 1 to 16 of them; a wavefront takes a
// token's heads in turn and keeps its cosines, sines and gammas.
//
// Measured: 32 + 8 heads of 128 in bf16, one token 2.5 us in a graph, 64 2.7, 8192
// (172 MB) 38 on new data, 4.5 TB/s; 1333 tokens of 32 heads of 96 in fp32,
// neighbours, 33 MB, 8.6 (3.8 TB/s).
#include "lcml_internal.hpp"

namespace lcml {
namespace {

constexpr int kThreads = 256;

typedef float f2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf2 __attribute__((ext_vector_type(2)));  // converted to nearest even, in hardware

// N elements from or to any element-aligned address
template <int N>
struct __attribute__((packed, aligned(2))) Halfs {
    uint16_t v[N];
};
template <int N>
struct __attribute__((packed, aligned(2))) Words {
    uint32_t v[N];
};
template <int N>
struct __attribute__((packed, aligned(4))) Floats {
    float v[N];
};
template <bool BF16, int N>
__device__ inline void load(const void *p, int64_t i, float *x) {
    if constexpr (BF16) {
        const Halfs<N> q = *reinterpret_cast<const Halfs<N> *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = bits_f32((uint32_t)q.v[e] << 16);
    } else {
        const Floats<N> q = *reinterpret_cast<const Floats<N> *>(static_cast<const float *>(p) + i);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = q.v[e];
    }
}
template <bool BF16, int N>
__device__ inline void store(void *p, int64_t i, const float *x) {
    if constexpr (BF16 && N == 1) {
        static_cast<uint16_t *>(p)[i] = bf16_rne(x[0]);
    } else if constexpr (BF16) {
        Words<N / 2> q;
#pragma unroll
        for (int e = 0; e < N; e += 2) q.v[e / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f2{x[e], x[e + 1]}, bf2));
        *reinterpret_cast<Words<N / 2> *>(static_cast<uint16_t *>(p) + i) = q;
    } else {
        Floats<N> q;
#pragma unroll
        for (int e = 0; e < N; ++e) q.v[e] = x[e];
        *reinterpret_cast<Floats<N> *>(static_cast<float *>(p) + i) = q;
    }
}

// sum over the LANES neighbours of a lane
template <int LANES>
__device__ inline float group_sum(float v) {
    const auto add = [&](auto ctrl) {
        v += bits_f32((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f32_bits(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if constexpr (LANES >= 2) add(std::integral_constant<int, 0xb1>{});   // lane ^ 1
    if constexpr (LANES >= 4) add(std::integral_constant<int, 0x4e>{});   // lane ^ 2
    if constexpr (LANES >= 8) add(std::integral_constant<int, 0x141>{});  // the other half of eight
    if constexpr (LANES >= 16) add(std::integral_constant<int, 0x140>{});  // the other half of sixteen
    return v;
}

// how a pair lies in memory: in the halves of the rotated part, or neighbours
enum { kHalves = 0, kNeighbours = 1 };

// A lane's eight pairs are runs of RUN, of 16 bytes of input where the halves'
// length is a multiple of that: run g of lane u starts at pair g * D / 2 / RUNS +
// RUN * u, so that every load of a wavefront is contiguous.
// LANES for each head; IB, OB: bf16 in and out
template <int LANES, int PAIRS, int RUN, bool IB, bool OB>
__global__ __launch_bounds__(kThreads) void k_qk_norm_rope(RopeArgs p) {
    constexpr int ROWS = 64 / LANES, RUNS = 8 / RUN;
    const int lane = threadIdx.x & 63, u = lane % LANES, r = lane / LANES;
    const int32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t id = blockIdx.x * (kThreads / 64) + wave;
    const uint32_t token = id / (uint32_t)p.parts, part = id - token * (uint32_t)p.parts;
    if (token >= (uint32_t)p.tokens) return;
    int32_t pos = 0;
    if (p.positions) {
        pos = p.positions[token];
        if (pos < 0 || pos >= p.table_rows) return;
    }
    const int32_t D = p.dim, half = p.rot >> 1, rest = (D - p.rot) >> 1;
    const bool in = 16 * u < D;
    const auto pair = [&](int e) { return (e / RUN) * (D / 2 / RUNS) + RUN * (in ? u : 0) + e % RUN; };
    // element of the first and second of pair i
    const auto first = [&](int32_t i) { return PAIRS == kNeighbours ? 2 * i : i < half ? i : p.rot + i - half; };
    const auto second = [&](int32_t i) { return PAIRS == kNeighbours ? 2 * i + 1 : i < half ? i + half : p.rot + i - half + rest; };
    float cs[8], sn[8];
#pragma unroll
    for (int g = 0; g < 8; g += RUN) {
        const float *t = p.table + (int64_t)pos * p.rot + pair(g);
        if (pair(g) + RUN <= half) {
            load<false, RUN>(t, 0, cs + g), load<false, RUN>(t, half, sn + g);
        } else {
#pragma unroll
            for (int e = g; e < g + RUN; ++e) {
                const bool turn = pair(e) < half;
                cs[e] = turn ? t[e - g] : 1.0f, sn[e] = turn ? t[half + e - g] : 0.0f;
            }
        }
    }
    // x: a lane's firsts, then its seconds
    const auto take = [&](const void *base, int64_t at, float *x, auto bf16) {
        constexpr bool B = decltype(bf16)::value;
#pragma unroll
        for (int g = 0; g < 8; g += RUN) {
            if constexpr (PAIRS != kNeighbours) {
                load<B, RUN>(base, at + first(pair(g)), x + g), load<B, RUN>(base, at + second(pair(g)), x + 8 + g);
            } else {
                float y[2 * RUN];
                load<B, 2 * RUN>(base, at + first(pair(g)), y);
#pragma unroll
                for (int e = 0; e < RUN; ++e) x[g + e] = y[2 * e], x[8 + g + e] = y[2 * e + 1];
            }
        }
    };
    const int32_t q_steps = (p.q_heads + ROWS - 1) / ROWS, steps = q_steps + (p.k_heads + ROWS - 1) / ROWS;
    float gamma[16];
    int32_t have = -1;  // whose gammas: 0 q's, 1 k's
    for (int32_t i = part; i < steps; i += p.parts) {
        const bool is_k = i >= q_steps;
        const int32_t head = (is_k ? i - q_steps : i) * ROWS + r, heads = is_k ? p.k_heads : p.q_heads;
        const bool live = in && head < heads;
        void *dst = is_k ? p.k_out : p.q_out;
        const float *g = is_k ? p.k_gamma : p.q_gamma;
        const int64_t row = head < heads ? head : 0;
        float x[16];
        take(is_k ? p.k : p.q, is_k ? token * p.k_token + row * p.k_head : token * p.q_token + row * p.q_head, x,
             std::integral_constant<bool, IB>{});
        if (g) {
            if (have != (int32_t)is_k) take(g, 0, gamma, std::false_type{});
            have = is_k;
            float sum = 0.0f;
#pragma unroll
            for (int e = 0; e < 16; ++e) sum = fmaf(x[e], x[e], sum);
            const float rstd = 1.0f / sqrtf(group_sum<LANES>(in ? sum : 0.0f) * p.inv_dim + p.eps);
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = x[e] * rstd * gamma[e];
        }
        if (!live) continue;
        float y[16];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            // (a product with a sine of 0 would make a NaN of a partner's infinity)
            const bool turn = pair(PAIRS == kNeighbours ? e : e / RUN * RUN) < half;
            const float a = fmaf(x[e], cs[e], -(x[8 + e] * sn[e])), b = fmaf(x[8 + e], cs[e], x[e] * sn[e]);
            y[e] = turn ? a : x[e], y[8 + e] = turn ? b : x[8 + e];
        }
        const int64_t to = is_k ? token * p.ko_token + row * p.ko_head : token * p.qo_token + row * p.qo_head;
#pragma unroll
        for (int g = 0; g < 8; g += RUN) {
            if constexpr (PAIRS != kNeighbours) {
                store<OB, RUN>(dst, to + first(pair(g)), y + g), store<OB, RUN>(dst, to + second(pair(g)), y + 8 + g);
            } else {
                float z[2 * RUN];
#pragma unroll
                for (int e = 0; e < RUN; ++e) z[2 * e] = y[g + e], z[2 * e + 1] = y[8 + g + e];
                store<OB, 2 * RUN>(dst, to + first(pair(g)), z);
            }
        }
    }
}

int lanes_of(int32_t dim) { return dim <= 16 ? 1 : dim <= 32 ? 2 : dim <= 64 ? 4 : dim <= 128 ? 8 : 16; }

template <int LANES, int PAIRS, int RUN, bool IB>
void start(const RopeArgs &p, bool ob, dim3 grid, hipStream_t s) {
    if (ob)
        hipLaunchKernelGGL((k_qk_norm_rope<LANES, PAIRS, RUN, IB, true>), grid, dim3(kThreads), 0, s, p);
    else
        hipLaunchKernelGGL((k_qk_norm_rope<LANES, PAIRS, RUN, IB, false>), grid, dim3(kThreads), 0, s, p);
}
// the longest runs that no half's end cuts: 8192 tokens of 40 heads of 128 in bf16
// with 128 elements rotated 28 us (runs of 8), 120 28 (4), 100 32 (2), 90 42 (1);
// 4096 tokens in fp32 27 (4), 28 (2), 30 (1)
template <int LANES>
void start_lanes(const RopeArgs &p, bool ib, bool ob, dim3 grid, hipStream_t s) {
    const int32_t half = p.rot >> 1;
    if (p.interleaved)
        ib ? start<LANES, kNeighbours, 4, true>(p, ob, grid, s) : start<LANES, kNeighbours, 2, false>(p, ob, grid, s);
    else if (ib)
        half % 8 == 0   ? start<LANES, kHalves, 8, true>(p, ob, grid, s)
        : half % 4 == 0 ? start<LANES, kHalves, 4, true>(p, ob, grid, s)
        : half % 2 == 0 ? start<LANES, kHalves, 2, true>(p, ob, grid, s)
                        : start<LANES, kHalves, 1, true>(p, ob, grid, s);
    else
        half % 4 == 0   ? start<LANES, kHalves, 4, false>(p, ob, grid, s)
        : half % 2 == 0 ? start<LANES, kHalves, 2, false>(p, ob, grid, s)
                        : start<LANES, kHalves, 1, false>(p, ob, grid, s);
}

}  // namespace

// A wavefront for each step of a token where there are few tokens (64: 2.7 us, one
// for all five steps 5.0; 512 3.7 and 5.6), and one for all from 8192 on, where it
// no longer matters (4096: 15.1 and 15.3).
int64_t qk_norm_rope_parts(int64_t tokens, int32_t q_heads, int32_t k_heads, int32_t dim) {
    const int rows = 64 / lanes_of(dim);
    const int64_t steps = (q_heads + rows - 1) / rows + (k_heads + rows - 1) / rows, parts = (8192 + tokens - 1) / tokens;
    return parts < steps ? parts : steps;
}

hipError_t launch_qk_norm_rope(RopeArgs p, bool in_bf16, bool out_bf16, hipStream_t s) {
    const int lanes = lanes_of(p.dim);
    p.parts = (int32_t)qk_norm_rope_parts(p.tokens, p.q_heads, p.k_heads, p.dim);
    const int64_t waves = p.tokens * p.parts, per = kThreads / 64;
    const dim3 grid((unsigned)((waves + per - 1) / per));
    lanes == 1    ? start_lanes<1>(p, in_bf16, out_bf16, grid, s)
    : lanes == 2  ? start_lanes<2>(p, in_bf16, out_bf16, grid, s)
    : lanes == 4  ? start_lanes<4>(p, in_bf16, out_bf16, grid, s)
    : lanes == 8  ? start_lanes<8>(p, in_bf16, out_bf16, grid, s)
                  : start_lanes<16>(p, in_bf16, out_bf16, grid, s);
    return hipGetLastError();
}

}  // namespace lcml
