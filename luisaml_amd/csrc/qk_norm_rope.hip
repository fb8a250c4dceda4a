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
#include "lcml_internal.hpp"

namespace lcml {
namespace {

constexpr int kThreads = 256;

struct __attribute__((packed, aligned(2))) H8 {
    uint16_t v[8];
};
struct __attribute__((packed, aligned(4))) F8 {
    float v[8];
};

template <bool BF16>
__device__ inline void load8(const void *p, int64_t i, float *x) {
    if constexpr (BF16) {
        const H8 q = *reinterpret_cast<const H8 *>(static_cast<const uint16_t *>(p) + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = bits_f32((uint32_t)q.v[e] << 16);
    } else {
        const F8 q = *reinterpret_cast<const F8 *>(static_cast<const float *>(p) + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = q.v[e];
    }
}
template <bool BF16>
__device__ inline float load1(const void *p, int64_t i) {
    if constexpr (BF16) return bits_f32((uint32_t)static_cast<const uint16_t *>(p)[i] << 16);
    return static_cast<const float *>(p)[i];
}
template <bool BF16>
__device__ inline void store8(void *p, int64_t i, const float *x) {
    if constexpr (BF16) {
        H8 q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q.v[e] = bf16_rne(x[e]);
        *reinterpret_cast<H8 *>(static_cast<uint16_t *>(p) + i) = q;
    } else {
        F8 q;
#pragma unroll
        for (int e = 0; e < 8; ++e) q.v[e] = x[e];
        *reinterpret_cast<F8 *>(static_cast<float *>(p) + i) = q;
    }
}
template <bool BF16>
__device__ inline void store1(void *p, int64_t i, float x) {
    if constexpr (BF16)
        static_cast<uint16_t *>(p)[i] = bf16_rne(x);
    else
        static_cast<float *>(p)[i] = x;
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

// how a lane's eight pairs lie in memory: two runs of eight elements, one run
// of sixteen, or anywhere (rot not a multiple of 16)
enum { kHalves = 0, kNeighbours = 1, kScattered = 2 };

// LANES for each head; IB, OB: bf16 in and out
template <int LANES, int PAIRS, bool IB, bool OB>
__global__ __launch_bounds__(kThreads) void k_qk_norm_rope(RopeArgs p) {
    constexpr int ROWS = 64 / LANES;
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
    const int32_t D = p.dim, half = p.rot >> 1, rest = (D - p.rot) >> 1, pair0 = 8 * u;
    const bool in = pair0 < D >> 1;
    // element of the first and second of pair i
    const auto first = [&](int32_t i) { return PAIRS == kNeighbours ? 2 * i : i < half ? i : p.rot + i - half; };
    const auto second = [&](int32_t i) { return PAIRS == kNeighbours ? 2 * i + 1 : i < half ? i + half : p.rot + i - half + rest; };
    float cs[8], sn[8];
    {
        const float *t = p.table + (int64_t)pos * p.rot;
#pragma unroll
        for (int e = 0; e < 8; ++e) cs[e] = 1.0f, sn[e] = 0.0f;
        if (in && pair0 + 8 <= half) {
            const F8 c = *reinterpret_cast<const F8 *>(t + pair0), s = *reinterpret_cast<const F8 *>(t + half + pair0);
#pragma unroll
            for (int e = 0; e < 8; ++e) cs[e] = c.v[e], sn[e] = s.v[e];
        } else if (in) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (pair0 + e < half) cs[e] = t[pair0 + e], sn[e] = t[half + pair0 + e];
        }
    }
    const int32_t fa = first(in ? pair0 : 0), fb = second(in ? pair0 : 0);
    // x: a lane's firsts, then its seconds
    const auto load = [&](const void *base, int64_t at, float *x, auto bf16) {
        constexpr bool B = decltype(bf16)::value;
        if constexpr (PAIRS == kHalves) {
            load8<B>(base, at + fa, x), load8<B>(base, at + fb, x + 8);
        } else if constexpr (PAIRS == kNeighbours) {
            float y[16];
            load8<B>(base, at + fa, y), load8<B>(base, at + fa + 8, y + 8);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = y[2 * e], x[8 + e] = y[2 * e + 1];
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int32_t i = in ? pair0 + e : 0;
                x[e] = load1<B>(base, at + first(i)), x[8 + e] = load1<B>(base, at + second(i));
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
        const void *src = is_k ? p.k : p.q;
        void *dst = is_k ? p.k_out : p.q_out;
        const float *g = is_k ? p.k_gamma : p.q_gamma;
        const int64_t row = head < heads ? head : 0;
        const int64_t at = (is_k ? token * p.k_token + row * p.k_head : token * p.q_token + row * p.q_head);
        float x[16];
        load(src, at, x, std::integral_constant<bool, IB>{});
        if (g && have != (int32_t)is_k) {
            load(g, 0, gamma, std::false_type{});
            have = is_k;
        }
        if (g) {
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
            const bool turn = PAIRS == kHalves ? pair0 < half : pair0 + e < half;
            const float a = fmaf(x[e], cs[e], -(x[8 + e] * sn[e])), b = fmaf(x[8 + e], cs[e], x[e] * sn[e]);
            y[e] = turn ? a : x[e], y[8 + e] = turn ? b : x[8 + e];
        }
        const int64_t to = (is_k ? token * p.ko_token + row * p.ko_head : token * p.qo_token + row * p.qo_head);
        if constexpr (PAIRS == kHalves) {
            store8<OB>(dst, to + fa, y), store8<OB>(dst, to + fb, y + 8);
        } else if constexpr (PAIRS == kNeighbours) {
            float z[16];
#pragma unroll
            for (int e = 0; e < 8; ++e) z[2 * e] = y[e], z[2 * e + 1] = y[8 + e];
            store8<OB>(dst, to + fa, z), store8<OB>(dst, to + fa + 8, z + 8);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) store1<OB>(dst, to + first(pair0 + e), y[e]), store1<OB>(dst, to + second(pair0 + e), y[8 + e]);
        }
    }
}

int lanes_of(int32_t dim) { return dim <= 16 ? 1 : dim <= 32 ? 2 : dim <= 64 ? 4 : dim <= 128 ? 8 : 16; }

template <int LANES, int PAIRS, bool IB, bool OB>
void start_typed(const RopeArgs &p, dim3 grid, hipStream_t s) {
    hipLaunchKernelGGL((k_qk_norm_rope<LANES, PAIRS, IB, OB>), grid, dim3(kThreads), 0, s, p);
}
template <int LANES, int PAIRS>
void start(const RopeArgs &p, bool ib, bool ob, dim3 grid, hipStream_t s) {
    if (ib)
        ob ? start_typed<LANES, PAIRS, true, true>(p, grid, s) : start_typed<LANES, PAIRS, true, false>(p, grid, s);
    else
        ob ? start_typed<LANES, PAIRS, false, true>(p, grid, s) : start_typed<LANES, PAIRS, false, false>(p, grid, s);
}
template <int LANES>
void start_lanes(const RopeArgs &p, bool ib, bool ob, dim3 grid, hipStream_t s) {
    if (p.interleaved)
        start<LANES, kNeighbours>(p, ib, ob, grid, s);
    else if (p.rot % 16 == 0)
        start<LANES, kHalves>(p, ib, ob, grid, s);
    else
        start<LANES, kScattered>(p, ib, ob, grid, s);
}

}  // namespace

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
