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

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kPBits = 14;  // probabilities are held times 2^14, in fp16's range
constexpr int kVBits = 7;   // and V's codes times 2^7

// ---------------------------------------------------------- operand pieces --

// four codes times a power of two, exact while the products are normal in fp16
__device__ inline h4 widen4(uint32_t w, float s) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, false);
    const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, true);
    return h4{a[0], a[1], b[0], b[1]};
}
__device__ inline h8 join8(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ inline h8 widen8(uint32_t w0, uint32_t w1, float s) { return join8(widen4(w0, s), widen4(w1, s)); }

// bytes that are the NaN codes 0x7f and 0xff: their top bits
__device__ inline uint32_t nan_bits(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }

// the maximum over the four 16-lane rows of a wavefront, for each lane of a row
__device__ inline float rows_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
    v = fmaxf(bits_f32(a[0]), bits_f32(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
    return fmaxf(bits_f32(b[0]), bits_f32(b[1]));
}
__device__ inline float rows_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
    v = bits_f32(a[0]) + bits_f32(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
    return bits_f32(b[0]) + bits_f32(b[1]);
}

// The power of two that brings a query row's largest finite element into
// [2^14, 2^15): fp16 then holds a bf16 element exactly down to 2^-31 of that
// one, and an fp32 element in two pieces to 2^-22 of itself.
__device__ inline float query_factor(float amax) {
    const int e = 127 + 14 + 127 - (int)(f32_bits(amax) >> 23);
    return bits_f32((uint32_t)(e > 253 ? 253 : e) << 23);
}

// the exponent field of vs / vref, times 2^kVBits, as cvt_scalef32's scale
__device__ inline float v_ratio(uint32_t vs, uint32_t vref) {
    const int e = (int)(vs >> 23) - (int)(vref >> 23) + 127 + kVBits;
    return bits_f32((uint32_t)(e < 1 ? 1 : e) << 23);
}

// 2^kPBits 2^(t - m).  Two pieces take the factor after the exponential: with
// it in the argument, the rounding of a sum near 14 costs three bits.
template <int NP>
__device__ inline float weights_at(float m) {
    m = m == -kInf ? 0.0f : m;
    return NP == 1 ? m - (float)kPBits : m;
}
template <int NP>
__device__ inline float weight_of(float t, float mm) {
    const float e = __builtin_amdgcn_exp2f(t - mm);
    return NP == 1 ? e : e * (float)(1 << kPBits);
}

__device__ inline float load_q(const AttentionArgs &a, int64_t i) {
    return a.q_bf16 ? bits_f32((uint32_t)static_cast<const uint16_t *>(a.q)[i] << 16) : static_cast<const float *>(a.q)[i];
}

// 16-token blocks of a page or its scales: what a lane knows of one block
struct Block {
    uint32_t lo, hi;  // the block's number in the cache, 16 * D bytes each
    uint32_t ks, vs;  // its page's scales, as bits; vs 0: no such page
};

__device__ inline Block find_block(const AttentionArgs &a, int32_t b, int32_t head, int32_t tok, int32_t end) {
    Block r{0, 0, 0, 0};
    const int32_t page = tok < end ? page_of(a.t, b, tok >> a.t.tshift) : -1;
    if (page >= 0) {
        const uint64_t at = (uint64_t)page * a.t.heads + head;
        const uint64_t blk = (at << (a.t.tshift - 4)) + ((tok >> 4) & ((1 << (a.t.tshift - 4)) - 1));
        r.lo = (uint32_t)blk, r.hi = (uint32_t)(blk >> 32);
        r.ks = f32_bits(a.ks[at]), r.vs = f32_bits(a.vs[at]);
    }
    return r;
}

struct __attribute__((packed, aligned(4))) F4 {
    float v[4];
};
struct __attribute__((packed, aligned(2))) H4 {
    uint16_t v[4];
};

__device__ inline void store_o4(const AttentionArgs &a, int64_t i, f4 v) {
    if (a.o_bf16)
        *reinterpret_cast<H4 *>(static_cast<uint16_t *>(a.o) + i) = H4{{bf16_rne(v[0]), bf16_rne(v[1]), bf16_rne(v[2]), bf16_rne(v[3])}};
    else
        *reinterpret_cast<F4 *>(static_cast<float *>(a.o) + i) = F4{{v[0], v[1], v[2], v[3]}};
}

// How a row's tokens are divided: `splits` parts of `chunk` tokens; with more
// than one, part results (normalised) and the base-2 logarithms of their
// weights go to the workspace, [token * q_heads + head][split].
struct Split {
    int32_t splits, chunk, tiles;  // tiles: row tiles of one sequence and KV head
    float *o, *lse;
};

// positions that query i of a sequence sees: lo .. hi-1
__device__ inline void sees(const AttentionArgs &a, const SeqRows &s, int32_t i, int32_t *lo, int32_t *hi) {
    const int64_t pos = (int64_t)s.pos0 + i;
    const int64_t h = a.causal && pos + 1 < s.len ? pos + 1 : s.len;
    const int64_t l = a.window > 0 && pos - a.window + 1 > 0 ? pos - a.window + 1 : 0;
    *hi = h > 0 ? (int32_t)h : 0;
    *lo = l < *hi ? (int32_t)l : *hi;
}

// ----------------------------------------------- few rows for each KV head --
//
// One workgroup: a tile of up to 16 rows (queries x heads of the group) of
// one sequence and KV head, over one part of the tokens; its wavefronts take
// turns of 64 tokens, straight from memory into registers, and join at the
// end.  S^T = K Q^T and O^T = V^T P^T on 16x16x32 instructions: a row is a
// lane's column in both, so the softmax is a lane's own but for one exchange,
// and S^T's accumulators are P^T's operands as they stand (the reduction's
// order over tokens is V's order in the cache).
template <int DC, int NQ, int NP, int NW>
__global__ __launch_bounds__(NW * 64, DC <= 2 ? 2 : 1) void k_attention_few(AttentionArgs a, Split sp) {
    constexpr int DP = DC * 64, kPitch = DP + 4;
    __shared__ float red_m[NW][16], red_l[NW][16];
    __shared__ float buf[NW][16][kPitch];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
    const int32_t D = a.t.dim, G = a.q_heads / a.t.heads;
    uint32_t id = blockIdx.x;
    const int32_t head = id % a.t.heads;
    id /= a.t.heads;
    const int32_t split = id % sp.splits;
    id /= sp.splits;
    const int32_t tile = id % sp.tiles, b = id / sp.tiles;
    const SeqRows s = seq_rows(a.t, b);
    const int64_t rows = (int64_t)s.n * G;
    const int32_t row0 = tile * 16;
    if (row0 >= rows) return;
    const int32_t last = rows - row0 < 16 ? (int32_t)rows - 1 : row0 + 15;  // of the tile
    const int32_t row = row0 + r < last ? row0 + r : last;                  // this lane's
    const int32_t qi = row / G, qh = head * G + row % G;
    int32_t lo, hi, lo_min, hi_min, lo_max, hi_max;
    sees(a, s, qi, &lo, &hi);
    sees(a, s, row0 / G, &lo_min, &hi_min);
    sees(a, s, last / G, &lo_max, &hi_max);
    const int64_t from = (lo_min & ~63) + (int64_t)split * sp.chunk;
    int64_t to = split + 1 < sp.splits ? from + sp.chunk : (int64_t)1 << 31;
    to = to < hi_max ? to : hi_max;
    const int32_t start = from < to ? (int32_t)from : 0;
    const int32_t steps = from < to && a.t.pages > 0 ? (int32_t)((to - from + 63) >> 6) : 0;
    const int64_t out_row = ((int64_t)s.row0 + qi) * a.q_heads + qh;
    if (steps == 0 && sp.splits > 1) {
        if (threadIdx.x < 16 && row0 + r <= last) sp.lse[out_row * sp.splits + split] = -kInf;
        return;
    }
    const int32_t mine = (steps - wave + NW - 1) / NW;

    Block blk;
    auto find = [&](int32_t k) {  // this lane's of the next 64 blocks of the wavefront's steps
        blk = find_block(a, b, head, start + (((k + (lane >> 2)) * NW + wave) << 6) + (lane & 3) * 16, (int32_t)to);
    };
    u4 kk[4][DC], vv[4][DC];
    uint32_t ks[4], vs[4];
    auto base = [&](const uint8_t *p, int32_t k, int sb) {
        const int i = (k & 15) * 4 + sb;
        const uint64_t n = (uint32_t)__builtin_amdgcn_readlane((int)blk.lo, i) |
                           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)blk.hi, i) << 32;
        return p + n * (uint64_t)(16 * D);
    };
    auto issue_k = [&](int32_t k) {
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            const uint8_t *p = base(a.k, k, sb);
#pragma unroll
            for (int j = 0; j < DC; ++j)
                kk[sb][j] = (4 * j + g) * 16 < D ? *reinterpret_cast<const u4 *>(p + (4 * j + g) * 256 + r * 16) : u4{0, 0, 0, 0};
        }
    };
    auto issue_v = [&](int32_t k) {
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            const uint8_t *p = base(a.v, k, sb);
#pragma unroll
            for (int j = 0; j < DC; ++j)
                vv[sb][j] = 64 * j + 4 * r < D ? *reinterpret_cast<const u4 *>(p + g * 4 * D + (64 * j + 4 * r) * 4) : u4{0, 0, 0, 0};
        }
    };
    if (mine > 0) {
        find(0);
        issue_k(0);
        issue_v(0);
    }

    // the row's query in the operand's order, times a power of two
    h8 qf[NQ][DC][2];
    float cq;
    {
        const int64_t at = ((int64_t)s.row0 + qi) * a.q_token + (int64_t)qh * a.q_head;
        float x[DC][2][8], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = 16 * (4 * j + g) + 8 * h + e;
                    x[j][h][e] = d < D ? load_q(a, at + d) : 0.0f;
                    const float v = fabsf(x[j][h][e]);
                    amax = v > amax && v < kInf ? v : amax;
                }
        const float f = query_factor(rows_max(amax));
        cq = a.scale * kLog2e * (1.0f / f);
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float v = x[j][h][e] * f;
                    qf[0][j][h][e] = (_Float16)v;
                    if constexpr (NQ == 2) qf[NQ - 1][j][h][e] = (_Float16)(v - (float)qf[0][j][h][e]);
                }
    }

    f4 o[DC][4];
#pragma unroll
    for (int j = 0; j < DC; ++j)
#pragma unroll
        for (int t = 0; t < 4; ++t) o[j][t] = f4{0.f, 0.f, 0.f, 0.f};
    float m = -kInf, l = 0.0f;
    uint32_t vref = 0;
    auto scale_o = [&](float f) {
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int t = 0; t < 4; ++t) o[j][t] *= f;
    };

    for (int32_t k = 0; k < mine; ++k) {
        const int32_t tok = start + ((k * NW + wave) << 6);
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            ks[sb] = (uint32_t)__builtin_amdgcn_readlane((int)blk.ks, (k & 15) * 4 + sb);
            vs[sb] = (uint32_t)__builtin_amdgcn_readlane((int)blk.vs, (k & 15) * 4 + sb);
        }
        f4 t[4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            f4 acc{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const h8 kh = widen8(kk[sb][j][2 * h], kk[sb][j][2 * h + 1], 1.0f);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qf[q][j][h], acc, 0, 0, 0);
                }
            t[sb] = acc * (cq * bits_f32(ks[sb]));
        }
        if (k + 1 < mine) {
            if (((k + 1) & 15) == 0) find(k + 1);
            issue_k(k + 1);
        }
        const bool full = tok >= lo_max && tok + 64 <= hi_min && vs[0] && vs[1] && vs[2] && vs[3];
        uint32_t seen = 0xffff;  // bit 4 * sb + i
        if (!full) {
            seen = 0;
#pragma unroll
            for (int sb = 0; sb < 4; ++sb)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int32_t j = tok + 16 * sb + 4 * g + i;
                    const bool ok = j >= lo && j < hi && vs[sb] != 0;
                    seen |= (ok ? 1u : 0u) << (4 * sb + i);
                    t[sb][i] = ok ? t[sb][i] : -kInf;
                }
        }
        float mx = m;
#pragma unroll
        for (int sb = 0; sb < 4; ++sb)
#pragma unroll
            for (int i = 0; i < 4; ++i) mx = fmaxf(mx, t[sb][i]);
        mx = rows_max(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
            const float f = mx > m ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
            l *= f;
            scale_o(f);
            m = mx;
        }
        uint32_t top = vs[0] > vs[1] ? vs[0] : vs[1];
        top = vs[2] > top ? vs[2] : top;
        top = vs[3] > top ? vs[3] : top;
        if (top > vref) {
            const int e = (int)(vref >> 23) - (int)(top >> 23) + 127;
            scale_o(bits_f32((uint32_t)(e < 0 ? 0 : e) << 23));
            vref = top;
        }
        const float mm = weights_at<NP>(m);
        h8 p[NP][2];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = weight_of<NP>(t[sb][i], mm);
                l += e;
                const _Float16 eh = (_Float16)e;
                p[0][sb >> 1][(sb & 1) * 4 + i] = eh;
                if constexpr (NP == 2) p[NP - 1][sb >> 1][(sb & 1) * 4 + i] = (_Float16)(e - (float)eh);
            }
        float ratio[4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) ratio[sb] = v_ratio(vs[sb], vref);
        uint32_t bad = 0;
        if (!full) {
#pragma unroll
            for (int sb = 0; sb < 4; ++sb)
#pragma unroll
                for (int j = 0; j < DC; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) bad |= nan_bits(vv[sb][j][c]);
            bad = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
        }
        if (!bad) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int j = 0; j < DC; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const h8 va = join8(widen4(vv[2 * h][j][c], ratio[2 * h]), widen4(vv[2 * h + 1][j][c], ratio[2 * h + 1]));
#pragma unroll
                        for (int q = 0; q < NP; ++q) o[j][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[q][h], o[j][c], 0, 0, 0);
                    }
        } else {
            // Among tokens that not every row sees there are NaN codes: they
            // count as zeros, and a product of "is NaN" and "is seen" says
            // which results they reach.
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    f4 hit{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        h8 va, is, on;
#pragma unroll
                        for (int u = 0; u < 2; ++u) {
                            const uint32_t w = vv[2 * h + u][j][c], n = nan_bits(w) >> 7;
                            const h4 x = widen4(w & ~(n * 0xffu), ratio[2 * h + u]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                va[4 * u + e] = x[e];
                                is[4 * u + e] = (n >> (8 * e)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
                                on[4 * u + e] = (seen >> (4 * (2 * h + u) + e)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
                            }
                        }
#pragma unroll
                        for (int q = 0; q < NP; ++q) o[j][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[q][h], o[j][c], 0, 0, 0);
                        hit = __builtin_amdgcn_mfma_f32_16x16x32_f16(is, on, hit, 0, 0, 0);
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) o[j][c][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[j][c][i];
                }
        }
        if (k + 1 < mine) issue_v(k + 1);
    }

    // join the wavefronts
    l = rows_sum(l);
    if (g == 0) red_m[wave][r] = m, red_l[wave][r] = l;
    __syncthreads();
    float top = -kInf, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, red_m[w][r]);
    auto weight = [&](float v) { return v == top ? 1.0f : __builtin_amdgcn_exp2f(v - top); };
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += red_l[w][r] * weight(red_m[w][r]);
    const float f = sum == 0.0f ? 0.0f : weight(m) / sum * (bits_f32(vref) * (1.0f / (1 << kVBits)));
#pragma unroll
    for (int j = 0; j < DC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f4 *>(&buf[wave][r][64 * j + 16 * g + 4 * i]) =
                sum == 0.0f ? f4{0.f, 0.f, 0.f, 0.f} : f4{o[j][0][i], o[j][1][i], o[j][2][i], o[j][3][i]} * f;
    if (sp.splits > 1 && wave == 0 && g == 0 && row0 + r <= last)
        sp.lse[out_row * sp.splits + split] = sum == 0.0f ? -kInf : top + __builtin_amdgcn_logf(sum);
    __syncthreads();
    const int32_t q4 = D >> 2;
    for (int32_t e = threadIdx.x; e < (last - row0 + 1) * q4; e += NW * 64) {
        const int32_t rr = e / q4, d = e % q4 * 4, i = (row0 + rr) / G, h = head * G + (row0 + rr) % G;
        f4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const f4 *>(&buf[w][rr][d]);
        if (sp.splits > 1)
            *reinterpret_cast<f4 *>(sp.o + ((((int64_t)s.row0 + i) * a.q_heads + h) * sp.splits + split) * D + d) = v;
        else
            store_o4(a, ((int64_t)s.row0 + i) * a.o_token + (int64_t)h * a.o_head + d, v);
    }
}

// ---------------------------------------------------------------- many rows --
//
// One workgroup: 128 rows (queries x heads of the group) of one sequence and
// KV head, 32 for each wavefront, over one part of the tokens.  K and V go
// through LDS as codes, 64 tokens a step and two steps in turn, and are widened
// to fp16 in registers, where a wavefront uses each for all its rows.  As
// above, S^T = K Q^T and O^T = V^T P^T, on 32x32x16 instructions.
constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;

template <int DP, bool EXACT, int NQ, int NP>
__global__ __launch_bounds__(kManyWaves * 64, DP <= 128 ? 2 : 1) void k_attention_many(AttentionArgs a, Split sp) {
    constexpr int KJ = DP / 32;                // pairs of 16-element pieces of K
    constexpr int MT = DP / 32;                // tiles of 32 columns of V
    constexpr int CPL = DP >= 128 ? 4 : 2;     // columns of V that a lane reads at once
    constexpr int VR = MT / CPL;               // such reads for a group of four tokens
    constexpr int kHalf = 64 * DP + 4 * DP;    // K's or V's bytes of a step, and room for reads past D
    constexpr int PL = (16 * DP / 16 + 63) / 64;  // 16-byte loads for a lane of a 16-token block
    __shared__ __attribute__((aligned(16))) uint8_t stage[2][2][kHalf];
    __shared__ uint32_t info[2][4][3];  // of a block: K's and V's scale, V has NaN codes
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t D = EXACT ? DP : a.t.dim, G = a.q_heads / a.t.heads;
    // workgroups of one sequence and KV head on one XCD (blockIdx modulo 8),
    // whose L2 then holds their K and V; the longest rows first
    const uint32_t pairs = (uint32_t)a.t.seqs * a.t.heads, per = (uint32_t)sp.tiles * sp.splits;
    uint32_t pair, rest;
    if (pairs % 8 == 0) {
        pair = blockIdx.x % 8 + 8 * (blockIdx.x / (8 * per));
        rest = blockIdx.x / 8 % per;
    } else {
        pair = blockIdx.x / per;
        rest = blockIdx.x % per;
    }
    const int32_t head = pair % a.t.heads, b = pair / a.t.heads;
    const int32_t split = rest % sp.splits, tile = sp.tiles - 1 - (int32_t)(rest / sp.splits);
    const SeqRows s = seq_rows(a.t, b);
    const int64_t rows = (int64_t)s.n * G, row0 = (int64_t)tile * kManyRows;
    if (row0 >= rows) return;
    const int64_t last = rows - row0 < kManyRows ? rows - 1 : row0 + kManyRows - 1;
    // this wavefront's rows and this lane's
    const int64_t w0 = row0 + 32 * wave < last ? row0 + 32 * wave : last, w1 = w0 + 31 < last ? w0 + 31 : last;
    const bool live = row0 + 32 * wave + r <= last;
    const int64_t row = live ? row0 + 32 * wave + r : w1;
    const int32_t qi = (int32_t)(row / G), qh = head * G + (int32_t)(row % G);
    int32_t lo, hi, lo_min, hi_min, lo_max, hi_max, w_lo, w_hi, skip0, skip1;
    sees(a, s, qi, &lo, &hi);
    sees(a, s, (int32_t)(row0 / G), &lo_min, &skip0);
    sees(a, s, (int32_t)(last / G), &skip1, &hi_max);
    sees(a, s, (int32_t)(w0 / G), &w_lo, &hi_min);  // of the wavefront: all tokens, and those that every row sees
    sees(a, s, (int32_t)(w1 / G), &lo_max, &w_hi);
    const int64_t from = (lo_min & ~63) + (int64_t)split * sp.chunk;
    int64_t to = split + 1 < sp.splits ? from + sp.chunk : (int64_t)1 << 31;
    to = to < hi_max ? to : hi_max;
    const int32_t start = from < to ? (int32_t)from : 0;
    const int32_t steps = from < to && a.t.pages > 0 ? (int32_t)((to - from + 63) >> 6) : 0;
    const int64_t out_row = ((int64_t)s.row0 + qi) * a.q_heads + qh;
    if (steps == 0 && sp.splits > 1) {
        if (h == 0 && live) sp.lse[out_row * sp.splits + split] = -kInf;
        return;
    }

    // a step's 64 tokens: this wavefront brings block `wave` of them
    u4 kr[PL], vr[PL];
    uint32_t ksr = 0, vsr = 0;
    auto fetch = [&](int32_t k) {
        const Block blk = find_block(a, b, head, start + (k << 6) + 16 * wave, (int32_t)to);
        ksr = blk.ks, vsr = blk.vs;
        const uint64_t at = (blk.lo | (uint64_t)blk.hi << 32) * (uint64_t)(16 * D);
#pragma unroll
        for (int x = 0; x < PL; ++x) {
            const bool in = blk.vs != 0 && (EXACT && DP % 64 == 0 ? true : 64 * x + lane < D);
            kr[x] = in ? *reinterpret_cast<const u4 *>(a.k + at + (64 * x + lane) * 16) : u4{0, 0, 0, 0};
            vr[x] = in ? *reinterpret_cast<const u4 *>(a.v + at + (64 * x + lane) * 16) : u4{0, 0, 0, 0};
        }
    };
    auto deposit = [&](int buf) {
        uint32_t bad = 0;
#pragma unroll
        for (int x = 0; x < PL; ++x) {
            if (EXACT || 64 * x + lane < D) {
                *reinterpret_cast<u4 *>(&stage[buf][0][wave * 16 * D + (64 * x + lane) * 16]) = kr[x];
                *reinterpret_cast<u4 *>(&stage[buf][1][wave * 16 * D + (64 * x + lane) * 16]) = vr[x];
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) bad |= nan_bits(vr[x][c]);
        }
        const bool any = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
        if (lane == 0) info[buf][wave][0] = ksr, info[buf][wave][1] = vsr, info[buf][wave][2] = any;
    };

    if (steps > 0) fetch(0);

    h8 qf[NQ][KJ][2];
    float cq;
    {
        const int64_t at = ((int64_t)s.row0 + qi) * a.q_token + (int64_t)qh * a.q_head;
        float amax = 0.0f;
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                const int d = 32 * j + 16 * h + u;
                const float v = d < D ? fabsf(load_q(a, at + d)) : 0.0f;
                amax = v > amax && v < kInf ? v : amax;
            }
        const auto sw = __builtin_amdgcn_permlane32_swap(f32_bits(amax), f32_bits(amax), false, false);
        const float f = query_factor(fmaxf(bits_f32(sw[0]), bits_f32(sw[1])));
        cq = a.scale * kLog2e * (1.0f / f);
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int u = 0; u < 16; ++u) {
                const int d = 32 * j + 16 * h + u;
                const float v = (d < D ? load_q(a, at + d) : 0.0f) * f;
                qf[0][j][u >> 3][u & 7] = (_Float16)v;
                if constexpr (NQ == 2) qf[NQ - 1][j][u >> 3][u & 7] = (_Float16)(v - (float)(_Float16)v);
            }
    }

    f16v o[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    float m = -kInf, l = 0.0f;
    uint32_t vref = 0;
    auto scale_o = [&](float f) {
#pragma unroll
        for (int t = 0; t < MT; ++t) o[t] *= f;
    };
    if (steps > 0) deposit(0);
    __syncthreads();

    for (int32_t k = 0; k < steps; ++k) {
        const int32_t tok = start + (k << 6);
        const int buf = k & 1;
        if (k + 1 < steps) fetch(k + 1);
        if (tok < w_hi && tok + 64 > w_lo) {
            const uint8_t *sk = stage[buf][0], *sv = stage[buf][1];
            uint32_t ks[4], vs[4], nan = 0;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                ks[q] = __builtin_amdgcn_readfirstlane(info[buf][q][0]);
                vs[q] = __builtin_amdgcn_readfirstlane(info[buf][q][1]);
                nan |= __builtin_amdgcn_readfirstlane(info[buf][q][2]);
            }
            f16v t[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                f16v acc;
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[i] = 0.0f;
                const uint8_t *p = sk + (2 * q + (r >> 4)) * 16 * D + h * 256 + (r & 15) * 16;
#pragma unroll
                for (int j = 0; j < KJ; ++j) {
                    if (!EXACT && 32 * j >= D) break;
                    u4 w = *reinterpret_cast<const u4 *>(p + j * 512);
                    if (!EXACT && 32 * j + 16 * h >= D) w = u4{0, 0, 0, 0};
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const h8 kh = widen8(w[2 * u], w[2 * u + 1], 1.0f);
#pragma unroll
                        for (int x = 0; x < NQ; ++x) acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qf[x][j][u], acc, 0, 0, 0);
                    }
                }
                const float c0 = cq * bits_f32(ks[2 * q]), c1 = cq * bits_f32(ks[2 * q + 1]);
#pragma unroll
                for (int i = 0; i < 16; ++i) t[q][i] = acc[i] * (i < 8 ? c0 : c1);
            }
            const bool full = tok >= lo_max && tok + 64 <= hi_min && vs[0] && vs[1] && vs[2] && vs[3];
            if (!full) {
#pragma unroll
                for (int q = 0; q < 2; ++q)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int32_t j = tok + 32 * q + 8 * (i >> 2) + 4 * h + (i & 3);
                        const bool ok = j >= lo && j < hi && vs[2 * q + (i >> 3)] != 0;
                        t[q][i] = ok ? t[q][i] : -kInf;
                    }
            }
            float mx = m;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, t[q][i]);
            const auto sw = __builtin_amdgcn_permlane32_swap(f32_bits(mx), f32_bits(mx), false, false);
            mx = fmaxf(bits_f32(sw[0]), bits_f32(sw[1]));
            if (__builtin_amdgcn_ballot_w64(mx > m) != 0) {
                const float f = mx > m ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
                l *= f;
                scale_o(f);
                m = mx;
            }
            uint32_t top = vs[0] > vs[1] ? vs[0] : vs[1];
            top = vs[2] > top ? vs[2] : top;
            top = vs[3] > top ? vs[3] : top;
            if (top > vref) {
                const int e = (int)(vref >> 23) - (int)(top >> 23) + 127;
                scale_o(bits_f32((uint32_t)(e < 0 ? 0 : e) << 23));
                vref = top;
            }
            const float mm = weights_at<NP>(m);
            h8 p[NP][4];
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float e = weight_of<NP>(t[q][i], mm);
                    l += e;
                    const _Float16 eh = (_Float16)e;
                    p[0][2 * q + (i >> 3)][i & 7] = eh;
                    if constexpr (NP == 2) p[NP - 1][2 * q + (i >> 3)][i & 7] = (_Float16)(e - (float)eh);
                }
            const bool mend = !full && nan;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const float ratio = v_ratio(vs[q], vref);
#pragma unroll
                for (int x = 0; x < VR; ++x) {
                    const uint8_t *pv = sv + q * 16 * D + h * 4 * D + (128 * x + CPL * r) * 4;
                    uint32_t w0[CPL], w1[CPL];
                    if constexpr (CPL == 4) {
                        const u4 u0 = *reinterpret_cast<const u4 *>(pv), u1 = *reinterpret_cast<const u4 *>(pv + 8 * D);
#pragma unroll
                        for (int c = 0; c < CPL; ++c) w0[c] = u0[c], w1[c] = u1[c];
                    } else {
                        const u2 u0 = *reinterpret_cast<const u2 *>(pv), u1 = *reinterpret_cast<const u2 *>(pv + 8 * D);
#pragma unroll
                        for (int c = 0; c < CPL; ++c) w0[c] = u0[c], w1[c] = u1[c];
                    }
#pragma unroll
                    for (int c = 0; c < CPL; ++c) {
                        if (!mend) {
                            const h8 va = widen8(w0[c], w1[c], ratio);
#pragma unroll
                            for (int y = 0; y < NP; ++y)
                                o[x * CPL + c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, p[y][q], o[x * CPL + c], 0, 0, 0);
                        } else {
                            // as above: NaN codes among tokens that not every row sees
                            const uint32_t n0 = nan_bits(w0[c]) >> 7, n1 = nan_bits(w1[c]) >> 7;
                            const h8 va = widen8(w0[c] & ~(n0 * 0xffu), w1[c] & ~(n1 * 0xffu), ratio);
                            h8 is, on;
#pragma unroll
                            for (int e = 0; e < 8; ++e) {
                                is[e] = ((e < 4 ? n0 : n1) >> (8 * (e & 3))) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
                                const int32_t j = tok + 16 * q + 8 * (e >> 2) + 4 * h + (e & 3);
                                on[e] = j >= lo && j < hi && vs[q] != 0 ? (_Float16)1.0f : (_Float16)0.0f;
                            }
#pragma unroll
                            for (int y = 0; y < NP; ++y)
                                o[x * CPL + c] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, p[y][q], o[x * CPL + c], 0, 0, 0);
                            f16v hit;
#pragma unroll
                            for (int i = 0; i < 16; ++i) hit[i] = 0.0f;
                            hit = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, on, hit, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 16; ++i)
                                o[x * CPL + c][i] = hit[i] > 0.0f ? __builtin_nanf("") : o[x * CPL + c][i];
                        }
                    }
                }
            }
        }
        if (k + 1 < steps) deposit(buf ^ 1);
        __syncthreads();
    }

    const auto sw = __builtin_amdgcn_permlane32_swap(f32_bits(l), f32_bits(l), false, false);
    l = bits_f32(sw[0]) + bits_f32(sw[1]);
    if (!live) return;
    const float f = l == 0.0f ? 0.0f : bits_f32(vref) * (1.0f / (1 << kVBits)) / l;
    float *po = nullptr;
    if (sp.splits > 1) {
        po = sp.o + (out_row * sp.splits + split) * D;
        if (h == 0) sp.lse[out_row * sp.splits + split] = l == 0.0f ? -kInf : m + __builtin_amdgcn_logf(l);
    }
    const int64_t oo = ((int64_t)s.row0 + qi) * a.o_token + (int64_t)qh * a.o_head;
    // row 8 a + 4 h + b of tile c: columns 128 x + CPL * that + c
#pragma unroll
    for (int x = 0; x < VR; ++x)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < CPL; ++e) {
                const int d = 128 * x + CPL * (8 * i + 4 * h) + 4 * e;
                f4 v;
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    v[u] = l == 0.0f ? 0.0f : o[x * CPL + (4 * e + u) % CPL][4 * i + (4 * e + u) / CPL] * f;
                if (!EXACT && d >= D) continue;
                if (po)
                    *reinterpret_cast<f4 *>(po + d) = v;
                else
                    store_o4(a, oo + d, v);
            }
}

// Joins a row's parts: one wavefront a row.
__global__ __launch_bounds__(256) void k_attention_join(AttentionArgs a, Split sp) {
    const int32_t D = a.t.dim, lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), per = a.max_q * a.q_heads;
    const int64_t b = id / per, i = id % per / a.q_heads, h = id % a.q_heads;
    if (b >= a.t.seqs) return;
    const SeqRows s = seq_rows(a.t, (int32_t)b);
    if (i >= s.n) return;
    const int64_t row = (s.row0 + i) * a.q_heads + h;
    const float *lse = sp.lse + row * sp.splits, *po = sp.o + row * sp.splits * D;
    float top = -kInf;
    for (int32_t k = 0; k < sp.splits; ++k) top = fmaxf(top, lse[k]);
    float sum = 0.0f;
    f4 v{0.f, 0.f, 0.f, 0.f};
    for (int32_t k = 0; k < sp.splits; ++k) {
        const float x = lse[k];
        if (x == -kInf) continue;
        const float w = x == top ? 1.0f : __builtin_amdgcn_exp2f(x - top);
        sum += w;
        if (lane * 4 < D) v += *reinterpret_cast<const f4 *>(po + (int64_t)k * D + lane * 4) * w;
    }
    if (lane * 4 < D)
        store_o4(a, (s.row0 + i) * a.o_token + h * a.o_head + lane * 4, sum == 0.0f ? f4{0.f, 0.f, 0.f, 0.f} : v * (1.0f / sum));
}

// ------------------------------------------------------------------- plan --

constexpr int kFewWaves = 4;

struct Plan {
    bool few;
    Split sp;
};

Plan make_plan(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t max_q, int64_t max_kv, int64_t window) {
    Plan p{};
    const int64_t rows = max_q * (q_heads / kv_heads);
    p.few = rows <= 64;
    const int64_t tile = p.few ? 16 : kManyRows;
    p.sp.tiles = (int32_t)((rows + tile - 1) / tile);
    // tokens that a row tile can see
    int64_t span = max_kv;
    if (window > 0 && window < span && window + max_q + 64 < span) span = window + max_q + 64;
    const int64_t groups = seqs * kv_heads * p.sp.tiles, steps = (span + 63) / 64;
    int64_t splits = ((p.few ? 1024 : 512) + groups - 1) / groups;
    const int64_t most = (steps + 3) / 4;  // a step for each wavefront, or four for the workgroup
    if (splits > most) splits = most;
    if (splits > 128) splits = 128;
    if (splits < 1) splits = 1;
    p.sp.chunk = (int32_t)(((steps + splits - 1) / splits) * 64);
    p.sp.splits = (int32_t)splits;
    return p;
}

template <int DC, int NQ, int NP>
void start_few(const AttentionArgs &a, const Split &sp, unsigned grid, hipStream_t s) {
    hipLaunchKernelGGL((k_attention_few<DC, NQ, NP, kFewWaves>), dim3(grid), dim3(kFewWaves * 64), 0, s, a, sp);
}

template <int DP, int NQ, int NP>
void start_many(const AttentionArgs &a, const Split &sp, unsigned grid, hipStream_t s) {
    if (a.t.dim == DP)
        hipLaunchKernelGGL((k_attention_many<DP, true, NQ, NP>), dim3(grid), dim3(kManyWaves * 64), 0, s, a, sp);
    else
        hipLaunchKernelGGL((k_attention_many<DP, false, NQ, NP>), dim3(grid), dim3(kManyWaves * 64), 0, s, a, sp);
}

template <int NQ, int NP>
void start(const AttentionArgs &a, const Plan &p, unsigned grid, hipStream_t s) {
    const int32_t D = a.t.dim;
    if (p.few)
        D <= 64 ? start_few<1, NQ, NP>(a, p.sp, grid, s) : D <= 128 ? start_few<2, NQ, NP>(a, p.sp, grid, s) : start_few<4, NQ, NP>(a, p.sp, grid, s);
    else
        D <= 64 ? start_many<64, NQ, NP>(a, p.sp, grid, s) : D <= 128 ? start_many<128, NQ, NP>(a, p.sp, grid, s) : start_many<256, NQ, NP>(a, p.sp, grid, s);
}

}  // namespace

int64_t attention_workspace(int64_t tokens, int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_q, int64_t max_kv) {
    const Plan p = make_plan(seqs, q_heads, kv_heads, max_q, max_kv, 0);
    return p.sp.splits > 1 ? tokens * q_heads * p.sp.splits * (dim + 1) * 4 : 0;
}

int64_t attention_groups(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t max_q, int64_t max_kv) {
    const Plan p = make_plan(seqs, q_heads, kv_heads, max_q, max_kv, 0);
    return seqs * kv_heads * p.sp.tiles * p.sp.splits;
}

hipError_t launch_attention(const AttentionArgs &a, void *work, hipStream_t s, const char **kernel) {
    Plan p = make_plan(a.t.seqs, a.q_heads, a.t.heads, a.max_q, a.max_kv, a.window);
    p.sp.o = static_cast<float *>(work);
    p.sp.lse = p.sp.o + (int64_t)a.t.tokens * a.q_heads * p.sp.splits * a.t.dim;
    if (p.few)
        *kernel = p.sp.splits > 1 ? "attention_few, attention_join" : "attention_few";
    else
        *kernel = p.sp.splits > 1 ? "attention_many, attention_join" : "attention_many";
    const unsigned grid = (unsigned)((int64_t)a.t.seqs * a.t.heads * p.sp.tiles * p.sp.splits);
    if (a.q_bf16)
        a.o_bf16 ? start<1, 1>(a, p, grid, s) : start<1, 2>(a, p, grid, s);
    else
        a.o_bf16 ? start<2, 1>(a, p, grid, s) : start<2, 2>(a, p, grid, s);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || p.sp.splits == 1) return err;
    const int64_t rows = (int64_t)a.t.seqs * a.max_q * a.q_heads;
    hipLaunchKernelGGL(k_attention_join, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, p.sp);
    return hipGetLastError();
}

}  // namespace lcml
