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

typedef float f2 __attribute__((ext_vector_type(2)));

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
        const float mm = (m == -kInf ? 0.0f : m) - (float)kPBits;
        h8 p[NP][2];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float e = __builtin_amdgcn_exp2f(t[sb][i] - mm);
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
    p.sp.tiles = (int32_t)((rows + 15) / 16);
    // tokens that a row tile can see
    int64_t span = max_kv;
    if (window > 0 && window < span && window + max_q + 64 < span) span = window + max_q + 64;
    const int64_t groups = seqs * kv_heads * p.sp.tiles, steps = (span + 63) / 64;
    int64_t splits = (1024 + groups - 1) / groups;
    if (splits > (steps + kFewWaves - 1) / kFewWaves) splits = (steps + kFewWaves - 1) / kFewWaves;
    if (splits > 128) splits = 128;
    if (splits < 1 || !p.few) splits = 1;
    p.sp.chunk = (int32_t)(((steps + splits - 1) / splits) * 64);
    p.sp.splits = (int32_t)splits;
    return p;
}

template <int DC, int NQ, int NP>
hipError_t launch_few(const AttentionArgs &a, const Split &sp, hipStream_t s) {
    const unsigned grid = (unsigned)((int64_t)a.t.heads * sp.splits * sp.tiles * a.t.seqs);
    hipLaunchKernelGGL((k_attention_few<DC, NQ, NP, kFewWaves>), dim3(grid), dim3(kFewWaves * 64), 0, s, a, sp);
    return hipGetLastError();
}

template <int DC>
hipError_t launch_few_t(const AttentionArgs &a, const Split &sp, hipStream_t s) {
    if (a.q_bf16) return a.o_bf16 ? launch_few<DC, 1, 1>(a, sp, s) : launch_few<DC, 1, 2>(a, sp, s);
    return a.o_bf16 ? launch_few<DC, 2, 1>(a, sp, s) : launch_few<DC, 2, 2>(a, sp, s);
}

}  // namespace

int64_t attention_workspace(int64_t tokens, int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_q, int64_t max_kv) {
    const Plan p = make_plan(seqs, q_heads, kv_heads, max_q, max_kv, 0);
    return p.sp.splits > 1 ? tokens * q_heads * p.sp.splits * (dim + 1) * 4 : 0;
}

hipError_t launch_attention(const AttentionArgs &a, void *work, hipStream_t s, const char **kernel) {
    Plan p = make_plan(a.t.seqs, a.q_heads, a.t.heads, a.max_q, a.max_kv, a.window);
    if (!p.few) {
        *kernel = "attention_rows";
        hipLaunchKernelGGL(k_attention_rows, dim3((unsigned)((int64_t)a.t.tokens * a.q_heads)), dim3(kThreads), 0, s, a);
        return hipGetLastError();
    }
    p.sp.o = static_cast<float *>(work);
    p.sp.lse = p.sp.o + (int64_t)a.t.tokens * a.q_heads * p.sp.splits * a.t.dim;
    *kernel = p.sp.splits > 1 ? "attention_few, attention_join" : "attention_few";
    hipError_t err = a.t.dim <= 64 ? launch_few_t<1>(a, p.sp, s) : a.t.dim <= 128 ? launch_few_t<2>(a, p.sp, s) : launch_few_t<4>(a, p.sp, s);
    if (err != hipSuccess || p.sp.splits == 1) return err;
    const int64_t rows = (int64_t)a.t.seqs * a.max_q * a.q_heads;
    hipLaunchKernelGGL(k_attention_join, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, a, p.sp);
    return hipGetLastError();
}

}  // namespace lcml
