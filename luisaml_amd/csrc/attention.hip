// attention.hip -- attention over the E4M3 KV cache (gfx950).
//
//   o = sum_j w_j v_j / sum_j w_j,   w_j = exp(scale q.k_j)
// over the tokens j that a query sees: j < kv_len, j <= its own position
// (causal), j > its position - window.  A query that sees none, or only scores
// of -inf, gives 0.
//
// One pass over the cache with a running maximum m and sum l.  Codes are
// widened to fp16, which holds every one of them, and both products run on the
// fp16 matrix instructions with fp32 sums:
//   * a query row is brought to [2^14, 2^15) by a power of two; a bf16 row is
//     then one fp16 operand, an fp32 row two (its rounding and the rest);
//   * weights are fp16 too: 11 bits, where bf16 would hold 8.  One piece where
//     the result is bf16, whose own rounding is eight times as coarse, also for
//     fp32 queries; two where it is fp32;
//   * K's page scale multiplies the scores, V's the codes as they are widened:
//     a power of two below the largest V scale so far (the widening
//     instruction takes the factor), which multiplies the end result; where
//     that largest one grows, the sums are scaled down.  All of that is exact
//     while the V scales are within 2^kSpread of each other; from the step on
//     that goes beyond, each 16-token block (which has one scale) is weighted
//     by its own maximum, multiplied by itself and added in fp32.
// Both kernels compute S^T = K Q^T and O^T = V^T P^T, so that a query row is a
// lane's column in all of S, P and O: maximum, sum and scaling are a lane's own
// but for one exchange between lanes, and S^T's accumulators are P^T's operand
// as they stand, because a reduction may run over the tokens in any order and
// V lies in the cache in just this one.
#include "kv_cache.hpp"
#include "lcml_internal.hpp"

namespace lcml {
namespace {

typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kVBits = 7;  // V's codes are held times 2^7

// ---------------------------------------------------------- operand pieces --

// four codes times a power of two, exact while the products are normal in fp16
__device__ inline h4 widen4(uint32_t w, float s) {
    const h2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, false);
    const h2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, s, true);
    return h4{a[0], a[1], b[0], b[1]};
}
__device__ inline h8 widen8(uint32_t w0, uint32_t w1, float s) {
    return __builtin_shufflevector(widen4(w0, s), widen4(w1, s), 0, 1, 2, 3, 4, 5, 6, 7);
}

// the top bits of the bytes that are the NaN codes 0x7f and 0xff
__device__ inline uint32_t nan_bits(uint32_t w) { return ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u; }
// those bytes cleared
__device__ inline uint32_t without_nan(uint32_t w) {
    const uint32_t n = nan_bits(w);
    return w & ~((n - (n >> 7)) | n);
}

__device__ inline float max_over_halves(float v) {  // lanes l and l ^ 32
    const auto a = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
    return fmaxf(bits_f32(a[0]), bits_f32(a[1]));
}
__device__ inline float sum_over_halves(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
    return bits_f32(a[0]) + bits_f32(a[1]);
}
__device__ inline float max_over_quarters(float v) {  // lanes of one l % 16
    v = max_over_halves(v);
    const auto b = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
    return fmaxf(bits_f32(b[0]), bits_f32(b[1]));
}
__device__ inline float sum_over_quarters(float v) {
    v = sum_over_halves(v);
    const auto b = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
    return bits_f32(b[0]) + bits_f32(b[1]);
}

// The power of two that brings a row's largest element to [2^14, 2^15): fp16
// then holds a bf16 element exactly down to 2^-31 of that one, and an fp32
// element in two pieces to 2^-22 of itself.  (Beside an infinity nothing else
// matters to a score.)
__device__ inline float query_factor(float amax) {
    const int e = 127 + 14 + 127 - (int)(f32_bits(amax) >> 23);
    return bits_f32((uint32_t)(e > 253 ? 253 : e) << 23);
}

__device__ inline float reciprocal(float f) { return bits_f32((254u << 23) - f32_bits(f)); }  // of a power of two

// The V scales of the steps so far, as their bits: the largest, and the
// smallest.  With codes down to 2^-9 relative to the largest scale, fp16 would
// hold all of them up to a spread of 2^22; 2^10 also keeps what the weights'
// own fp16 loses (2^-31 of the largest weight, times the largest values) below
// a bf16 result's rounding where only values of the smallest scale count.
// Beyond, a step takes longer (every other page 2^20 smaller: 32 queries over up
// to 16384 tokens 165 us for 124, a prompt of 8192 1372 for 610).
constexpr int kSpread = 10;
struct Scales {
    uint32_t top = 0, low = 0x7f800000u;
    __device__ inline void take(const uint32_t (&vs)[4]) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            top = vs[q] > top ? vs[q] : top;
            low = vs[q] && vs[q] < low ? vs[q] : low;
        }
    }
    __device__ inline bool apart() const { return (int)(top >> 23) - (int)(low >> 23) > kSpread; }
};

// How a block of maximum mb and sum lb joins a row of maximum m and sum l whose
// result is already divided by l: the factors of the row's result and of the
// block's products.
__device__ inline void join_block(float &m, float &l, float mb, float lb, float *keep, float *add) {
    const float top = fmaxf(m, mb);
    const float fa = m == top ? l : l * __builtin_amdgcn_exp2f(m - top);
    const float wb = mb == top ? 1.0f : __builtin_amdgcn_exp2f(mb - top), fb = lb * wb;
    m = top, l = fa + fb;
    const float inv = 1.0f / l;
    *keep = fb == 0.0f ? 1.0f : fa * inv;  // nothing to add: the row as it is
    *add = fb == 0.0f ? 0.0f : wb * inv;
}

// vs / vref times 2^kVBits, powers of two as their bits
__device__ inline float v_ratio(uint32_t vs, uint32_t vref) {
    const int e = (int)(vs >> 23) - (int)(vref >> 23) + 127 + kVBits;
    return bits_f32((uint32_t)(e < 1 ? 1 : e) << 23);
}

// A weight is 2^(t - m) times a power of two that keeps it in fp16's range.
// One piece: times 2^6 in the exponential's argument, and m may stay up to 8
// below the maximum (sums are scaled by a rising maximum in one step of two
// otherwise, and that is a fifth of the vector work); 11 bits down to 2^-20 of
// the largest weight, an error of 2^-31 of it below.  Two pieces: times 2^14
// after the exponential (in its argument, the rounding of a sum near 14 would
// cost three bits), and m is the maximum.
template <int NP>
__device__ constexpr float weight_slack() {
    return NP == 1 ? 8.0f : 0.0f;
}
template <int NP>
__device__ inline float weight_base(float m) {
    m = m == -kInf ? 0.0f : m;
    return NP == 1 ? m - 6.0f : m;
}
template <int NP>
__device__ inline float weight_scale(float e) {
    return NP == 1 ? e : e * 0x1p14f;
}
// l plus a pair of weights: as rounded where one piece is all there is
template <int NP>
__device__ inline float add_weights(float l, f2 e, h2 eh) {
    return NP == 1 ? __builtin_amdgcn_fdot2(eh, h2{(_Float16)1.0f, (_Float16)1.0f}, l, false) : l + (e[0] + e[1]);
}

// eight elements of a query at any element-aligned address, as fp32
struct __attribute__((packed, aligned(2))) Q16 {
    uint16_t v[8];
};
struct __attribute__((packed, aligned(4))) Q32 {
    float v[8];
};
template <bool BF16>
__device__ inline void load_q8(const void *q, int64_t i, float *x) {
    if constexpr (BF16) {
        const Q16 w = *reinterpret_cast<const Q16 *>(static_cast<const uint16_t *>(q) + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = bits_f32((uint32_t)w.v[e] << 16);
    } else {
        const Q32 w = *reinterpret_cast<const Q32 *>(static_cast<const float *>(q) + i);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = w.v[e];
    }
}

// eight elements times f, as one piece or two; zeros where the row has none
template <int NQ>
__device__ inline void to_pieces(const float *x, float f, bool in, h8 *hi, h8 *lo) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const f2 v{x[e] * f, x[e + 1] * f};
        const h2 p = __builtin_convertvector(v, h2);
        (*hi)[e] = p[0], (*hi)[e + 1] = p[1];
        if constexpr (NQ == 2) {
            // an infinity is all in its first piece: the rest of it is no NaN
            const f2 rest{fabsf(v[0]) == kInf ? 0.0f : v[0] - (float)p[0], fabsf(v[1]) == kInf ? 0.0f : v[1] - (float)p[1]};
            const h2 q = __builtin_convertvector(rest, h2);
            (*lo)[e] = q[0], (*lo)[e + 1] = q[1];
        }
    }
    const h8 zero{0, 0, 0, 0, 0, 0, 0, 0};
    *hi = in ? *hi : zero;
    if constexpr (NQ == 2) *lo = in ? *lo : zero;
}

// 16 bytes that this call reads once: non-temporal (32 queries over up to 16384
// tokens, 619 MB: 134 us without, 123 with)
__device__ inline u4 load_once(const uint8_t *p) { return __builtin_nontemporal_load(reinterpret_cast<const u4 *>(p)); }

struct __attribute__((packed, aligned(2))) O16 {
    uint16_t v[4];
};
struct __attribute__((packed, aligned(4))) O32 {
    float v[4];
};
template <bool BF16>
__device__ inline void store_o4(void *o, int64_t i, f4 v) {
    if constexpr (BF16)
        *reinterpret_cast<O16 *>(static_cast<uint16_t *>(o) + i) =
            O16{{bf16_rne(v[0]), bf16_rne(v[1]), bf16_rne(v[2]), bf16_rne(v[3])}};
    else
        *reinterpret_cast<O32 *>(static_cast<float *>(o) + i) = O32{{v[0], v[1], v[2], v[3]}};
}

// A 16-token block of the cache.
struct Block {
    uint32_t lo, hi;  // its number, in units of 16 * D bytes
    uint32_t ks, vs;  // its page's scales as bits; vs 0: no such page
};

// the page of tokens tok .. tok+15 of a sequence, none (-1) from `end` on
__device__ inline int32_t find_page(const AttentionArgs &a, int32_t b, int32_t tok, int32_t end) {
    return tok < end ? page_of(a.t, b, tok >> a.t.tshift) : -1;
}
__device__ inline Block block_of(const AttentionArgs &a, int32_t head, int32_t tok, int32_t page) {
    Block r{0, 0, 0, 0};
    if (page >= 0) {
        const uint64_t at = (uint64_t)page * a.t.heads + head;
        const uint64_t blk = (at << (a.t.tshift - 4)) + ((tok >> 4) & ((1 << (a.t.tshift - 4)) - 1));
        r.lo = (uint32_t)blk, r.hi = (uint32_t)(blk >> 32);
        r.ks = f32_bits(a.ks[at]), r.vs = f32_bits(a.vs[at]);
    }
    return r;
}
__device__ inline uint32_t lane_of(uint32_t v, int i) { return (uint32_t)__builtin_amdgcn_readlane((int)v, i); }

// n / d for n < 2^31, d >= 1, by a multiplication: with 2^(k-1) < d <= 2^k and
// m = ceil(2^(31+k) / d), n m / 2^(31+k) exceeds n / d by less than 1 / d.  The
// divisions of a workgroup's start took a third of a short call.
struct Divider {
    uint32_t d, m, s;
    static Divider of(int64_t d) {
        uint32_t k = 0;
        while (((int64_t)1 << k) < d) ++k;
        return Divider{(uint32_t)d, d == 1 ? 0u : (uint32_t)((((unsigned __int128)1 << (31 + k)) + d - 1) / d), k ? k - 1 : 0};
    }
    __host__ __device__ uint32_t div(uint32_t n) const {
        return d == 1 ? n : (uint32_t)(((uint64_t)n * m) >> 32) >> s;
    }
};

// How a row's tokens are divided: `splits` parts of `chunk` tokens; with more
// than one, part results (normalised) and the base-2 logarithms of their
// weights go to the workspace, [token * q_heads + head][split].
struct Split {
    int32_t splits, chunk, tiles;  // tiles: row tiles of one sequence and KV head
    int32_t group;                 // q heads of a KV head
    float *o, *lse;
    Divider by_splits, by_tiles, by_heads, by_group, by_per;  // by_per: of tiles * splits
};

// positions that query i of a sequence sees: lo .. hi-1, neither falling with i
__device__ inline void sees(const AttentionArgs &a, const SeqRows &s, int32_t i, int32_t *lo, int32_t *hi) {
    const int32_t pos = s.pos0 + i, w = (int32_t)a.window;  // below 2^31; 0: no window
    const int32_t h = a.causal && pos < s.len ? pos + 1 : s.len;
    const int32_t l = w > 0 && pos >= w ? pos - w + 1 : 0;
    *hi = h > 0 ? h : 0;
    *lo = l < *hi ? l : *hi;
}

// the part of positions lo .. hi-1 that is this workgroup's, from a multiple of
// 64 on, in steps of 64
struct Part {
    int32_t start, end, steps;
};
__device__ inline Part part_of(const AttentionArgs &a, const Split &sp, int32_t split, int32_t lo, int32_t hi) {
    const int64_t from = (lo & ~63) + (int64_t)split * sp.chunk;
    int64_t to = split + 1 < sp.splits ? from + sp.chunk : hi;
    to = to < hi ? to : hi;
    if (from >= to || a.t.pages == 0) return Part{0, 0, 0};
    return Part{(int32_t)from, (int32_t)to, (int32_t)((to - from + 63) >> 6)};
}

// ----------------------------------------------- few rows for each KV head --
//
// One workgroup: up to 16 rows (queries x heads of the group) of one sequence
// and KV head, over one part of the tokens; its wavefronts take turns of 64
// tokens, straight from memory into registers, and join at the end.
// 16x16x32 instructions.
//
// Bound by the cache's bytes: 16 KB of loads a wavefront under way (212
// registers, two wavefronts a SIMD; three spilled and took 213 us where this
// takes 120, eight in a workgroup 166).  32 queries of 32 heads over up to 16384
// tokens of 8 KV heads of 128, 619 MB: 120 us, 5.2 TB/s; fp32 queries and
// results 130.  One over 500 tokens: 8.4 us, five dependent round trips to
// memory (lengths, table, scales, codes, the join's LDS); fp32 10.
template <int DC, int NQ, int NP, int NW>
__global__ __launch_bounds__(NW * 64, DC <= 2 ? 2 : 1) void k_attention_few(AttentionArgs a, Split sp) {
    constexpr int DP = DC * 64, kPitch = DP + 4;
    __shared__ float red_m[NW][16], red_l[NW][16];
    __shared__ __attribute__((aligned(16))) float buf[NW][16][kPitch];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t D = a.t.dim, G = sp.group;
    const uint32_t id0 = blockIdx.x, id1 = sp.by_heads.div(id0), id2 = sp.by_splits.div(id1);
    const int32_t head = id0 - id1 * a.t.heads, split = id1 - id2 * sp.splits;
    const int32_t b = sp.by_tiles.div(id2), tile = id2 - b * sp.tiles;
    const SeqRows s = seq_rows(a.t, b);
    const int32_t rows = (s.n < (int32_t)a.max_q ? s.n : (int32_t)a.max_q) * G;
    const int32_t row0 = tile * 16;
    if (row0 >= rows) return;
    const int32_t last = rows - row0 < 16 ? rows - 1 : row0 + 15;  // of the tile
    const int32_t row = row0 + r < last ? row0 + r : last;         // this lane's
    const int32_t qi = sp.by_group.div(row), qh = head * G + row - qi * G;
    int32_t lo, hi, lo_min, hi_min, lo_max, hi_max;
    sees(a, s, qi, &lo, &hi);
    sees(a, s, sp.by_group.div(row0), &lo_min, &hi_min);
    sees(a, s, sp.by_group.div(last), &lo_max, &hi_max);
    const Part part = part_of(a, sp, split, lo_min, hi_max);
    const int64_t out_row = ((int64_t)s.row0 + qi) * a.q_heads + qh;
    if (part.steps == 0 && sp.splits > 1) {
        if (threadIdx.x < 16 && row0 + r <= last) sp.lse[out_row * sp.splits + split] = -kInf;
        return;
    }
    const int32_t mine = (part.steps - wave + NW - 1) / NW;

    Block blk;
    auto find = [&](int32_t k) {  // lane i: block i of the wavefront's next 16 steps
        const int32_t tok = part.start + (((k + (lane >> 2)) * NW + wave) << 6) + (lane & 3) * 16;
        blk = block_of(a, head, tok, find_page(a, b, tok, part.end));
    };
    u4 kk[4][DC], vv[4][DC];
    auto base = [&](const uint8_t *p, int32_t k, int sb) {
        const int i = (k & 15) * 4 + sb;
        return p + (lane_of(blk.lo, i) | (uint64_t)lane_of(blk.hi, i) << 32) * (uint64_t)(16 * D);
    };
    const u4 zero{0, 0, 0, 0};
    auto issue_k = [&](int32_t k) {
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            const uint8_t *p = base(a.k, k, sb);
#pragma unroll
            for (int j = 0; j < DC; ++j)
                kk[sb][j] = (4 * j + g) * 16 < D ? load_once(p + (4 * j + g) * 256 + r * 16) : zero;
        }
    };
    auto issue_v = [&](int32_t k) {
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            const uint8_t *p = base(a.v, k, sb) + g * 4 * D;
#pragma unroll
            for (int j = 0; j < DC; ++j)
                vv[sb][j] = 64 * j + 4 * r < D ? load_once(p + (64 * j + 4 * r) * 4) : zero;
        }
    };
    // the row's query in the operand's order: pieces 4 j + g of 16 elements
    h8 qf[NQ][DC][2];
    float cq;
    {
        const int64_t at = ((int64_t)s.row0 + qi) * a.q_token + (int64_t)qh * a.q_head;
        float x[DC][2][8], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int d = 16 * (4 * j + g) + 8 * h;
                load_q8<NQ == 1>(a.q, at + (d < D ? d : 0), x[j][h]);
            }
        if (mine > 0) {
            find(0);
            issue_k(0);
            issue_v(0);
        }
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[j][h][e]));
        const float f = query_factor(max_over_quarters(amax));
        cq = a.scale * kLog2e * reciprocal(f);
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                to_pieces<NQ>(x[j][h], f, 16 * (4 * j + g) < D, &qf[0][j][h], &qf[NQ - 1][j][h]);
    }

    f4 o[DC][4];  // columns 64 j + 16 g + 4 i + c in o[j][c][i]
#pragma unroll
    for (int j = 0; j < DC; ++j)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[j][c] = f4{0.f, 0.f, 0.f, 0.f};
    float m = -kInf, l = 0.0f;
    uint32_t vref = 0;
    auto scale_o = [&](float f) {
#pragma unroll
        for (int j = 0; j < DC; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[j][c] *= f;
    };

    bool nan = false;
    uint32_t ks[4], vs[4];
    Scales scales;
    // one step's scores; then the next one's K is on its way
    auto products = [&](int32_t k, f4 (&t)[4]) {
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            t[sb] = f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const h8 kh = widen8(kk[sb][j][2 * h], kk[sb][j][2 * h + 1], 1.0f);
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
                        t[sb] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qf[q][j][h], t[sb], 0, 0, 0);
                }
        }
        if (k + 1 < mine) {
            if (((k + 1) & 15) == 0) find(k + 1);
            issue_k(k + 1);
        }
    };
    // hides what the lane's row does not see; V's NaN codes count as zeros for now
    auto mask = [&](int32_t tok, f4 (&t)[4]) {
        uint32_t bad = 0;
        const uint32_t from = tok + 4 * g - lo;
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            const uint32_t span = vs[sb] ? hi - lo : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) t[sb][i] = from + 16 * sb + i < span ? t[sb][i] : -kInf;
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) bad |= nan_bits(vv[sb][j][c]);
        }
        if (__builtin_amdgcn_ballot_w64(bad != 0) != 0) {  // NaN codes: of tokens that a row sees?
            bad = 0;
            const uint32_t all = tok + 4 * g - lo_min;
#pragma unroll
            for (int sb = 0; sb < 4; ++sb) {
                const uint32_t span = vs[sb] ? hi_max - lo_min : 0;
                uint32_t seen = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) seen |= all + 16 * sb + i < span ? 0x80u << (8 * i) : 0u;
#pragma unroll
                for (int j = 0; j < DC; ++j)
#pragma unroll
                    for (int y = 0; y < 4; ++y) {
                        bad |= nan_bits(vv[sb][j][y]) & seen;
                        vv[sb][j][y] = without_nan(vv[sb][j][y]);
                    }
            }
            nan = nan || __builtin_amdgcn_ballot_w64(bad != 0) != 0;
        }
    };
    // one step; MASKED: some rows do not see all of its tokens
    auto step = [&](int32_t k, int32_t tok, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        f4 t[4];
        products(k, t);
        if constexpr (MASKED) mask(tok, t);
        float mx = m, c[4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            c[sb] = cq * bits_f32(ks[sb]);
            const float b = fmaxf(fmaxf(t[sb][0], t[sb][1]), fmaxf(t[sb][2], t[sb][3]));
            // a factor of 0 (scales below the range) must not make a NaN of a hidden token's -inf
            mx = fmaxf(mx, MASKED && b == -kInf ? b : b * c[sb]);
        }
        mx = max_over_quarters(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m + weight_slack<NP>()) != 0) {
            const float f = mx > m ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
            l *= f;
            scale_o(f);
            m = mx > m ? mx : m;
        }
        if (scales.top > vref) {
            const int e = (int)(vref >> 23) - (int)(scales.top >> 23) + 127;  // vref 0: sums of 0
            scale_o(bits_f32((uint32_t)(e < 0 ? 0 : e) << 23));
            vref = scales.top;
        }
        const float mm = weight_base<NP>(m);
        h8 p[NP][2];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                f2 e;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    float v = fmaf(t[sb][i + y], c[sb], -mm);
                    if (MASKED) v = t[sb][i + y] == -kInf ? -kInf : v;
                    e[y] = weight_scale<NP>(__builtin_amdgcn_exp2f(v));
                }
                const h2 eh = __builtin_convertvector(e, h2);
                l = add_weights<NP>(l, e, eh);
                const int at0 = (sb & 1) * 4 + i;
                p[0][sb >> 1][at0] = eh[0], p[0][sb >> 1][at0 + 1] = eh[1];
                if constexpr (NP == 2) {
                    const h2 el = __builtin_convertvector(f2{e[0] - (float)eh[0], e[1] - (float)eh[1]}, h2);
                    p[NP - 1][sb >> 1][at0] = el[0], p[NP - 1][sb >> 1][at0 + 1] = el[1];
                }
            }
        float ratio[4];
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) ratio[sb] = v_ratio(vs[sb], vref);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const h8 va = __builtin_shufflevector(widen4(vv[2 * h][j][y], ratio[2 * h]),
                                                          widen4(vv[2 * h + 1][j][y], ratio[2 * h + 1]), 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
                    for (int q = 0; q < NP; ++q)
                        o[j][y] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[q][h], o[j][y], 0, 0, 0);
                }
        if (k + 1 < mine) issue_v(k + 1);
    };
    // one step where V's scales are far apart; o is the result so far, divided
    // by l, and l the row's whole sum
    auto step_apart = [&](int32_t k, int32_t tok) {
        f4 t[4];
        products(k, t);
        mask(tok, t);
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            if (!vs[sb]) continue;
            const float c = cq * bits_f32(ks[sb]), s = bits_f32(vs[sb]);
            const float b = fmaxf(fmaxf(t[sb][0], t[sb][1]), fmaxf(t[sb][2], t[sb][3]));
            const float mb = max_over_quarters(b == -kInf ? b : b * c), mm = weight_base<NP>(mb);
            float lb = 0.0f, keep, add;
            h8 p[NP];  // this block's weights, and zeros for the operand's other four
#pragma unroll
            for (int q = 0; q < NP; ++q) p[q] = h8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                f2 e;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float x = t[sb][i + y];
                    e[y] = weight_scale<NP>(__builtin_amdgcn_exp2f(x == -kInf ? x : fmaf(x, c, -mm)));
                }
                const h2 eh = __builtin_convertvector(e, h2);
                lb = add_weights<NP>(lb, e, eh);
                p[0][i] = eh[0], p[0][i + 1] = eh[1];
                if constexpr (NP == 2) {
                    const h2 el = __builtin_convertvector(f2{e[0] - (float)eh[0], e[1] - (float)eh[1]}, h2);
                    p[NP - 1][i] = el[0], p[NP - 1][i + 1] = el[1];
                }
            }
            join_block(m, l, mb, sum_over_quarters(lb), &keep, &add);
#pragma unroll
            for (int j = 0; j < DC; ++j)
#pragma unroll
                for (int y = 0; y < 4; ++y) {
                    const h8 va = __builtin_shufflevector(widen4(vv[sb][j][y], 1.0f), h4{0, 0, 0, 0}, 0, 1, 2, 3, 4, 5, 6, 7);
                    f4 x{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int q = 0; q < NP; ++q) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, p[q], x, 0, 0, 0);
                    o[j][y] = o[j][y] * keep + x * add * s;
                }
        }
        if (k + 1 < mine) issue_v(k + 1);
    };
    auto scales_of = [&](int32_t k) {
#pragma unroll
        for (int sb = 0; sb < 4; ++sb) {
            ks[sb] = lane_of(blk.ks, (k & 15) * 4 + sb);
            vs[sb] = lane_of(blk.vs, (k & 15) * 4 + sb);
        }
        scales.take(vs);
    };
    // steps that all rows see whole, in a loop of their own
    int32_t k = 0;
    for (; k < mine; ++k) {
        int32_t tok;
        for (; k < mine; ++k) {
            tok = part.start + ((k * NW + wave) << 6);
            scales_of(k);
            if (!(tok >= lo_max && tok + 64 <= hi_min && vs[0] && vs[1] && vs[2] && vs[3]) || scales.apart()) break;
            step(k, tok, std::false_type{});
        }
        if (k >= mine || scales.apart()) break;
        step(k, tok, std::true_type{});
    }
    l = sum_over_quarters(l);
    const bool apart = k < mine;
    if (__builtin_expect(apart, 0)) {
        scale_o(l == 0.0f ? 0.0f : 1.0f / (1 << kVBits) / l);
        scale_o(bits_f32(vref));
        for (; k < mine; ++k) {
            scales_of(k);
            step_apart(k, part.start + ((k * NW + wave) << 6));
        }
    }

    // join the wavefronts
    if (g == 0) red_m[wave][r] = m, red_l[wave][r] = l;
    __syncthreads();
    float top = -kInf, sum = 0.0f;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, red_m[w][r]);
    auto weight = [&](float v) { return v == top ? 1.0f : __builtin_amdgcn_exp2f(v - top); };
#pragma unroll
    for (int w = 0; w < NW; ++w) sum += red_l[w][r] * weight(red_m[w][r]);
    // (the scale last: with a factor of the other two it could leave fp32's range)
    scale_o(sum == 0.0f ? 0.0f : weight(m) / sum * (apart ? l : 1.0f / (1 << kVBits)));
    if (!apart) scale_o(bits_f32(vref));
#pragma unroll
    for (int j = 0; j < DC; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
            *reinterpret_cast<f4 *>(&buf[wave][r][64 * j + 16 * g + 4 * i]) = f4{o[j][0][i], o[j][1][i], o[j][2][i], o[j][3][i]};
    if (__builtin_expect(nan, 0))  // V's NaN codes reach the rows that see their token, and no others
        for (int32_t k = 0; k < mine; ++k) {
            const int32_t tok = part.start + ((k * NW + wave) << 6);
            for (int32_t j = tok > lo_min ? tok : lo_min; j < tok + 64 && j < part.end; ++j) {
                const Block w = block_of(a, head, j, find_page(a, b, j, part.end));
                if (!w.vs) continue;
                const uint8_t *p = a.v + (w.lo | (uint64_t)w.hi << 32) * (uint64_t)(16 * D);
                for (int32_t d = lane; d < D; d += 64)
                    if ((p[v_place(j & 15, d, D)] & 0x7f) == 0x7f)
                        for (int rr = 0; rr < 16; ++rr)
                            if (j >= (int32_t)lane_of(lo, rr) && j < (int32_t)lane_of(hi, rr)) buf[wave][rr][d] = __builtin_nanf("");
            }
        }
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
            store_o4<NP == 1>(a.o, ((int64_t)s.row0 + i) * a.o_token + (int64_t)h * a.o_head + d, v);
    }
}

// ---------------------------------------------------------------- many rows --
//
// One workgroup: 128 rows (queries x heads of the group) of one sequence and
// KV head, 32 for each wavefront, over one part of the tokens, 64 a step.
// Each wavefront brings 16 of a step's tokens into LDS, K as codes and V
// widened: bound by the vector ALU and the matrix cores in turn, the kernel
// shares the widening of V (64 conversions a wavefront and step would be
// repeated by each of the four), and reads K's codes in half the bytes (K
// widened as well: 2% slower).  32x32x16 instructions.
//
// A prompt of 8192 tokens, 32 heads over 8 of 128, 0.55 TFLOP: 610 us, 900
// TFLOP/s, where a product of 8192^3 in bf16 reaches 1190.  A step's 32 matrix
// instructions take 1024 cycles of a SIMD, its 320 vector ones 1280, and two
// wavefronts a SIMD overlap them to two thirds of the sum.  (Two groups of
// wavefronts half a step apart: 1075 us, for the registers spilled.)  D > 128
// has one wavefront a SIMD, and nothing to overlap LDS reads with: 220 TFLOP/s
// on a prompt of 2048 tokens, 260 on one of 4000.  What happens around a step is
// in three loops, always inlined: out of line, its registers lie in scratch.
constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;

template <int DP, bool EXACT, int NQ, int NP>
__global__ __launch_bounds__(kManyWaves * 64, DP <= 128 ? 2 : 1) void k_attention_many(AttentionArgs a, Split sp) {
    constexpr int KJ = DP / 32;  // pairs of 16-element pieces of K
    constexpr int MT = DP / 32;  // tiles of 32 columns of V
    constexpr int PL = DP / 64;  // 16-byte loads for a lane of a 16-token block
    // LDS holds DP columns: past D, zeros for K and anything for V, whose
    // columns there are not stored.  K: [4 blocks][DP / 16][16 tokens][16].  V:
    // [4 blocks][2][DP][8 tokens], in the halves the groups 0 and 2, 1 and 3 of
    // four tokens, and column 4 u + e in place e * DP / 4 + u: what the lanes
    // write and what they read is contiguous.
    __shared__ __attribute__((aligned(16))) uint8_t stage_k[2][64 * DP];
    __shared__ __attribute__((aligned(16))) _Float16 stage_v[2][64 * DP];
    __shared__ uint32_t has_nan;  // V, in steps that some row does not see whole
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t D = EXACT ? DP : a.t.dim, G = sp.group;
    // workgroups of one sequence and KV head on one XCD (blockIdx modulo 8),
    // whose L2 then holds their K and V; the longest rows first
    const uint32_t pairs = (uint32_t)a.t.seqs * a.t.heads, per = (uint32_t)sp.tiles * sp.splits;
    const bool by_xcd = pairs % 8 == 0;
    const uint32_t id = by_xcd ? blockIdx.x / 8 : blockIdx.x, over = sp.by_per.div(id), rest = id - over * per;
    const uint32_t pair = by_xcd ? blockIdx.x % 8 + 8 * over : over;
    const int32_t b = sp.by_heads.div(pair), head = pair - b * a.t.heads;
    const int32_t place = sp.by_splits.div(rest), split = rest - place * sp.splits, tile = sp.tiles - 1 - place;
    const SeqRows s = seq_rows(a.t, b);
    const int32_t rows = (s.n < (int32_t)a.max_q ? s.n : (int32_t)a.max_q) * G, row0 = tile * kManyRows;
    if (row0 >= rows) return;
    const int32_t last = rows - row0 < kManyRows ? rows - 1 : row0 + kManyRows - 1;
    // this wavefront's rows and this lane's
    const int32_t w0 = row0 + 32 * wave < last ? row0 + 32 * wave : last, w1 = w0 + 31 < last ? w0 + 31 : last;
    const bool live = row0 + 32 * wave + r <= last;
    const int32_t row = live ? row0 + 32 * wave + r : w1;
    const int32_t qi = sp.by_group.div(row), qh = head * G + row - qi * G;
    // tokens that this lane's row sees, that any row sees and that all do, of
    // the workgroup and (any) of the wavefront
    int32_t lo, hi, lo_min, hi_min, lo_max, hi_max, w_lo, w_hi, unused;
    sees(a, s, qi, &lo, &hi);
    sees(a, s, sp.by_group.div(row0), &lo_min, &hi_min);
    sees(a, s, sp.by_group.div(last), &lo_max, &hi_max);
    sees(a, s, sp.by_group.div(w0), &w_lo, &unused);
    sees(a, s, sp.by_group.div(w1), &unused, &w_hi);
    const Part part = part_of(a, sp, split, lo_min, hi_max);
    const int64_t out_row = ((int64_t)s.row0 + qi) * a.q_heads + qh;
    if (part.steps == 0 && sp.splits > 1) {
        if (h == 0 && live) sp.lse[out_row * sp.splits + split] = -kInf;
        return;
    }

    // lane i: block i of 16 steps; the next 16 steps' pages and blocks are
    // looked up while these are worked on
    Block blk, next;
    int32_t next_page = -1;
    auto token_of = [&](int32_t k) { return part.start + ((k + (lane >> 2)) << 6) + (lane & 3) * 16; };
    uint32_t ks[4], vs[4], ks_next[4], vs_next[4];
    bool whole, whole_next = false;  // whether every row sees all of a step's tokens
    Scales scales;                   // of the steps fetched so far, the same for all wavefronts
    // this wavefront's block of step k
    u4 kr[PL], vr[PL];
    auto fetch = [&](int32_t k) __attribute__((always_inline)) {
        const int i = (k & 15) * 4;
#pragma unroll
        for (int q = 0; q < 4; ++q) ks_next[q] = lane_of(blk.ks, i + q), vs_next[q] = lane_of(blk.vs, i + q);
        const int32_t tok = part.start + (k << 6);
        uint32_t least = vs_next[0] < vs_next[1] ? vs_next[0] : vs_next[1];
        least = vs_next[2] < least ? vs_next[2] : least;
        least = vs_next[3] < least ? vs_next[3] : least;
        whole_next = tok >= lo_max && tok + 64 <= hi_min && least;
        scales.take(vs_next);
        const uint64_t at = (lane_of(blk.lo, i + wave) | (uint64_t)lane_of(blk.hi, i + wave) << 32) * (uint64_t)(16 * D);
        const uint8_t *pk = a.k + at, *pv = a.v + at;
#pragma unroll
        for (int x = 0; x < PL; ++x) {
            const bool in = EXACT || 64 * x + lane < D;
            kr[x] = in ? *reinterpret_cast<const u4 *>(pk + (64 * x + lane) * 16) : u4{0, 0, 0, 0};
            vr[x] = in ? *reinterpret_cast<const u4 *>(pv + (64 * x + lane) * 16) : u4{0, 0, 0, 0};
        }
    };
    uint32_t vref = 0;  // the largest V scale up to the step that is worked on
    auto deposit = [&](int32_t k, int buf) __attribute__((always_inline)) {
        const uint32_t mine = wave == 0 ? vs_next[0] : wave == 1 ? vs_next[1] : wave == 2 ? vs_next[2] : vs_next[3];
        const float ratio = scales.apart() ? 1.0f : v_ratio(mine, scales.top);
        if (__builtin_expect(!whole_next, 0)) {
            // what lies past the last token counts as zeros, and so do NaN codes
            // for now
            const int32_t left = part.end - (part.start + (k << 6) + 16 * wave);
            uint32_t bad = 0;
#pragma unroll
            for (int x = 0; x < PL; ++x) {
                const int32_t n = left - (64 * x + lane) / (D >> 2) * 4;
                const uint32_t keep = n >= 4 ? ~0u : n <= 0 ? 0u : (1u << (8 * n)) - 1;
                vr[x] &= u4{keep, keep, keep, keep};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    bad |= nan_bits(vr[x][c]);
                    vr[x][c] = without_nan(vr[x][c]);
                }
            }
            if (bad) has_nan = 1;
        }
#pragma unroll
        for (int x = 0; x < PL; ++x) {
            const int u = 64 * x + lane, g = u / (D >> 2), d4 = u - g * (D >> 2);  // a group of tokens, columns 4 d4 ..
            *reinterpret_cast<u4 *>(&stage_k[buf][wave * 16 * DP + u * 16]) = kr[x];  // zeros past D
            if (EXACT || u < D)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *reinterpret_cast<h4 *>(&stage_v[buf][wave * 16 * DP + (g & 1) * 8 * DP + (e * (DP / 4) + d4) * 8 + (g >> 1) * 4]) =
                        widen4(vr[x][e], ratio);
        }
    };
    if (part.steps > 0) {
        blk = block_of(a, head, token_of(0), find_page(a, b, token_of(0), part.end));
        fetch(0);
    }

    h8 qf[NQ][KJ][2];  // pieces 2 j + h of 16 elements of the row's query
    float cq;
    {
        const int64_t at = ((int64_t)s.row0 + qi) * a.q_token + (int64_t)qh * a.q_head;
        float x[KJ][2][8], amax = 0.0f;
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int d = 32 * j + 16 * h + 8 * u;
                load_q8<NQ == 1>(a.q, at + (EXACT || d < D ? d : 0), x[j][u]);
            }
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[j][u][e]));
        const float f = query_factor(max_over_halves(amax));
        cq = a.scale * kLog2e * reciprocal(f);
#pragma unroll
        for (int j = 0; j < KJ; ++j)
#pragma unroll
            for (int u = 0; u < 2; ++u)
                to_pieces<NQ>(x[j][u], f, EXACT || 32 * j + 16 * h < D, &qf[0][j][u], &qf[NQ - 1][j][u]);
    }

    f16v o[MT];  // tile t, row i: place 32 t + 8 (i / 4) + 4 h + i % 4 of V's columns
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    auto column = [&](int t, int i) {
        const int p = 32 * t + 8 * (i >> 2) + 4 * h + (i & 3);
        return 4 * (p % (DP / 4)) + p / (DP / 4);
    };
    float m = -kInf, l = 0.0f;
    auto scale_o = [&](float f) {
#pragma unroll
        for (int t = 0; t < MT; ++t) o[t] *= f;
    };

    // one step's scores from LDS; MASKED: some rows do not see all of its tokens
    auto scores = [&](int32_t tok, int buf, f16v (&t)[2], float (&c)[4], auto masked) __attribute__((always_inline)) {
        const uint8_t *sk = stage_k[buf];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
#pragma unroll
            for (int i = 0; i < 16; ++i) t[q][i] = 0.0f;
            const uint8_t *p = sk + (2 * q + (r >> 4)) * 16 * DP + h * 256 + (r & 15) * 16;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                const u4 w = *reinterpret_cast<const u4 *>(p + j * 512);
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const h8 kh = widen8(w[2 * u], w[2 * u + 1], 1.0f);
#pragma unroll
                    for (int x = 0; x < NQ; ++x)
                        t[q] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kh, qf[x][j][u], t[q], 0, 0, 0);
                }
            }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) c[q] = cq * bits_f32(ks[q]);
        if constexpr (decltype(masked)::value) {
            const uint32_t from = tok + 4 * h - lo;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t span = vs[q] ? hi - lo : 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = (q & 1) * 8 + i;
                    t[q >> 1][at] = from + 16 * q + 8 * (i >> 2) + (i & 3) < span ? t[q >> 1][at] : -kInf;
                }
            }
        }
    };
    auto step = [&](int32_t tok, int buf, auto masked) {
        constexpr bool MASKED = decltype(masked)::value;
        const _Float16 *sv = stage_v[buf];
        f16v t[2];
        float c[4];
        scores(tok, buf, t, c, masked);
        float mx = m;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float b = t[q >> 1][(q & 1) * 8];
#pragma unroll
            for (int i = 1; i < 8; ++i) b = fmaxf(b, t[q >> 1][(q & 1) * 8 + i]);
            // a factor of 0 (scales below the range) must not make a NaN of a hidden token's -inf
            mx = fmaxf(mx, MASKED && b == -kInf ? b : b * c[q]);
        }
        mx = max_over_halves(mx);
        if (__builtin_amdgcn_ballot_w64(mx > m + weight_slack<NP>()) != 0) {
            const float f = mx > m ? __builtin_amdgcn_exp2f(m - mx) : 1.0f;
            l *= f;
            scale_o(f);
            m = mx > m ? mx : m;
        }
        const float mm = weight_base<NP>(m);
        h8 p[NP][4];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                f2 e;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float x = t[q >> 1][(q & 1) * 8 + i + y];
                    float v = fmaf(x, c[q], -mm);
                    if (MASKED) v = x == -kInf ? x : v;
                    e[y] = weight_scale<NP>(__builtin_amdgcn_exp2f(v));
                }
                const h2 eh = __builtin_convertvector(e, h2);
                l = add_weights<NP>(l, e, eh);
                p[0][q][i] = eh[0], p[0][q][i + 1] = eh[1];
                if constexpr (NP == 2) {
                    const h2 el = __builtin_convertvector(f2{e[0] - (float)eh[0], e[1] - (float)eh[1]}, h2);
                    p[NP - 1][q][i] = el[0], p[NP - 1][q][i + 1] = el[1];
                }
            }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int y = 0; y < MT; ++y) {
                const h8 va = *reinterpret_cast<const h8 *>(sv + q * 16 * DP + h * 8 * DP + (32 * y + r) * 8);
#pragma unroll
                for (int z = 0; z < NP; ++z) o[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, p[z][q], o[y], 0, 0, 0);
            }
    };
    // one step where V's scales are far apart (its codes lie in LDS as they are);
    // o is the result so far, divided by l, and l the row's whole sum
    auto step_apart = [&](int32_t tok, int buf) __attribute__((always_inline)) {
        const _Float16 *sv = stage_v[buf];
        f16v t[2];
        float c[4];
        scores(tok, buf, t, c, std::true_type{});
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (!vs[q]) continue;
            float b = t[q >> 1][(q & 1) * 8], lb = 0.0f, keep, add;
#pragma unroll
            for (int i = 1; i < 8; ++i) b = fmaxf(b, t[q >> 1][(q & 1) * 8 + i]);
            const float mb = max_over_halves(b == -kInf ? b : b * c[q]), mm = weight_base<NP>(mb), s = bits_f32(vs[q]);
            h8 p[NP];
#pragma unroll
            for (int i = 0; i < 8; i += 2) {
                f2 e;
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    const float x = t[q >> 1][(q & 1) * 8 + i + y];
                    e[y] = weight_scale<NP>(__builtin_amdgcn_exp2f(x == -kInf ? x : fmaf(x, c[q], -mm)));
                }
                const h2 eh = __builtin_convertvector(e, h2);
                lb = add_weights<NP>(lb, e, eh);
                p[0][i] = eh[0], p[0][i + 1] = eh[1];
                if constexpr (NP == 2) {
                    const h2 el = __builtin_convertvector(f2{e[0] - (float)eh[0], e[1] - (float)eh[1]}, h2);
                    p[NP - 1][i] = el[0], p[NP - 1][i + 1] = el[1];
                }
            }
            join_block(m, l, mb, sum_over_halves(lb), &keep, &add);
#pragma unroll
            for (int y = 0; y < MT; ++y) {
                const h8 va = *reinterpret_cast<const h8 *>(sv + q * 16 * DP + h * 8 * DP + (32 * y + r) * 8);
                f16v x;
#pragma unroll
                for (int i = 0; i < 16; ++i) x[i] = 0.0f;
#pragma unroll
                for (int z = 0; z < NP; ++z) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(va, p[z], x, 0, 0, 0);
                o[y] = o[y] * keep + x * add * s;
            }
        }
    };

    // around a step: its scales and the next one's loads, and what they brought
    auto before = [&](int32_t k) __attribute__((always_inline)) {
#pragma unroll
        for (int q = 0; q < 4; ++q) ks[q] = ks_next[q], vs[q] = vs_next[q];
        whole = whole_next;
        if ((k & 15) == 15) blk = next;
        if (k + 1 < part.steps) fetch(k + 1);
        if ((k & 15) == 0) next_page = find_page(a, b, token_of(k + 16), part.end);
        if ((k & 15) == 4) next = block_of(a, head, token_of(k + 12), next_page);
    };
    auto after = [&](int32_t k) __attribute__((always_inline)) {
        if (k + 1 < part.steps) deposit(k + 1, (k + 1) & 1);
        __syncthreads();
    };
    if (threadIdx.x == 0) has_nan = 0;
    __syncthreads();
    if (part.steps > 0) deposit(0, 0);
    __syncthreads();
    // steps that all rows see whole, in a loop of their own
    int32_t k = 0;
    bool apart = false;
    for (; k < part.steps; ++k) {
        for (; k < part.steps; ++k) {
            apart = scales.apart();
            if (__builtin_expect(apart, 0)) break;
            if (scales.top != vref) {
                const int e = (int)(vref >> 23) - (int)(scales.top >> 23) + 127;  // vref 0: sums of 0
                scale_o(bits_f32((uint32_t)(e < 0 ? 0 : e) << 23));
                vref = scales.top;
            }
            before(k);
            if (__builtin_expect(!whole, 0)) break;
            step(part.start + (k << 6), k & 1, std::false_type{});
            after(k);
        }
        if (k >= part.steps || apart) break;
        const int32_t tok = part.start + (k << 6);
        if (tok < w_hi && tok + 64 > w_lo) step(tok, k & 1, std::true_type{});
        after(k);
    }
    l = sum_over_halves(l);
    if (__builtin_expect(apart, 0)) {
        scale_o(l == 0.0f ? 0.0f : 1.0f / (1 << kVBits) / l);
        scale_o(bits_f32(vref));
        for (; k < part.steps; ++k) {
            before(k);
            const int32_t tok = part.start + (k << 6);
            if (tok < w_hi && tok + 64 > w_lo) step_apart(tok, k & 1);
            after(k);
        }
    }

    if (__builtin_expect(has_nan, 0)) {
        // V's NaN codes reach the rows that see their token, and no others: a
        // product of "is NaN" and "is seen", over the steps that took them for
        // zeros
        f16v hit[MT];
#pragma unroll
        for (int y = 0; y < MT; ++y)
#pragma unroll
            for (int i = 0; i < 16; ++i) hit[y][i] = 0.0f;
#pragma unroll 1
        for (int32_t tok = part.start; tok < part.end; tok += 16) {
            const Block w = block_of(a, head, tok, find_page(a, b, tok, part.end));
            if (!w.vs) continue;
            const uint8_t *p = a.v + (w.lo | (uint64_t)w.hi << 32) * (uint64_t)(16 * D) + h * 4 * D;
            const uint32_t from = tok + 4 * h - lo, span = hi - lo;
            h8 on;
#pragma unroll
            for (int e = 0; e < 8; ++e) on[e] = from + 8 * (e >> 2) + (e & 3) < span ? (_Float16)1.0f : (_Float16)0.0f;
#pragma unroll
            for (int y = 0; y < MT; ++y) {
                const int place = 32 * y + r, d = 4 * (place % (DP / 4)) + place / (DP / 4);
                const bool in = EXACT || d < D;
                const uint32_t n0 = in ? nan_bits(*reinterpret_cast<const uint32_t *>(p + 4 * d)) : 0;
                const uint32_t n1 = in ? nan_bits(*reinterpret_cast<const uint32_t *>(p + 4 * d + 8 * D)) : 0;
                h8 is;
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    is[e] = ((e < 4 ? n0 : n1) >> (8 * (e & 3) + 7)) & 1 ? (_Float16)1.0f : (_Float16)0.0f;
                hit[y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(is, on, hit[y], 0, 0, 0);
            }
        }
#pragma unroll
        for (int y = 0; y < MT; ++y)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[y][i] = hit[y][i] > 0.0f ? __builtin_nanf("") : o[y][i];
    }
    if (!live) return;
    // (the scale last: with the other factor it could leave fp32's range)
    const float f = apart ? 1.0f : 1.0f / (1 << kVBits) / l, scale = apart ? 1.0f : bits_f32(vref);
    // four columns 4 u .. 4 u + 3: places u, DP / 4 + u, ..
    auto results = [&](auto put) {
#pragma unroll
        for (int x = 0; x < (DP + 127) / 128; ++x)
#pragma unroll
            for (int i = 0; i < (DP < 128 ? DP / 8 : 16); ++i) {
                const int d = column(x, i);  // e = 0
                f4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = (e * (DP / 4) + 32 * x) / 32, up = (e * (DP / 4) + 32 * x) % 32;  // DP 64: half a tile on
                    v[e] = l == 0.0f ? 0.0f : o[t][i + up / 2] * f * scale;
                }
                if (EXACT || d < D) put(d, v);
            }
    };
    if (sp.splits > 1) {
        float *po = sp.o + (out_row * sp.splits + split) * D;
        if (h == 0) sp.lse[out_row * sp.splits + split] = l == 0.0f ? -kInf : m + __builtin_amdgcn_logf(l);
        results([&](int d, f4 v) { *reinterpret_cast<f4 *>(po + d) = v; });
    } else {
        const int64_t oo = ((int64_t)s.row0 + qi) * a.o_token + (int64_t)qh * a.o_head;
        results([&](int d, f4 v) { store_o4<NP == 1>(a.o, oo + d, v); });
    }
}

constexpr int kMostSplits = 128, kRowsSplits = 16;

// Joins few parts of many rows: D / 4 threads a row, as many rows a workgroup
// as fit, and no barriers; every thread weighs all of its row's parts.
template <bool BF16>
__global__ __launch_bounds__(256) void k_attention_join_rows(AttentionArgs a, Split sp, uint32_t total) {
    const int32_t D = a.t.dim, q4 = D >> 2, per = 256 / q4;
    const int32_t grp = threadIdx.x / q4, d = (threadIdx.x - grp * q4) * 4;
    const uint32_t id = blockIdx.x * (uint32_t)per + grp;
    if (grp >= per || id >= total) return;
    const uint32_t per_seq = (uint32_t)(a.max_q * a.q_heads);
    const int32_t b = id / per_seq, at = id - b * per_seq, i = at / a.q_heads, h = at - i * a.q_heads;
    const SeqRows s = seq_rows(a.t, b);
    if (i >= s.n) return;
    const int64_t row = ((int64_t)s.row0 + i) * a.q_heads + h;
    const float *lse = sp.lse + row * sp.splits, *po = sp.o + row * sp.splits * D + d;
    float x[kRowsSplits], w[kRowsSplits], top = -kInf, sum = 0.0f;
#pragma unroll
    for (int k = 0; k < kRowsSplits; ++k) x[k] = lse[k < sp.splits ? k : 0];
#pragma unroll
    for (int k = 0; k < kRowsSplits; ++k) top = fmaxf(top, x[k]);
#pragma unroll
    for (int k = 0; k < kRowsSplits; ++k) {
        w[k] = k >= sp.splits || x[k] == -kInf ? 0.0f : x[k] == top ? 1.0f : __builtin_amdgcn_exp2f(x[k] - top);
        sum += w[k];
    }
    // weights divided by their sum: the parts' own could leave fp32's range
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    f4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k0 = 0; k0 < kRowsSplits; k0 += 4) {
        if (k0 >= sp.splits) break;
        f4 p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)  // a part of weight 0 wrote nothing
            p[u] = k0 + u < sp.splits && x[k0 + u] != -kInf ? *reinterpret_cast<const f4 *>(po + (int64_t)(k0 + u) * D)
                                                            : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 4; ++u) v += p[u] * (w[k0 + u] * inv);
    }
    store_o4<BF16>(a.o, ((int64_t)s.row0 + i) * a.o_token + (int64_t)h * a.o_head + d, v);
}

// Joins a row's parts, a workgroup a row: the weights first, then the parts by
// as many groups of D / 4 threads as there are, four loads each under way.

template <bool BF16>
__global__ __launch_bounds__(256) void k_attention_join(AttentionArgs a, Split sp) {
    __shared__ float weight[kMostSplits];
    __shared__ f4 buf[256];
    const int32_t D = a.t.dim, q4 = D >> 2, lane = threadIdx.x & 63;
    const int64_t per = a.max_q * a.q_heads;
    const int32_t b = (int32_t)(blockIdx.x / per), i = (int32_t)(blockIdx.x % per / a.q_heads), h = (int32_t)(blockIdx.x % a.q_heads);
    const SeqRows s = seq_rows(a.t, b);
    if (i >= s.n) return;
    const int64_t row = ((int64_t)s.row0 + i) * a.q_heads + h;
    const float *lse = sp.lse + row * sp.splits, *po = sp.o + row * sp.splits * D;
    const float x0 = lane < sp.splits ? lse[lane] : -kInf, x1 = lane + 64 < sp.splits ? lse[lane + 64] : -kInf;
    float top = fmaxf(x0, x1);
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor(top, m));
    // a part of weight 0 wrote nothing
    const float w0 = x0 == -kInf ? 0.0f : x0 == top ? 1.0f : __builtin_amdgcn_exp2f(x0 - top);
    const float w1 = x1 == -kInf ? 0.0f : x1 == top ? 1.0f : __builtin_amdgcn_exp2f(x1 - top);
    float sum = w0 + w1;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m);
    // weights divided by their sum: the parts' own could leave fp32's range
    const float inv = 1.0f / sum;
    if (threadIdx.x < 64) weight[lane] = x0 == -kInf ? -1.0f : w0 * inv, weight[lane + 64] = x1 == -kInf ? -1.0f : w1 * inv;
    __syncthreads();
    const int32_t groups = 256 / q4, grp = threadIdx.x / q4, d = threadIdx.x % q4 * 4;
    f4 v{0.f, 0.f, 0.f, 0.f};
    if (grp < groups)
        for (int32_t k0 = grp; k0 < sp.splits; k0 += 4 * groups) {
            f4 p[4];
            float w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int32_t k = k0 + u * groups;
                w[u] = k < sp.splits ? weight[k] : -1.0f;
                p[u] = w[u] >= 0.0f || w[u] != w[u] ? *reinterpret_cast<const f4 *>(po + (int64_t)k * D + d) : f4{0.f, 0.f, 0.f, 0.f};
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) v += p[u] * (w[u] == -1.0f ? 0.0f : w[u]);
        }
    buf[threadIdx.x] = v;
    __syncthreads();
    if (grp > 0) return;
    for (int32_t g = 1; g < groups; ++g) v += buf[g * q4 + threadIdx.x];
    store_o4<BF16>(a.o, ((int64_t)s.row0 + i) * a.o_token + (int64_t)h * a.o_head + d, v);
}

// ------------------------------------------------------------------- plan --

constexpr int kFewWaves = 4;

struct Plan {
    bool few;
    int64_t groups;  // workgroups
    Split sp;
};

int width_of(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }  // columns that the kernels are built for

// one kernel's division of rows of `pairs` (sequence, KV head), that see `span`
// tokens at most
Plan divide(bool few, int64_t pairs, int64_t rows, int64_t span) {
    Plan p{};
    p.few = few;
    const int64_t tile = few ? 16 : kManyRows;
    p.sp.tiles = (int32_t)((rows + tile - 1) / tile);
    const int64_t groups = pairs * p.sp.tiles, steps = (span + 63) / 64;
    // Few rows: 512 workgroups of a step for each wavefront at least, and up to
    // 2048 of four steps, so that ragged lengths even out (4096: 1 x 32000 28 us
    // against 20).  Many rows: parts of 15 steps up to two workgroups a CU, of
    // eight up to one, as joining them reads and writes every result again in
    // fp32 (3 x 383 x 5292 in three parts 102 us, in two 135; 1 x 400 x 4000 in
    // four 61, in two 73; 1 x 1500 x 1500, 24 steps, in two 66, in one 52).
    int64_t splits;
    if (few) {
        const int64_t fine = (steps + 4 * kFewWaves - 1) / (4 * kFewWaves), coarse = (steps + kFewWaves - 1) / kFewWaves;
        splits = (2048 + groups - 1) / groups;
        splits = splits < fine ? splits : fine;
        const int64_t least = (512 + groups - 1) / groups;
        splits = splits > least ? splits : least < coarse ? least : coarse;
        // joining costs a launch: not for two steps of a wavefront, nor four on a full GPU
        if (steps <= 2 * kFewWaves || (groups >= 256 && steps <= 4 * kFewWaves)) splits = 1;
    } else {
        const int64_t two = (512 + groups / 2) / groups, one = 256 / groups, coarse = steps / 15, fine = steps / 8;
        splits = two < coarse ? two : coarse;
        const int64_t least = one < fine ? one : fine;
        splits = splits > least ? splits : least;
    }
    if (splits > kMostSplits) splits = kMostSplits;
    if (splits < 1) splits = 1;
    p.sp.chunk = (int32_t)(((steps + splits - 1) / splits) * 64);
    p.sp.splits = (int32_t)splits;
    p.groups = groups * splits;
    return p;
}

// Up to 64 rows the kernel for few rows is the faster one (64 rows: 8 sequences
// of 4000 tokens 43.2 us against 44.6, 32 of 1000 36.2 against 39.0, one of 4000
// 16 against 25).  Above, the sum of what either takes decides, in us by
// measurement: a start, a step of 64 tokens, as many workgroups as run at once, a
// join.  Of 91 cases of 1 to 32 sequences, 16 to 4000 queries and all widths,
// bf16 but for nine, it takes one that is more than 5% slower in three (10.5 us
// for 8.5, 44 for 37, 65 for 53).  Some: 1 x 256 9.2 us in the kernel for few
// rows, 14 in the one for many; 1 x 512 19 and 21; 1 x 700 28 and 27; 8 x 128 30
// and 14; 32 after 4000 18 and 29; 4 x 100 after 900 31 and 36; one KV head of
// 256, 512 queries of 8 heads, 15 and 37.  Types do not enter: fp32's two pieces
// cost both kernels twice the products (2 x 200 19.1 and 18.6, 4 x 333 over 4000
// 59 and 56).
// max_kv decides, not the window: the workspace then covers any window.
Plan make_plan(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_q, int64_t max_kv,
               int64_t window) {
    const int64_t rows = max_q * (q_heads / kv_heads), pairs = seqs * kv_heads;
    bool few = rows <= 64;
    if (!few) {
        const Plan f = divide(true, pairs, rows, max_kv), m = divide(false, pairs, rows, max_kv);
        const int width = width_of(dim);
        const double at_once = 65536.0 / width, step = width == 64 ? 1.1 : width == 128 ? 1.65 : 3.3;
        const double rf = f.groups / at_once, rm = m.groups / 512.0;
        const int64_t sf = (f.sp.chunk / 64 + kFewWaves - 1) / kFewWaves, sm = m.sp.chunk / 64;
        few = 3.0 + (rf > 1.0 ? rf : 1.0) * (3.5 + 2.5 * sf) + (f.sp.splits > 1 ? 4.0 : 0.0) <
              8.0 + (rm > 1.0 ? rm : 1.0) * step * sm + (m.sp.splits > 1 ? 6.0 : 0.0);
    }
    int64_t span = max_kv;  // tokens that a row tile can see
    if (window > 0 && window < span && window + max_q + 64 < span) span = window + max_q + 64;
    return divide(few, pairs, rows, span);
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

// NQ = 1: q is bf16; NP = 1: o is
template <int NQ, int NP>
hipError_t launch_t(const AttentionArgs &a, const Plan &p, hipStream_t s) {
    const unsigned grid = (unsigned)p.groups;
    const int width = width_of(a.t.dim);
    if (p.few)
        width == 64    ? start_few<1, NQ, NP>(a, p.sp, grid, s)
        : width == 128 ? start_few<2, NQ, NP>(a, p.sp, grid, s)
                       : start_few<4, NQ, NP>(a, p.sp, grid, s);
    else
        width == 64    ? start_many<64, NQ, NP>(a, p.sp, grid, s)
        : width == 128 ? start_many<128, NQ, NP>(a, p.sp, grid, s)
                       : start_many<256, NQ, NP>(a, p.sp, grid, s);
    const hipError_t err = hipGetLastError();
    if (err != hipSuccess || p.sp.splits == 1) return err;
    const unsigned rows = (unsigned)((int64_t)a.t.seqs * a.max_q * a.q_heads);
    const unsigned per = 1024u / a.t.dim;
    // from 512 rows on many rows a workgroup (8 x 16 x 32 rows of 4 parts 40.5 us
    // with attention, a workgroup a row 44; 16384 rows of 2 parts 22 and 43; 128
    // rows of 16 parts 15.7 and 15.0, before the parts' weights were divided)
    if (rows >= 512 && p.sp.splits <= kRowsSplits) {
        hipLaunchKernelGGL((k_attention_join_rows<NP == 1>), dim3((rows + per - 1) / per), dim3(256), 0, s, a, p.sp, rows);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((k_attention_join<NP == 1>), dim3(rows), dim3(256), 0, s, a, p.sp);
    return hipGetLastError();
}

}  // namespace

int64_t attention_workspace(int64_t tokens, int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim,
                            int64_t max_q, int64_t max_kv) {
    const Plan p = make_plan(seqs, q_heads, kv_heads, dim, max_q, max_kv, 0);  // a window only takes parts away
    return p.sp.splits > 1 ? tokens * q_heads * p.sp.splits * (dim + 1) * 4 : 0;
}

int64_t attention_groups(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_q, int64_t max_kv) {
    return make_plan(seqs, q_heads, kv_heads, dim, max_q, max_kv, 0).groups;
}

hipError_t launch_attention(const AttentionArgs &a, void *work, hipStream_t s, const char **kernel) {
    Plan p = make_plan(a.t.seqs, a.q_heads, a.t.heads, a.t.dim, a.max_q, a.max_kv, a.window);
    p.sp.group = a.q_heads / a.t.heads;
    p.sp.by_splits = Divider::of(p.sp.splits), p.sp.by_tiles = Divider::of(p.sp.tiles);
    p.sp.by_heads = Divider::of(a.t.heads), p.sp.by_group = Divider::of(p.sp.group);
    p.sp.by_per = Divider::of((int64_t)p.sp.tiles * p.sp.splits);
    p.sp.o = static_cast<float *>(work);
    p.sp.lse = p.sp.o + (int64_t)a.t.tokens * a.q_heads * p.sp.splits * a.t.dim;
    const bool join = p.sp.splits > 1;
    *kernel = p.few ? (join ? "attention_few, attention_join" : "attention_few")
                    : (join ? "attention_many, attention_join" : "attention_many");
    if (a.q_bf16) return a.o_bf16 ? launch_t<1, 1>(a, p, s) : launch_t<1, 2>(a, p, s);
    return a.o_bf16 ? launch_t<2, 1>(a, p, s) : launch_t<2, 2>(a, p, s);
}

}  // namespace lcml
