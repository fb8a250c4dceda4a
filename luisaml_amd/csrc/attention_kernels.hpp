// attention_kernels.hpp -- attention over the E4M3 KV cache (gfx950): the
// kernels and their plans, for attention.hip, attention_sinks.hip and
// attention_shared.hip, which build them for their calls.
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
#pragma once

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
    int32_t parts, first;  // kPrefix, kOwn: a row's parts of both, and where this one's begin
};

// Which tokens a call reads of a sequence:
//   kPlain   one range, as causality and the window bound it
//   kSinks   also the first `sinks` positions, wherever the window has gone.
//            Steps run over an axis that leaves out whole steps between the two.
//   kPrefix  for all rows of a group of sequences, the tokens that these share
//   kOwn     the tokens from there on, or all where a sequence's rows do not
//            lie behind what it shares
// The last two leave parts in the workspace, which one join puts together.
enum Form { kPlain, kSinks, kPrefix, kOwn };
template <Form F>
constexpr bool kShares = F == kPrefix || F == kOwn;

template <Form F>
__device__ inline bool in_parts(const Split &sp) {
    return kShares<F> || sp.splits > 1;
}
// a row's part in the workspace
template <Form F>
__device__ inline int64_t part_at(const Split &sp, int64_t row, int32_t split) {
    return kShares<F> ? row * sp.parts + sp.first + split : row * sp.splits + split;
}

// the rows of group g, and the tokens that it shares; n 0: none
__device__ inline SeqRows group_rows(const AttentionArgs &a, int32_t g) {
    SeqRows s{0, 0, 0, 0};
    if (g >= a.groups) return s;
    int32_t b0 = a.group_seq[g], b1 = a.group_seq[g + 1];
    const int32_t len = a.prefix_len[g];
    // (cut to what there is: a sequence out of range must not take the others'
    // parts with it)
    b0 = b0 > 0 ? b0 : 0, b1 = b1 < a.t.seqs ? b1 : a.t.seqs;
    if (b1 <= b0 || len <= 0) return s;
    int32_t row0 = a.t.cu[b0], end = a.t.cu[b1];
    row0 = row0 > 0 ? row0 : 0, end = end < a.t.tokens ? end : a.t.tokens;
    return end > row0 ? SeqRows{row0, end - row0, len, len} : s;
}

// the tokens that sequence b reads with its group; 0: none, also where its rows
// do not all lie behind them (b the same in all lanes, and all lanes active)
__device__ inline int32_t shared_tokens(const AttentionArgs &a, int32_t b, const SeqRows &s) {
    const int32_t lane = threadIdx.x & 63;
    int32_t len = 0;
    for (int32_t g0 = 0; g0 < a.groups; g0 += 64) {
        const int32_t g = g0 + lane;
        const bool in = g < a.groups;
        const int32_t end = in ? a.group_seq[g + 1] : 0x7fffffff, own = in && b >= a.group_seq[g] ? a.prefix_len[g] : 0;
        const uint64_t over = __builtin_amdgcn_ballot_w64(end > b);  // b's group, and those after it
        if (!over) continue;
        len = __builtin_amdgcn_readlane(own, __builtin_ctzll(over));
        break;
    }
    return len > 0 && s.pos0 >= len ? len : 0;
}

// the same, for a sequence of a lane's own
__device__ inline int32_t shared_tokens_of_lane(const AttentionArgs &a, int32_t b, const SeqRows &s) {
    int32_t lo = 0, hi = a.groups;  // the first group that ends behind b
    while (lo < hi) {
        const int32_t m = (lo + hi) >> 1;
        if (a.group_seq[m + 1] > b)
            hi = m;
        else
            lo = m + 1;
    }
    const int32_t len = lo < a.groups && b >= a.group_seq[lo] ? a.prefix_len[lo] : 0;
    return len > 0 && s.pos0 >= len ? len : 0;
}

// A workgroup's rows: of which sequence (kPrefix: group), which tile of them,
// and the first position that they may see.
struct Work {
    SeqRows s;
    int32_t b, tile, from;
};
// tile `id` of sequence b; kPrefix: among the tiles that the groups have, one
// group's after the other's
template <Form F, int ROWS>
__device__ inline Work work_of(const AttentionArgs &a, const Split &sp, int32_t b, uint32_t id) {
    if constexpr (F == kPrefix) {
        const int32_t lane = threadIdx.x & 63;
        uint32_t before = 0;
        for (int32_t g0 = 0; g0 < a.groups; g0 += 64) {
            const SeqRows s = group_rows(a, g0 + lane);
            const uint32_t tiles = ((uint32_t)s.n * sp.group + ROWS - 1) / ROWS;
            uint32_t sum = tiles;  // of the lanes up to this one
#pragma unroll
            for (int m = 1; m < 64; m <<= 1) {
                const uint32_t v = __shfl_up(sum, m);
                sum += lane >= m ? v : 0;
            }
            const uint64_t over = __builtin_amdgcn_ballot_w64(before + sum > id);
            if (over) {
                const int at = __builtin_ctzll(over);
                const auto of = [&](int32_t v) { return __builtin_amdgcn_readlane(v, at); };
                const uint32_t tile = id - before - of((int32_t)(sum - tiles));
                if (tile >= (uint32_t)of((int32_t)tiles)) break;  // groups that overlap
                return Work{SeqRows{of(s.row0), of(s.n), of(s.pos0), of(s.len)}, g0 + at, (int32_t)tile, 0};
            }
            before += __builtin_amdgcn_readlane((int32_t)sum, 63);
        }
        return Work{SeqRows{0, 0, 0, 0}, 0, 0, 0};
    } else {
        const SeqRows s = seq_rows(a.t, b);
        return Work{s, b, (int32_t)id, F == kOwn ? shared_tokens(a, b, s) : 0};
    }
}

// positions that query i of a sequence sees: lo .. hi-1, neither falling with
// i; kSinks: and 0 .. sinks-1 below hi; kOwn: from `from` on
template <Form F>
__device__ inline void sees(const AttentionArgs &a, const SeqRows &s, int32_t from, int32_t i, int32_t *lo, int32_t *hi) {
    const int32_t pos = s.pos0 + i, w = (int32_t)a.window;  // below 2^31; 0: no window
    const int32_t h = a.causal && pos < s.len ? pos + 1 : s.len;
    int32_t l = w > 0 && pos >= w ? pos - w + 1 : 0;
    if (F == kOwn) l = l > from ? l : from;
    *hi = h > 0 ? h : 0;
    *lo = l < *hi ? l : *hi;
}
// whether position j is seen by a row of lo, hi
template <Form F>
__device__ inline bool seen(const AttentionArgs &a, int32_t j, int32_t lo, int32_t hi) {
    return j < hi && (j >= lo || (F == kSinks && j < a.sinks));
}

// the part of positions lo .. hi-1 that is this workgroup's, from a multiple of
// 64 on, in steps of 64; kSinks: start lies on the axis that leaves out `gap`
// positions (whole steps) after the first `edge` ones, which hold the sinks
struct Part {
    int32_t start, end, steps, edge, gap;
};
template <Form F>
__device__ inline Part part_of(const AttentionArgs &a, const Split &sp, int32_t split, int32_t lo, int32_t hi) {
    int32_t edge = 0, gap = 0;
    if (F == kSinks) {
        const int64_t up = ((int64_t)(a.sinks < hi ? a.sinks : hi) + 63) & ~63;
        edge = (int32_t)(up < 0x7fffffc0 ? up : 0x7fffffc0), gap = (lo & ~63) > edge ? (lo & ~63) - edge : 0;
        lo = 0, hi -= gap;
    }
    const int64_t from = (lo & ~63) + (int64_t)split * sp.chunk;
    int64_t to = split + 1 < sp.splits ? from + sp.chunk : hi;
    to = to < hi ? to : hi;
    if (from >= to || a.t.pages == 0) return Part{0, 0, 0, 0, 0};
    return Part{(int32_t)from, (int32_t)(F == kSinks && to > edge ? to + gap : to), (int32_t)((to - from + 63) >> 6), edge, gap};
}
// the first token of the part's step k
template <Form F>
__device__ inline int32_t step_token(const Part &p, int32_t k) {
    const int32_t at = p.start + (k << 6);
    return F == kSinks && at >= p.edge ? at + p.gap : at;
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
template <int DC, int NW>
struct FewLds {
    float red_m[NW][16], red_l[NW][16];
    __attribute__((aligned(16))) float buf[NW][16][DC * 64 + 4];
};
template <int DC, int NQ, int NP, int NW, Form F>
__device__ __attribute__((always_inline)) inline void few_rows(const AttentionArgs &a, const Split &sp, uint32_t id0,
                                                               FewLds<DC, NW> &lds) {
    auto &red_m = lds.red_m, &red_l = lds.red_l;
    auto &buf = lds.buf;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t D = a.t.dim, G = sp.group;
    const uint32_t id1 = sp.by_heads.div(id0), id2 = sp.by_splits.div(id1);
    const int32_t head = id0 - id1 * a.t.heads, split = id1 - id2 * sp.splits;
    const int32_t seq = F == kPrefix ? 0 : sp.by_tiles.div(id2);
    const Work work = work_of<F, 16>(a, sp, seq, id2 - seq * sp.tiles);
    const SeqRows s = work.s;
    const int32_t b = work.b;
    const int32_t rows = (s.n < (int32_t)a.max_q ? s.n : (int32_t)a.max_q) * G;
    const int32_t row0 = work.tile * 16;
    if (row0 >= rows) return;
    const int32_t last = rows - row0 < 16 ? rows - 1 : row0 + 15;  // of the tile
    const int32_t row = row0 + r < last ? row0 + r : last;         // this lane's
    const int32_t qi = sp.by_group.div(row), qh = head * G + row - qi * G;
    int32_t lo, hi, lo_min, hi_min, lo_max, hi_max;
    sees<F>(a, s, work.from, qi, &lo, &hi);
    sees<F>(a, s, work.from, sp.by_group.div(row0), &lo_min, &hi_min);
    sees<F>(a, s, work.from, sp.by_group.div(last), &lo_max, &hi_max);
    const Part part = part_of<F>(a, sp, split, lo_min, hi_max);
    const int64_t out_row = ((int64_t)s.row0 + qi) * a.q_heads + qh;
    if (part.steps == 0 && in_parts<F>(sp)) {
        if (threadIdx.x < 16 && row0 + r <= last) sp.lse[part_at<F>(sp, out_row, split)] = -kInf;
        return;
    }
    const int32_t mine = (part.steps - wave + NW - 1) / NW;

    Block blk;
    auto find = [&](int32_t k) {  // lane i: block i of the wavefront's next 16 steps
        const int32_t tok = step_token<F>(part, (k + (lane >> 2)) * NW + wave) + (lane & 3) * 16;
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
    // kSinks: positions below these are seen by the lane's row, by any row, by all
    const uint32_t sinks = a.sinks < hi ? a.sinks : hi, sinks_max = a.sinks < hi_max ? a.sinks : hi_max,
                   sinks_min = a.sinks < hi_min ? a.sinks : hi_min;
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
            const uint32_t span = vs[sb] ? hi - lo : 0, first = F == kSinks && vs[sb] ? sinks : 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool in = from + 16 * sb + i < span || (F == kSinks && (uint32_t)(tok + 4 * g + 16 * sb + i) < first);
                t[sb][i] = in ? t[sb][i] : -kInf;
            }
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
                const uint32_t span = vs[sb] ? hi_max - lo_min : 0, first = F == kSinks && vs[sb] ? sinks_max : 0;
                uint32_t seen = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = all + 16 * sb + i < span || (F == kSinks && (uint32_t)(tok + 4 * g + 16 * sb + i) < first);
                    seen |= in ? 0x80u << (8 * i) : 0u;
                }
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
            tok = step_token<F>(part, k * NW + wave);
            scales_of(k);
            const bool all = (tok >= lo_max && tok + 64 <= hi_min) || (F == kSinks && (uint32_t)tok + 64 <= sinks_min);
            if (!(all && vs[0] && vs[1] && vs[2] && vs[3]) || scales.apart()) break;
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
            step_apart(k, step_token<F>(part, k * NW + wave));
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
            const int32_t tok = step_token<F>(part, k * NW + wave);
            for (int32_t j = F == kSinks || tok > lo_min ? tok : lo_min; j < tok + 64 && j < part.end; ++j) {
                const Block w = block_of(a, head, j, find_page(a, b, j, part.end));
                if (!w.vs) continue;
                const uint8_t *p = a.v + (w.lo | (uint64_t)w.hi << 32) * (uint64_t)(16 * D);
                for (int32_t d = lane; d < D; d += 64)
                    if ((p[v_place(j & 15, d, D)] & 0x7f) == 0x7f)
                        for (int rr = 0; rr < 16; ++rr)
                            if (seen<F>(a, j, (int32_t)lane_of(lo, rr), (int32_t)lane_of(hi, rr))) buf[wave][rr][d] = __builtin_nanf("");
            }
        }
    if (in_parts<F>(sp) && wave == 0 && g == 0 && row0 + r <= last)
        sp.lse[part_at<F>(sp, out_row, split)] = sum == 0.0f ? -kInf : top + __builtin_amdgcn_logf(sum);
    __syncthreads();
    const int32_t q4 = D >> 2;
    for (int32_t e = threadIdx.x; e < (last - row0 + 1) * q4; e += NW * 64) {
        const int32_t rr = e / q4, d = e % q4 * 4, i = (row0 + rr) / G, h = head * G + (row0 + rr) % G;
        f4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < NW; ++w) v += *reinterpret_cast<const f4 *>(&buf[w][rr][d]);
        if (in_parts<F>(sp))
            *reinterpret_cast<f4 *>(sp.o + part_at<F>(sp, ((int64_t)s.row0 + i) * a.q_heads + h, split) * D + d) = v;
        else
            store_o4<NP == 1>(a.o, ((int64_t)s.row0 + i) * a.o_token + (int64_t)h * a.o_head + d, v);
    }
}

template <int DC, int NQ, int NP, int NW, Form F>
__global__ __launch_bounds__(NW * 64, DC <= 2 ? 2 : 1) void k_attention_few(AttentionArgs a, Split sp) {
    __shared__ FewLds<DC, NW> lds;
    few_rows<DC, NQ, NP, NW, F>(a, sp, blockIdx.x, lds);
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
// A prompt of 8192 tokens, 32 heads over 8 of 128, 0.55 TFLOP: 588 to 605 us,
// 920 TFLOP/s, where a library's product of 8192^3 in bf16 reaches 1190 to 1625 by
// the order of its operands.  A step's 32 matrix instructions take 1024 cycles of
// a SIMD, its 320 vector ones 1280, and two wavefronts a SIMD overlap them to two
// thirds of the sum.  (Two groups of wavefronts half a step apart: 1075 us, for the
// registers spilled.)  D > 128 has one wavefront a SIMD, and nothing to overlap LDS
// reads with: 220 TFLOP/s on a prompt of 2048 tokens, 260 on one of 4000, 510 on one
// of 8192 through a window of 2048 (heads of 256).  What happens around a step is
// in three loops, always inlined: out of line, its registers lie in scratch.
constexpr int kManyWaves = 4, kManyRows = 32 * kManyWaves;

// LDS holds DP columns: past D, zeros for K and anything for V, whose columns
// there are not stored.  K: [4 blocks][DP / 16][16 tokens][16].  V: [4
// blocks][2][DP][8 tokens], in the halves the groups 0 and 2, 1 and 3 of four
// tokens, and column 4 u + e in place e * DP / 4 + u: what the lanes write and
// what they read is contiguous.
template <int DP>
struct ManyLds {
    __attribute__((aligned(16))) uint8_t k[2][64 * DP];
    __attribute__((aligned(16))) _Float16 v[2][64 * DP];
    uint32_t has_nan;  // V, in steps that some row does not see whole
};
template <int DP, bool EXACT, int NQ, int NP, Form F>
__device__ __attribute__((always_inline)) inline void many_rows(const AttentionArgs &a, const Split &sp, uint32_t id0,
                                                                ManyLds<DP> &lds) {
    constexpr int KJ = DP / 32;  // pairs of 16-element pieces of K
    constexpr int MT = DP / 32;  // tiles of 32 columns of V
    constexpr int PL = (DP + 63) / 64;  // 16-byte loads for a lane of a 16-token block
    auto &stage_k = lds.k;
    auto &stage_v = lds.v;
    uint32_t &has_nan = lds.has_nan;
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int32_t D = EXACT ? DP : a.t.dim, G = sp.group;
    // workgroups of one sequence and KV head on one XCD (id0 modulo 8),
    // whose L2 then holds their K and V; the longest rows first
    const uint32_t pairs = F == kPrefix ? a.t.heads : (uint32_t)a.t.seqs * a.t.heads, per = (uint32_t)sp.tiles * sp.splits;
    const bool by_xcd = pairs % 8 == 0;
    const uint32_t id = by_xcd ? id0 / 8 : id0, over = sp.by_per.div(id), rest = id - over * per;
    const uint32_t pair = by_xcd ? id0 % 8 + 8 * over : over;
    const int32_t place = sp.by_splits.div(rest), split = rest - place * sp.splits;
    const int32_t seq = F == kPrefix ? 0 : sp.by_heads.div(pair), head = pair - seq * a.t.heads;
    const Work work = work_of<F, kManyRows>(a, sp, seq, F == kPrefix ? place : sp.tiles - 1 - place);
    const SeqRows s = work.s;
    const int32_t b = work.b;
    const int32_t rows = (s.n < (int32_t)a.max_q ? s.n : (int32_t)a.max_q) * G, row0 = work.tile * kManyRows;
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
    sees<F>(a, s, work.from, qi, &lo, &hi);
    sees<F>(a, s, work.from, sp.by_group.div(row0), &lo_min, &hi_min);
    sees<F>(a, s, work.from, sp.by_group.div(last), &lo_max, &hi_max);
    sees<F>(a, s, work.from, sp.by_group.div(w0), &w_lo, &unused);
    sees<F>(a, s, work.from, sp.by_group.div(w1), &unused, &w_hi);
    const Part part = part_of<F>(a, sp, split, lo_min, hi_max);
    const int64_t out_row = ((int64_t)s.row0 + qi) * a.q_heads + qh;
    if (part.steps == 0 && in_parts<F>(sp)) {
        if (h == 0 && live) sp.lse[part_at<F>(sp, out_row, split)] = -kInf;
        return;
    }
    // kSinks: positions below these are seen by the lane's row, by any row of
    // the wavefront, by all rows
    const uint32_t sinks = a.sinks < hi ? a.sinks : hi, sinks_wave = a.sinks < w_hi ? a.sinks : w_hi,
                   sinks_min = a.sinks < hi_min ? a.sinks : hi_min;
    // whether any row of the wavefront sees one of the step's tokens
    auto touches = [&](int32_t tok) { return (tok < w_hi && tok + 64 > w_lo) || (F == kSinks && (uint32_t)tok < sinks_wave); };

    // lane i: block i of 16 steps; the next 16 steps' pages and blocks are
    // looked up while these are worked on
    Block blk, next;
    int32_t next_page = -1;
    auto token_of = [&](int32_t k) { return step_token<F>(part, k + (lane >> 2)) + (lane & 3) * 16; };
    uint32_t ks[4], vs[4], ks_next[4], vs_next[4];
    bool whole, whole_next = false;  // whether every row sees all of a step's tokens
    Scales scales;                   // of the steps fetched so far, the same for all wavefronts
    // this wavefront's block of step k
    u4 kr[PL], vr[PL];
    auto fetch = [&](int32_t k) __attribute__((always_inline)) {
        const int i = (k & 15) * 4;
        const uint64_t at = (lane_of(blk.lo, i + wave) | (uint64_t)lane_of(blk.hi, i + wave) << 32) * (uint64_t)(16 * D);
        const uint8_t *pk = a.k + at, *pv = a.v + at;
#pragma unroll
        for (int x = 0; x < PL; ++x) {
            const bool in = (EXACT && DP % 64 == 0) || 64 * x + lane < D;
            kr[x] = in ? *reinterpret_cast<const u4 *>(pk + (64 * x + lane) * 16) : u4{0, 0, 0, 0};
            vr[x] = in ? *reinterpret_cast<const u4 *>(pv + (64 * x + lane) * 16) : u4{0, 0, 0, 0};
        }
        // (the scales after them: they were asked for last)
#pragma unroll
        for (int q = 0; q < 4; ++q) ks_next[q] = lane_of(blk.ks, i + q), vs_next[q] = lane_of(blk.vs, i + q);
        const int32_t tok = step_token<F>(part, k);
        uint32_t least = vs_next[0] < vs_next[1] ? vs_next[0] : vs_next[1];
        least = vs_next[2] < least ? vs_next[2] : least;
        least = vs_next[3] < least ? vs_next[3] : least;
        whole_next = ((tok >= lo_max && tok + 64 <= hi_min) || (F == kSinks && (uint32_t)tok + 64 <= sinks_min)) && least;
        scales.take(vs_next);
    };
    uint32_t vref = 0;  // the largest V scale up to the step that is worked on
    auto deposit = [&](int32_t k, int buf) __attribute__((always_inline)) {
        const uint32_t mine = wave == 0 ? vs_next[0] : wave == 1 ? vs_next[1] : wave == 2 ? vs_next[2] : vs_next[3];
        const float ratio = scales.apart() ? 1.0f : v_ratio(mine, scales.top);
        if (__builtin_expect(!whole_next, 0)) {
            // what lies past the last token counts as zeros, and so do NaN codes
            // for now
            const int32_t left = part.end - (step_token<F>(part, k) + 16 * wave);
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
            if (DP % 64 == 0 || u < DP) *reinterpret_cast<u4 *>(&stage_k[buf][wave * 16 * DP + u * 16]) = kr[x];  // zeros past D
            if ((EXACT && DP % 64 == 0) || u < D)
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
                const uint32_t span = vs[q] ? hi - lo : 0, first = F == kSinks && vs[q] ? sinks : 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int at = (q & 1) * 8 + i, off = 16 * q + 8 * (i >> 2) + (i & 3);
                    const bool in = from + off < span || (F == kSinks && (uint32_t)(tok + 4 * h + off) < first);
                    t[q >> 1][at] = in ? t[q >> 1][at] : -kInf;
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
            step(step_token<F>(part, k), k & 1, std::false_type{});
            after(k);
        }
        if (k >= part.steps || apart) break;
        const int32_t tok = step_token<F>(part, k);
        if (touches(tok)) step(tok, k & 1, std::true_type{});
        after(k);
    }
    l = sum_over_halves(l);
    if (__builtin_expect(apart, 0)) {
        scale_o(l == 0.0f ? 0.0f : 1.0f / (1 << kVBits) / l);
        scale_o(bits_f32(vref));
        for (; k < part.steps; ++k) {
            before(k);
            const int32_t tok = step_token<F>(part, k);
            if (touches(tok)) step_apart(tok, k & 1);
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
        for (int32_t at = part.start; at < part.start + part.steps * 64; at += 16) {
            const int32_t tok = F == kSinks && at >= part.edge ? at + part.gap : at;
            if (tok >= part.end) break;
            const Block w = block_of(a, head, tok, find_page(a, b, tok, part.end));
            if (!w.vs) continue;
            const uint8_t *p = a.v + (w.lo | (uint64_t)w.hi << 32) * (uint64_t)(16 * D) + h * 4 * D;
            const uint32_t from = tok + 4 * h - lo, span = hi - lo;
            h8 on;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int off = 8 * (e >> 2) + (e & 3);
                const bool in = from + off < span || (F == kSinks && (uint32_t)(tok + 4 * h + off) < sinks);
                on[e] = in ? (_Float16)1.0f : (_Float16)0.0f;
            }
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
    // four columns 4 u .. 4 u + 3: places u, DP / 4 + u, .., eight places a group
    // of four rows of o
    auto results = [&](auto put) {
#pragma unroll
        for (int c = 0; c < DP / 32; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int d = 4 * (8 * c + 4 * h + i);
                f4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int at = e * (DP / 32) + c;
                    v[e] = l == 0.0f ? 0.0f : o[at / 4][at % 4 * 4 + i] * f * scale;
                }
                if (EXACT || d < D) put(d, v);
            }
    };
    if (in_parts<F>(sp)) {
        float *po = sp.o + part_at<F>(sp, out_row, split) * D;
        if (h == 0) sp.lse[part_at<F>(sp, out_row, split)] = l == 0.0f ? -kInf : m + __builtin_amdgcn_logf(l);
        results([&](int d, f4 v) { *reinterpret_cast<f4 *>(po + d) = v; });
    } else {
        const int64_t oo = ((int64_t)s.row0 + qi) * a.o_token + (int64_t)qh * a.o_head;
        results([&](int d, f4 v) { store_o4<NP == 1>(a.o, oo + d, v); });
    }
}

template <int DP, bool EXACT, int NQ, int NP, Form F>
__global__ __launch_bounds__(kManyWaves * 64, DP <= 128 ? 2 : 1) void k_attention_many(AttentionArgs a, Split sp) {
    __shared__ ManyLds<DP> lds;
    many_rows<DP, EXACT, NQ, NP, F>(a, sp, blockIdx.x, lds);
}

constexpr int kMostSplits = 128, kRowsSplits = 16;

// how many parts a row has, and how many of the first ones do not count: the
// prefix's, for rows that read it with their own tokens
template <Form F>
__device__ inline int32_t parts_of(const Split &sp) {
    return kShares<F> ? sp.parts : sp.splits;
}
template <Form F, bool PER_LANE>
__device__ inline int32_t skipped(const AttentionArgs &a, const Split &sp, int32_t b, const SeqRows &s) {
    if constexpr (kShares<F>) return (PER_LANE ? shared_tokens_of_lane(a, b, s) : shared_tokens(a, b, s)) > 0 ? 0 : sp.first;
    return 0;
}

// the first sequence that ends behind row t of the batch, or seqs (t the same
// in all lanes, and all lanes active): every lane looks at one of 64 places,
// between two of which a next round looks
__device__ inline int32_t sequence_of(const AttentionArgs &a, int32_t t) {
    int32_t lo = 0, hi = a.t.seqs;
    while (hi > lo) {
        const int32_t step = (hi - lo + 63) >> 6, up = lo + (int32_t)((threadIdx.x & 63) + 1) * step, at = up < hi ? up : hi;
        const uint64_t over = __builtin_amdgcn_ballot_w64(a.t.cu[at] > t);
        if (!over) return hi;
        const int32_t f = __builtin_ctzll(over), end = lo + (f + 1) * step;
        hi = (end < hi ? end : hi) - 1, lo += f * step;
    }
    return hi;
}
// the same for a row of a lane's own, at least `lo`
__device__ inline int32_t sequence_of_lane(const AttentionArgs &a, int32_t lo, int32_t t) {
    int32_t hi = a.t.seqs;
    while (lo < hi) {
        const int32_t m = (lo + hi) >> 1;
        if (a.t.cu[m + 1] > t)
            hi = m;
        else
            lo = m + 1;
    }
    return lo;
}

// Joins few parts of many rows: D / 4 threads a row, as many rows a workgroup
// as fit, and no barriers; every thread weighs all of its row's parts.  Rows
// are max_q of each sequence, or (kPrefix, kOwn, which always join) those of the
// batch, each of which looks for its sequence: beside one chunk of a prompt most
// others would be empty (63 single queries and 2000, 32 heads of 128, behind
// 2048: 505 us and 265 with attention; 8 x 100 behind 8192 177.5 and 179.5).
template <bool BF16, Form F>
__global__ __launch_bounds__(256) void k_attention_join_rows(AttentionArgs a, Split sp, uint32_t total) {
    const int32_t D = a.t.dim, q4 = D >> 2, per = 256 / q4;
    const int32_t grp = threadIdx.x / q4, d = (threadIdx.x - grp * q4) * 4;
    const uint32_t id0 = blockIdx.x * (uint32_t)per, id = id0 + grp;
    const int32_t parts = parts_of<F>(sp);
    float x[kRowsSplits];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int k = 0; k < kRowsSplits; ++k) x[k] = sp.lse[row * parts + (k < parts ? k : 0)];
    };
    int32_t b = 0, i, h;
    if constexpr (kShares<F>) {
        load(id < total ? id : id0);  // under way while the sequence is looked for
        b = sequence_of(a, id0 / a.q_heads);
    }
    if (grp >= per || id >= total) return;
    if constexpr (kShares<F>) {
        i = id / a.q_heads, h = id - i * a.q_heads;
        if (b < a.t.seqs && a.t.cu[b + 1] <= i) b = sequence_of_lane(a, b + 1, i);
        if (b >= a.t.seqs) return;
    } else {
        const uint32_t per_seq = (uint32_t)(a.max_q * a.q_heads);
        b = id / per_seq;
        const int32_t at = id - b * per_seq;
        i = at / a.q_heads, h = at - i * a.q_heads;
    }
    const SeqRows s = seq_rows(a.t, b);
    if constexpr (kShares<F>) {
        i -= s.row0;
        if (i < 0 || i >= a.max_q) return;
    }
    if (i >= s.n) return;
    const int64_t row = ((int64_t)s.row0 + i) * a.q_heads + h;
    const int32_t skip = skipped<F, true>(a, sp, b, s);
    const float *po = sp.o + row * parts * D + d;
    float w[kRowsSplits], top = -kInf, sum = 0.0f;
    if (!kShares<F>) load(row);
    if (kShares<F>)
#pragma unroll
        for (int k = 0; k < kRowsSplits; ++k) x[k] = k < skip || k >= parts ? -kInf : x[k];
#pragma unroll
    for (int k = 0; k < kRowsSplits; ++k) top = fmaxf(top, x[k]);
#pragma unroll
    for (int k = 0; k < kRowsSplits; ++k) {
        w[k] = k >= parts || x[k] == -kInf ? 0.0f : x[k] == top ? 1.0f : __builtin_amdgcn_exp2f(x[k] - top);
        sum += w[k];
    }
    // weights divided by their sum: the parts' own could leave fp32's range
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    f4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k0 = 0; k0 < kRowsSplits; k0 += 4) {
        if (k0 >= parts) break;
        f4 p[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)  // a part of weight 0 wrote nothing
            p[u] = k0 + u < parts && x[k0 + u] != -kInf ? *reinterpret_cast<const f4 *>(po + (int64_t)(k0 + u) * D)
                                                            : f4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 4; ++u) v += p[u] * (w[k0 + u] * inv);
    }
    store_o4<BF16>(a.o, ((int64_t)s.row0 + i) * a.o_token + (int64_t)h * a.o_head + d, v);
}

// Joins a row's parts, a workgroup a row: the weights first, then the parts by
// as many groups of D / 4 threads as there are, four loads each under way.

template <bool BF16, Form F>
__global__ __launch_bounds__(256) void k_attention_join(AttentionArgs a, Split sp) {
    __shared__ float weight[kMostSplits];
    __shared__ f4 buf[256];
    const int32_t D = a.t.dim, q4 = D >> 2, lane = threadIdx.x & 63;
    const int32_t parts = parts_of<F>(sp);
    int32_t b, i, h;
    SeqRows s;
    float x0 = -kInf, x1 = -kInf;
    auto load = [&](int64_t row, int32_t skip) {
        x0 = lane < parts && lane >= skip ? sp.lse[row * parts + lane] : -kInf;
        x1 = lane + 64 < parts && lane + 64 >= skip ? sp.lse[row * parts + lane + 64] : -kInf;
    };
    if constexpr (kShares<F>) {
        load(blockIdx.x, 0);  // under way while the sequence is looked for
        i = blockIdx.x / a.q_heads, h = blockIdx.x - i * a.q_heads;
        b = sequence_of(a, i);
        if (b >= a.t.seqs) return;
        s = seq_rows(a.t, b);
        i -= s.row0;
        if (i < 0 || i >= a.max_q) return;
    } else {
        const int64_t per = a.max_q * a.q_heads;
        b = (int32_t)(blockIdx.x / per), i = (int32_t)(blockIdx.x % per / a.q_heads), h = (int32_t)(blockIdx.x % a.q_heads);
        s = seq_rows(a.t, b);
    }
    if (i >= s.n) return;
    const int64_t row = ((int64_t)s.row0 + i) * a.q_heads + h;
    const int32_t skip = skipped<F, false>(a, sp, b, s);
    const float *po = sp.o + row * parts * D;
    if constexpr (kShares<F>)
        x0 = lane < skip ? -kInf : x0, x1 = lane + 64 < skip ? -kInf : x1;
    else
        load(row, skip);
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
    const float inv = kShares<F> && sum == 0.0f ? 0.0f : 1.0f / sum;
    if (threadIdx.x < 64) weight[lane] = x0 == -kInf ? -1.0f : w0 * inv, weight[lane + 64] = x1 == -kInf ? -1.0f : w1 * inv;
    __syncthreads();
    const int32_t groups = 256 / q4, grp = threadIdx.x / q4, d = threadIdx.x % q4 * 4;
    f4 v{0.f, 0.f, 0.f, 0.f};
    if (grp < groups)
        for (int32_t k0 = grp; k0 < parts; k0 += 4 * groups) {
            f4 p[4];
            float w[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int32_t k = k0 + u * groups;
                w[u] = k < parts ? weight[k] : -1.0f;
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

// columns that the kernels are built for; the one for many rows also for 96,
// whose products are three quarters of 128's (4 x 300 queries of heads of 96 in
// fp32 behind a window and sinks 42.5 us, on 128 columns 47.8; without sinks 4 x
// 333 45.2, 52.1)
inline int width_of(int64_t dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
inline int many_width_of(int64_t dim) { return dim > 64 && dim <= 96 ? 96 : width_of(dim); }

// one kernel's division of rows of `pairs` (sequence, KV head), that see `span`
// tokens at most
inline Plan divide(bool few, int64_t pairs, int64_t rows, int64_t span) {
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
inline bool few_rows(int64_t pairs, int64_t dim, int64_t rows, int64_t max_kv) {
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
    return few;
}
inline Plan make_plan(int64_t seqs, int64_t q_heads, int64_t kv_heads, int64_t dim, int64_t max_q, int64_t max_kv,
                      int64_t window, int64_t sinks) {
    const int64_t rows = max_q * (q_heads / kv_heads), pairs = seqs * kv_heads;
    int64_t span = max_kv;  // tokens that a row tile can see
    const int64_t tile = window + max_q + 64 + (sinks + 63) / 64 * 64;
    if (window > 0 && tile < span) span = tile;
    return divide(few_rows(pairs, dim, rows, max_kv), pairs, rows, span);
}

template <Form F, int DC, int NQ, int NP>
void start_few(const AttentionArgs &a, const Split &sp, unsigned grid, hipStream_t s) {
    hipLaunchKernelGGL((k_attention_few<DC, NQ, NP, kFewWaves, F>), dim3(grid), dim3(kFewWaves * 64), 0, s, a, sp);
}

template <Form F, int DP, int NQ, int NP>
void start_many(const AttentionArgs &a, const Split &sp, unsigned grid, hipStream_t s) {
    if (a.t.dim == DP)
        hipLaunchKernelGGL((k_attention_many<DP, true, NQ, NP, F>), dim3(grid), dim3(kManyWaves * 64), 0, s, a, sp);
    else
        hipLaunchKernelGGL((k_attention_many<DP, false, NQ, NP, F>), dim3(grid), dim3(kManyWaves * 64), 0, s, a, sp);
}

// NQ = 1: q is bf16; NP = 1: o is
template <Form F, int NQ, int NP>
hipError_t start_attention_few(const AttentionArgs &a, const Plan &p, hipStream_t s) {
    const unsigned grid = (unsigned)p.groups;
    const int width = width_of(a.t.dim);
    width == 64    ? start_few<F, 1, NQ, NP>(a, p.sp, grid, s)
    : width == 128 ? start_few<F, 2, NQ, NP>(a, p.sp, grid, s)
                   : start_few<F, 4, NQ, NP>(a, p.sp, grid, s);
    return hipGetLastError();
}
template <Form F, int NQ, int NP>
hipError_t start_attention_many(const AttentionArgs &a, const Plan &p, hipStream_t s) {
    const unsigned grid = (unsigned)p.groups;
    const int width = many_width_of(a.t.dim);
    width == 64    ? start_many<F, 64, NQ, NP>(a, p.sp, grid, s)
    : width == 96  ? start_many<F, 96, NQ, NP>(a, p.sp, grid, s)
    : width == 128 ? start_many<F, 128, NQ, NP>(a, p.sp, grid, s)
                   : start_many<F, 256, NQ, NP>(a, p.sp, grid, s);
    return hipGetLastError();
}

// rows that a join goes through, and its workgroups: from 512 rows on many rows
// a workgroup (8 x 16 x 32 rows of 4 parts 40.5 us with attention, a workgroup a
// row 44; 16384 rows of 2 parts 22 and 43; 128 rows of 16 parts 15.7 and 15.0,
// before the parts' weights were divided)
struct Join {
    int64_t rows, groups;
    bool many;
};
inline Join make_join(int64_t rows, int64_t parts, int64_t dim) {
    const int64_t per = 1024 / dim;
    const bool many = rows >= 512 && parts <= kRowsSplits;
    return Join{rows, many ? (rows + per - 1) / per : rows, many};
}

template <Form F, int NP>
hipError_t start_join(const AttentionArgs &a, const Split &sp, int32_t parts, hipStream_t s) {
    const Join j = make_join((kShares<F> ? a.t.tokens : a.t.seqs * a.max_q) * a.q_heads, parts, a.t.dim);
    if (j.many)
        hipLaunchKernelGGL((k_attention_join_rows<NP == 1, F>), dim3((unsigned)j.groups), dim3(256), 0, s, a, sp, (uint32_t)j.rows);
    else
        hipLaunchKernelGGL((k_attention_join<NP == 1, F>), dim3((unsigned)j.groups), dim3(256), 0, s, a, sp);
    return hipGetLastError();
}

// the divisors of a plan's indexes
inline void set_divisors(Split &sp, const AttentionArgs &a) {
    sp.group = a.q_heads / a.t.heads;
    sp.by_splits = Divider::of(sp.splits), sp.by_tiles = Divider::of(sp.tiles);
    sp.by_heads = Divider::of(a.t.heads), sp.by_group = Divider::of(sp.group);
    sp.by_per = Divider::of((int64_t)sp.tiles * sp.splits);
}

// a call over one plan: attention, and the join where its rows are in parts
template <Form F, int NQ, int NP>
hipError_t launch_t(const AttentionArgs &a, const Plan &p, hipStream_t s) {
    const hipError_t err = p.few ? start_attention_few<F, NQ, NP>(a, p, s) : start_attention_many<F, NQ, NP>(a, p, s);
    return err != hipSuccess || p.sp.splits == 1 ? err : start_join<F, NP>(a, p.sp, p.sp.splits, s);
}
template <Form F>
hipError_t launch_form(const AttentionArgs &a, Plan &p, void *work, hipStream_t s, const char **kernel) {
    set_divisors(p.sp, a);
    p.sp.o = static_cast<float *>(work);
    p.sp.lse = p.sp.o + (int64_t)a.t.tokens * a.q_heads * p.sp.splits * a.t.dim;
    const bool join = p.sp.splits > 1;
    *kernel = p.few ? (join ? "attention_few, attention_join" : "attention_few")
                    : (join ? "attention_many, attention_join" : "attention_many");
    if (a.q_bf16) return a.o_bf16 ? launch_t<F, 1, 1>(a, p, s) : launch_t<F, 1, 2>(a, p, s);
    return a.o_bf16 ? launch_t<F, 2, 1>(a, p, s) : launch_t<F, 2, 2>(a, p, s);
}

}  // namespace
}  // namespace lcml
