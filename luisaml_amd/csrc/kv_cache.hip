// kv_cache.hip -- tokens into an E4M3 cache of pages, and back (gfx950).
//
// Both directions stream: a written token costs 2 or 4 bytes in and one out
// for each element, a read one the inverse.  A thread's unit is 4 tokens x 8
// elements: four row loads of 16 or 32 bytes, and in the cache 4 x 8 bytes of K
// or 32 contiguous bytes of V, which transposes V in registers.  Writing, one
// workgroup takes one page of one head, of K or of V, so the page's maximum,
// its scale and the codes that stay are its own and no order between
// workgroups matters; the new rows stay in registers between the maximum and
// the codes.  Reading, threads take units of consecutive heads, so that a
// workgroup's rows are contiguous across them.
//
// Measured: 64 sequences' tokens of a decode step 4.7 us, a launch's latency
// (index arrays, page, rows and scale, one after the other); 8 x 512 tokens of
// 8 heads of 128 in bf16 10.5 us (25 MB); 16 sequences of up to 8192 tokens,
// 394 MB, 103 us written (3.8 TB/s) and 88 us read back (4.5 TB/s, where a copy
// reaches 4.8).
#include "kv_cache.hpp"
#include "lcml_internal.hpp"

namespace lcml {
namespace {

constexpr int kThreads = 256;  // of a read

struct __attribute__((packed, aligned(2))) H8 {
    uint16_t v[8];
};
struct __attribute__((packed, aligned(4))) F8x32 {
    float v[8];
};
typedef uint32_t u2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));

struct Rows {
    const char *k, *v;      // write: the call's K and V
    char *ko, *vo;          // read: its outputs
    int64_t kt, kh, vt, vh;  // strides in elements: token, head
};

template <bool BF16>
__device__ inline void load8(const char *p, float *x) {
    if constexpr (BF16) {
        const H8 q = *reinterpret_cast<const H8 *>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = bits_f32((uint32_t)q.v[e] << 16);
    } else {
        const F8x32 q = *reinterpret_cast<const F8x32 *>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = q.v[e];
    }
}

// one page that the call touches: K or V, head, and the page's new slots
struct Spot {
    bool is_v;
    int32_t head, page, lo, hi;  // new slots lo .. hi-1
    int64_t row;                 // the call's row of slot 0
};

// spot i of [seqs][pages_per_seq][K, V][heads]; false: no new slot there
__device__ inline bool find_spot(const KvTokens &t, int32_t pages_per_seq, uint32_t i, Spot *s) {
    s->head = i % t.heads;
    i /= t.heads;
    s->is_v = i & 1;
    i >>= 1;
    const int32_t r = i % pages_per_seq, b = i / pages_per_seq;
    const SeqRows q = seq_rows(t, b);
    if (q.n <= 0) return false;
    const int32_t p0 = q.pos0 > 0 ? q.pos0 : 0;
    const int32_t c = (p0 >> t.tshift) + r, T = 1 << t.tshift;
    const int64_t base = (int64_t)c << t.tshift;
    if (base >= q.len) return false;
    s->lo = p0 > base ? (int32_t)(p0 - base) : 0;
    s->hi = q.len - base < T ? (int32_t)(q.len - base) : T;
    s->page = page_of(t, b, c);
    s->row = q.row0 + (base - q.pos0);
    return s->page >= 0 && s->lo < s->hi;
}

// a thread's unit in the cache: 4 slots from t0, 8 elements from e0
template <bool V>
__device__ inline void load_codes(const uint8_t *blk, int32_t t0, int32_t e0, int32_t D, uint32_t w[8]) {
    if constexpr (V) {
        const u4 *p = reinterpret_cast<const u4 *>(blk + v_place(t0, e0, D));
        const u4 a = p[0], b = p[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = a[e], w[4 + e] = b[e];
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const u2 a = *reinterpret_cast<const u2 *>(blk + k_place(t0 + i, e0, D));
            w[2 * i] = a[0], w[2 * i + 1] = a[1];
        }
    }
}

// the code of token i, element e within a unit's eight words
template <bool V>
__device__ constexpr int word_of(int i, int e) {
    return V ? e : 2 * i + (e >> 2);
}
template <bool V>
__device__ constexpr int byte_of(int i, int e) {
    return V ? i : e & 3;
}

__device__ inline uint32_t encode_again(uint32_t w, float k) {
    const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return e4m3x2_hw(a[0] * k, a[1] * k) | (e4m3x2_hw(b[0] * k, b[1] * k) << 16);
}

// NT threads, a unit each in registers; where more hold new tokens, their rows
// are loaded again
template <bool V, bool BF16, int NT>
__device__ inline void write_page(const KvTokens &t, const Spot &sp, const Rows &rows, uint8_t *cache, float *scales,
                                  float *red) {
    const int32_t D = t.dim, d8 = D >> 3;
    const int64_t at = (int64_t)sp.page * t.heads + sp.head;
    uint8_t *blk = cache + (at << t.tshift) * D;
    const char *src = V ? rows.v + (sp.row * rows.vt + sp.head * rows.vh) * (BF16 ? 2 : 4)
                        : rows.k + (sp.row * rows.kt + sp.head * rows.kh) * (BF16 ? 2 : 4);
    const int64_t pitch = (V ? rows.vt : rows.kt) * (BF16 ? 2 : 4);
    const int32_t g0 = (sp.lo >> 2) * d8, g1 = ((sp.hi + 3) >> 2) * d8;  // units with new tokens
    float old = scales[at];
    float m = 0.0f;
    // the new rows of unit g; zeros for the others
    auto load = [&](int32_t g, float (*x)[8]) {
        const int32_t t0 = g / d8 * 4;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[i][e] = 0.0f;
            if (g < g1 && t0 + i >= sp.lo && t0 + i < sp.hi)
                load8<BF16>(src + (int64_t)(t0 + i) * pitch + (int64_t)(g % d8) * 8 * (BF16 ? 2 : 4), x[i]);
        }
    };
    auto amax = [&](const float (*x)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float a = fabsf(x[i][e]);
                m = a > m && a < __builtin_inff() ? a : m;
            }
    };
    float x[4][8];
    load(g0 + threadIdx.x, x);
    amax(x);
    for (int32_t g = g0 + NT + threadIdx.x; g < g1; g += NT) {
        float y[4][8];
        load(g, y);
        amax(y);
    }
    asm volatile("" : "+v"(old));  // every wavefront has it before the barrier that the new one's store follows
    m = NT == 64 ? wave_max(m) : block_max<NT>(m, red);
    float s = page_scale(m), grow = 1.0f;
    if (sp.lo > 0) {  // tokens that stay
        if (old >= s)
            s = old;
        else
            grow = old / s;
    }
    if (threadIdx.x == 0) scales[at] = s;
    const float inv = 1.0f / s;  // a power of two: x * inv is x / s
    auto put = [&](int32_t g, const float (*x)[8]) {
        const int32_t t0 = g / d8 * 4, e0 = g % d8 * 8;
        const bool fresh = t0 < sp.hi && t0 + 4 > sp.lo, stays = t0 < sp.lo && grow != 1.0f;
        if (g >= g1 || !(fresh || stays)) return;
        uint32_t w[8], out[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) w[q] = out[q] = 0;
        if (t0 < sp.lo || t0 + 4 > sp.hi) {  // tokens that stay, or slots past the last one, which keep their bytes
            load_codes<V>(blk, t0, e0, D, w);
            if (stays)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (t0 + i < sp.lo)
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const int wi = word_of<V>(i, e), sh = 8 * byte_of<V>(i, e);
                            const float c = __builtin_amdgcn_cvt_f32_fp8((int)(w[wi] >> sh), 0);
                            w[wi] = (w[wi] & ~(0xffu << sh)) | ((e4m3x2_hw(c * grow, 0.0f) & 0xffu) << sh);
                        }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool now = t0 + i >= sp.lo && t0 + i < sp.hi;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const int wi = word_of<V>(i, e), wj = word_of<V>(i, e + 1);
                const int si = 8 * byte_of<V>(i, e), sj = 8 * byte_of<V>(i, e + 1);
                const uint32_t c = e4m3x2_hw(x[i][e] * inv, x[i][e + 1] * inv);
                out[wi] |= (now ? c & 0xffu : w[wi] >> si & 0xffu) << si;
                out[wj] |= (now ? c >> 8 : w[wj] >> sj & 0xffu) << sj;
            }
        }
        if constexpr (V) {
            u4 *p = reinterpret_cast<u4 *>(blk + v_place(t0, e0, D));
            p[0] = u4{out[0], out[1], out[2], out[3]};
            p[1] = u4{out[4], out[5], out[6], out[7]};
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<u2 *>(blk + k_place(t0 + i, e0, D)) = u2{out[2 * i], out[2 * i + 1]};
        }
    };
    put(g0 + threadIdx.x, x);
    for (int32_t g = g0 + NT + threadIdx.x; g < g1; g += NT) {
        float y[4][8];
        load(g, y);
        put(g, y);
    }
    if (grow != 1.0f)
        for (int32_t g = threadIdx.x; g < g0; g += NT) {
            const float none[4][8] = {};
            put(g, none);
        }
}

template <bool BF16, int NT>
__global__ __launch_bounds__(NT) void k_kv_write(KvTokens t, Rows rows, uint8_t *kc, uint8_t *vc, float *ks, float *vs,
                                                 int32_t pages_per_seq) {
    __shared__ float red[NT / 64];
    Spot sp;
    if (!find_spot(t, pages_per_seq, blockIdx.x, &sp)) return;
    if (sp.is_v)
        write_page<true, BF16, NT>(t, sp, rows, vc, vs, red);
    else
        write_page<false, BF16, NT>(t, sp, rows, kc, ks, red);
}

template <bool V, bool BF16>
__device__ inline void read_unit(const KvTokens &t, const Spot &sp, const Rows &rows, const uint8_t *cache,
                                 const float *scales, int32_t g) {
    const int32_t D = t.dim, d8 = D >> 3, t0 = g / d8 * 4, e0 = g % d8 * 8;
    if (t0 + 4 <= sp.lo || t0 >= sp.hi) return;
    const int64_t at = (int64_t)sp.page * t.heads + sp.head;
    uint32_t w[8];
    load_codes<V>(cache + (at << t.tshift) * D, t0, e0, D, w);
    const float s = scales[at];
    char *dst = V ? rows.vo + ((sp.row + t0) * rows.vt + sp.head * rows.vh + e0) * (BF16 ? 2 : 4)
                  : rows.ko + ((sp.row + t0) * rows.kt + sp.head * rows.kh + e0) * (BF16 ? 2 : 4);
    const int64_t pitch = (V ? rows.vt : rows.kt) * (BF16 ? 2 : 4);
    float x[8][4];  // [word][byte]
#pragma unroll
    for (int q = 0; q < 8; ++q) {
        const f2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], false);
        const f2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[q], true);
        x[q][0] = a[0] * s, x[q][1] = a[1] * s, x[q][2] = b[0] * s, x[q][3] = b[1] * s;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (t0 + i < sp.lo || t0 + i >= sp.hi) continue;
        if constexpr (BF16) {
            H8 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] = bf16_rne(x[word_of<V>(i, e)][byte_of<V>(i, e)]);
            *reinterpret_cast<H8 *>(dst + i * pitch) = o;
        } else {
            F8x32 o;
#pragma unroll
            for (int e = 0; e < 8; ++e) o.v[e] = x[word_of<V>(i, e)][byte_of<V>(i, e)];
            *reinterpret_cast<F8x32 *>(dst + i * pitch) = o;
        }
    }
}

// a unit a thread, in the order [spots][units of a page and head]
template <bool BF16>
__global__ __launch_bounds__(kThreads) void k_kv_read(KvTokens t, Rows rows, const uint8_t *kc, const uint8_t *vc,
                                                      const float *ks, const float *vs, int32_t pages_per_seq,
                                                      uint32_t spots) {
    const uint32_t units = (uint32_t)(t.dim >> 3) << (t.tshift - 2);
    const uint64_t id = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
    const uint32_t i = (uint32_t)(id / units), g = (uint32_t)(id - (uint64_t)i * units);
    Spot sp;
    if (i >= spots || !find_spot(t, pages_per_seq, i, &sp)) return;
    if (sp.is_v)
        read_unit<true, BF16>(t, sp, rows, vc, vs, g);
    else
        read_unit<false, BF16>(t, sp, rows, kc, ks, g);
}

}  // namespace

// pages that max_q tokens of one sequence can touch
int64_t kv_pages_per_seq(int64_t max_q, int tshift) { return ((max_q - 2 + ((int64_t)1 << tshift)) >> tshift) + 1; }

// Threads of a write's workgroup, which has a page of one head: one for each
// unit that can hold a new token.  8 x 512 tokens of 8 heads of 128: 10.3 to
// 10.6 us whatever the page, where 64 and 256 threads alone took 13.7 at pages
// of 32 and 13.4 at pages of 128 tokens (four units a thread there); one token
// in pages of 128 4.7, with threads for the whole page 9.
int kv_write_threads(int64_t max_q, int32_t dim, int tshift) {
    const int64_t groups = (max_q + 2) / 4 + 1, all = (int64_t)1 << (tshift - 2);
    const int64_t units = (groups < all ? groups : all) * (dim >> 3);
    return units <= 64 ? 64 : units <= 128 ? 128 : units <= 256 ? 256 : units <= 512 ? 512 : 1024;
}

template <bool BF16>
static void start_kv_write(const KvTokens &t, const Rows &r, uint8_t *kc, uint8_t *vc, float *ks, float *vs, int64_t max_q,
                           hipStream_t s) {
    const int32_t pp = (int32_t)kv_pages_per_seq(max_q, t.tshift);
    const dim3 grid((unsigned)(2 * (int64_t)t.heads * pp * t.seqs));
    auto start = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        hipLaunchKernelGGL((k_kv_write<BF16, NT>), grid, dim3(NT), 0, s, t, r, kc, vc, ks, vs, pp);
    };
    switch (kv_write_threads(max_q, t.dim, t.tshift)) {
        case 64: return start(std::integral_constant<int, 64>{});
        case 128: return start(std::integral_constant<int, 128>{});
        case 256: return start(std::integral_constant<int, 256>{});
        case 512: return start(std::integral_constant<int, 512>{});
        default: return start(std::integral_constant<int, 1024>{});
    }
}

hipError_t launch_kv_write(const KvTokens &t, int64_t max_q, const void *k, const void *v, bool bf16, int64_t kt,
                           int64_t kh, int64_t vt, int64_t vh, uint8_t *kc, uint8_t *vc, float *ks, float *vs,
                           hipStream_t s) {
    const Rows rows{(const char *)k, (const char *)v, nullptr, nullptr, kt, kh, vt, vh};
    bf16 ? start_kv_write<true>(t, rows, kc, vc, ks, vs, max_q, s)
         : start_kv_write<false>(t, rows, kc, vc, ks, vs, max_q, s);
    return hipGetLastError();
}

hipError_t launch_kv_read(const KvTokens &t, int64_t max_q, void *k, void *v, bool bf16, int64_t kt, int64_t kh,
                          int64_t vt, int64_t vh, const uint8_t *kc, const uint8_t *vc, const float *ks,
                          const float *vs, hipStream_t s) {
    const Rows rows{nullptr, nullptr, (char *)k, (char *)v, kt, kh, vt, vh};
    const int64_t pp = kv_pages_per_seq(max_q, t.tshift), spots = 2 * t.heads * pp * t.seqs;
    const int64_t units = (int64_t)(t.dim >> 3) << (t.tshift - 2);
    const dim3 grid((unsigned)((spots * units + kThreads - 1) / kThreads));
    if (bf16)
        hipLaunchKernelGGL((k_kv_read<true>), grid, dim3(kThreads), 0, s, t, rows, kc, vc, ks, vs, (int32_t)pp, (uint32_t)spots);
    else
        hipLaunchKernelGGL((k_kv_read<false>), grid, dim3(kThreads), 0, s, t, rows, kc, vc, ks, vs, (int32_t)pp, (uint32_t)spots);
    return hipGetLastError();
}

}  // namespace lcml
