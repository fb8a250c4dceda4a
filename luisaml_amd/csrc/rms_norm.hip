// rms_norm.hip -- residual addition, root-mean-square norm and E4M3 codes of
// the result in one kernel (gfx950).
//
//   h = x + residual (rounded to the residual's type, and stored)
//   v = h * r * gamma,  r = 1 / sqrt(mean(h^2) + eps)        (fp32)
//   y = E4M3(v / s),    s given, amax|v|/448 of each row, or of the tensor
//
// HBM-bound: one workgroup holds a row in registers between its sum of
// squares, its maximum and its codes, so each input is read once.  Only the
// scale of a whole tensor needs a second pass (the maximum over all rows
// comes first): the first one leaves h, r and one partial maximum for each
// workgroup, the second reads h again, from the memory-side cache where it
// fits there.
//
// Measured: a row of 4096 takes 3.7 us, a launch with one round trip to memory
// and two barriers.  4096 x 4096 with x in bf16, an fp32 residual and one scale
// for the tensor, 185 MB at the least: 29.7 us for the first pass (168 MB, 5.6
// TB/s) and 22 for the second (84 MB, 3.8 TB/s).  4096 x 6144 in bf16 with a
// scale a row, 176 MB: 41 us, 4.2 TB/s.
#include "lcml_internal.hpp"

namespace lcml {
namespace {

typedef float f4 __attribute__((ext_vector_type(4)));

// four elements from any element-aligned address
struct __attribute__((packed, aligned(4))) F4 {
    float v[4];
};
struct __attribute__((packed, aligned(2))) H4 {
    uint16_t v[4];
};
struct __attribute__((packed, aligned(1))) C4 {
    uint32_t v;
};

__device__ inline float widen(uint16_t h) { return bits_f32((uint32_t)h << 16); }

template <bool BF16>
__device__ inline f4 load4(const void *p, int64_t i) {
    if constexpr (BF16) {
        const H4 q = *reinterpret_cast<const H4 *>(static_cast<const uint16_t *>(p) + i);
        return f4{widen(q.v[0]), widen(q.v[1]), widen(q.v[2]), widen(q.v[3])};
    } else {
        const F4 q = *reinterpret_cast<const F4 *>(static_cast<const float *>(p) + i);
        return f4{q.v[0], q.v[1], q.v[2], q.v[3]};
    }
}

template <bool BF16>
__device__ inline float load1(const void *p, int64_t i) {
    if constexpr (BF16)
        return widen(static_cast<const uint16_t *>(p)[i]);
    else
        return static_cast<const float *>(p)[i];
}

// how a row of H is taken in groups of four
enum { kWhole = 0, kOdd = 1, kTiny = 2 };  // H % 4 == 0; H > 4; H < 4

// elements i .. i+3 of a row of H, zero past its end, without a branch: past
// the last whole group the row's last four are loaded, and moved into place
template <bool BF16, int CUT>
__device__ inline f4 load_row4(const void *p, int64_t i, int64_t H) {
    const f4 zero{0.f, 0.f, 0.f, 0.f};
    if constexpr (CUT == kTiny) {
        f4 v = zero;
#pragma unroll
        for (int e = 0; e < 3; ++e)
            if (i + e < H) v[e] = load1<BF16>(p, i + e);
        return v;
    }
    f4 v = load4<BF16>(p, i + 4 <= H ? i : H - 4);
    if constexpr (CUT == kOdd) {
        const int64_t by = i + 4 - H;  // 1, 2, 3: that many past the end
        if (by >= 2) v = f4{v[2], v[3], 0.f, 0.f};
        if (by == 1 || by == 3) v = f4{v[1], v[2], v[3], 0.f};
    }
    return i < H ? v : zero;
}

__device__ inline float wave_sum(float v) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
    return v;
}

template <int THREADS>
__device__ inline float block_sum(float v, float *red) {
    v = wave_sum(v);
    if constexpr (THREADS > 64) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = 0.0f;
#pragma unroll
        for (int w = 0; w < THREADS / 64; ++w) v += red[w];
        __syncthreads();
    }
    return v;
}

struct NormArgs {
    const void *x, *res;
    void *res_out;
    const float *gamma;
    uint8_t *y;
    float *scale;
    float *rstd;     // [M], mode kTensor
    uint32_t *part;  // [gridDim.x], mode kTensor
    int64_t M, H, ldx, ldr, ldro, ldy;
    float eps;
    int mode;
};

enum { kStatic = 0, kTensor = 1, kRow = 2 };
// residual: none, fp32, bf16
enum { kNoRes = 0, kResF32 = 1, kResBf16 = 2 };

// x and the residual of four elements of row m, and h from them, rounded to
// the residual's type
template <bool XB, int RES, int CUT>
struct Raw {
    f4 x, r;
    __device__ inline void load(const NormArgs &a, int64_t m, int64_t i) {
        x = load_row4<XB, CUT>(static_cast<const char *>(a.x) + m * a.ldx * (XB ? 2 : 4), i, a.H);
        if constexpr (RES != kNoRes)
            r = load_row4<RES == kResBf16, CUT>(static_cast<const char *>(a.res) + m * a.ldr * (RES == kResBf16 ? 2 : 4), i, a.H);
    }
    __device__ inline f4 h() const {
        if constexpr (RES == kNoRes) return x;
        f4 v = x + r;
        if constexpr (RES == kResBf16)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = widen(bf16_rne(v[e]));
        return v;
    }
};

template <int RES, int CUT>
__device__ inline void store_h(const NormArgs &a, int64_t m, int64_t i, f4 h) {
    if (i >= a.H) return;
    const bool whole = CUT == kWhole || i + 4 <= a.H;
    if constexpr (RES == kResBf16) {
        uint16_t *o = static_cast<uint16_t *>(a.res_out) + m * a.ldro + i;
        H4 q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = (uint16_t)(f32_bits(h[e]) >> 16);
        if (whole)
            *reinterpret_cast<H4 *>(o) = q;
        else
            for (int e = 0; e < 3; ++e)
                if (i + e < a.H) o[e] = q.v[e];
    } else if constexpr (RES == kResF32) {
        float *o = static_cast<float *>(a.res_out) + m * a.ldro + i;
        if (whole)
            *reinterpret_cast<F4 *>(o) = F4{{h[0], h[1], h[2], h[3]}};
        else
            for (int e = 0; e < 3; ++e)
                if (i + e < a.H) o[e] = h[e];
    }
}

template <int CUT>
__device__ inline void store_codes(const NormArgs &a, int64_t m, int64_t i, uint32_t c) {
    if (i >= a.H) return;
    uint8_t *o = a.y + m * a.ldy + i;
    if (CUT == kWhole || i + 4 <= a.H)
        reinterpret_cast<C4 *>(o)->v = c;
    else
        for (int e = 0; e < 3; ++e)
            if (i + e < a.H) o[e] = (uint8_t)(c >> (8 * e));
}

__device__ inline float abs_max4(float m, f4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float b = fabsf(v[e]);
        m = b > m ? b : m;  // false for NaN
    }
    return m;
}

// TPR threads a row (64: four rows of a workgroup side by side, no barriers),
// NV groups of four elements for each thread in registers.  TAIL: rows longer
// than TPR * NV * 4, which read the rest again.  Every input's loads are under
// way before the first is waited for, without a branch (with branches, 52 us
// where this takes 30).
template <bool XB, int RES, int CUT, int TPR, int NV, bool TAIL>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void k_rms_norm(NormArgs a) {
    constexpr int kThreads = TPR < 256 ? 256 : TPR, kRows = kThreads / TPR;
    constexpr int64_t kHeld = (int64_t)TPR * NV * 4;
    __shared__ float red[kThreads / 64];
    const int t = threadIdx.x % TPR;
    auto tail = [&](int64_t m, auto f) {
        if constexpr (TAIL)
            for (int64_t i = kHeld + t * 4; i < a.H; i += TPR * 4) {
                Raw<XB, RES, CUT> raw;
                raw.load(a, m, i);
                f(raw.h(), i);
            }
    };
    const bool store = RES != kNoRes && a.res_out;
    float tensor_max = 0.0f;
    for (int64_t m = (int64_t)blockIdx.x * kRows + threadIdx.x / TPR; m < a.M; m += (int64_t)gridDim.x * kRows) {
        Raw<XB, RES, CUT> raw[NV];
        f4 h[NV], gamma[NV];
        float ss = 0.0f;
        auto at = [&](int u) { return ((int64_t)u * TPR + t) * 4; };
#pragma unroll
        for (int u = 0; u < NV; ++u) raw[u].load(a, m, at(u));
#pragma unroll
        for (int u = 0; u < NV; ++u) gamma[u] = load_row4<false, CUT>(a.gamma, at(u), a.H);
        auto sum = [&](f4 v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(v[e], v[e], ss);
        };
#pragma unroll
        for (int u = 0; u < NV; ++u) sum(h[u] = raw[u].h());
        if (store)
#pragma unroll
            for (int u = 0; u < NV; ++u) store_h<RES, CUT>(a, m, at(u), h[u]);
        tail(m, [&](f4 v, int64_t) { sum(v); });
        ss = block_sum<TPR>(ss, red);
        const float r = 1.0f / sqrtf(ss / (float)a.H + a.eps);
        auto norm = [&](f4 v, int64_t i) { return v * r * load_row4<false, CUT>(a.gamma, i, a.H); };
        float mx = 0.0f, s;
#pragma unroll
        for (int u = 0; u < NV; ++u) mx = abs_max4(mx, h[u] = h[u] * r * gamma[u]);
        if (a.mode == kStatic) {
            s = a.scale[0];
        } else {
            tail(m, [&](f4 v, int64_t i) {
                mx = abs_max4(mx, norm(v, i));
                if (store && a.mode == kTensor) store_h<RES, CUT>(a, m, i, v);  // its last reader in this pass
            });
            if (a.mode == kTensor) {
                tensor_max = fmaxf(tensor_max, mx);
                if (t == 0) a.rstd[m] = r;
                continue;
            }
            if constexpr (TPR == 64)
                mx = wave_max(mx);
            else
                mx = block_max<TPR>(mx, red);
            s = scale_from_amax_bits(f32_bits(mx));
            if (t == 0) a.scale[m] = s;
        }
        const Recip d = make_recip(s);
        auto encode = [&](auto fast) {
            constexpr bool FAST = decltype(fast)::value;
#pragma unroll
            for (int u = 0; u < NV; ++u)
                store_codes<CUT>(a, m, at(u), quantize4_t<FAST>(h[u][0], h[u][1], h[u][2], h[u][3], d));
            tail(m, [&](f4 v, int64_t i) {
                if (store) store_h<RES, CUT>(a, m, i, v);
                const f4 n = norm(v, i);
                store_codes<CUT>(a, m, i, quantize4_t<FAST>(n[0], n[1], n[2], n[3], d));
            });
        };
        if (__builtin_amdgcn_ballot_w64(!d.fast) == 0)
            encode(std::true_type{});
        else
            encode(std::false_type{});
    }
    if (a.mode == kTensor) {
        const float b = block_max<kThreads>(tensor_max, red);
        if (threadIdx.x == 0) a.part[blockIdx.x] = f32_bits(b);
    }
}

// The second pass of one scale for the tensor: codes of h (the stored one, or
// x + residual again), from the rows' r and the partial maxima.
template <bool XB, int RES, int CUT, int NV>
__global__ __launch_bounds__(256) void k_norm_encode(NormArgs a, int npart) {
    __shared__ float red[4];
    const bool stored = RES != kNoRes && a.res_out;
    auto load = [&](int64_t m, int64_t i) {
        if (stored)
            return load_row4<RES == kResBf16, CUT>(
                static_cast<const char *>(a.res_out) + m * a.ldro * (RES == kResBf16 ? 2 : 4), i, a.H);
        Raw<XB, RES, CUT> raw;
        raw.load(a, m, i);
        return raw.h();
    };
    // last rows first: the caches hold what the first pass stored last
    int64_t m = (a.M - 1 - (int64_t)blockIdx.x) / gridDim.x * gridDim.x + blockIdx.x;
    f4 h[NV], gamma[NV];
    float r;
    auto begin = [&](int64_t i0) {
        r = a.rstd[m];
#pragma unroll
        for (int u = 0; u < NV; ++u) h[u] = load(m, i0 + u * 1024);
#pragma unroll
        for (int u = 0; u < NV; ++u) gamma[u] = load_row4<false, CUT>(a.gamma, i0 + u * 1024, a.H);
    };
    const int64_t first = threadIdx.x * 4;
    begin(first);
    // the maxima 16 at a time (one after the other they took 8 us of 25)
    float mx = 0.0f;
    for (int i0 = 0; i0 < npart; i0 += 16 * 256) {
        uint32_t v[16];
#pragma unroll
        for (int k = 0; k < 16; ++k) {
            const int i = i0 + k * 256 + threadIdx.x;
            v[k] = a.part[i < npart ? i : npart - 1];
        }
#pragma unroll
        for (int k = 0; k < 16; ++k) mx = fmaxf(mx, bits_f32(v[k]));
    }
    const float s = scale_from_amax_bits(f32_bits(block_max<256>(mx, red)));
    if (blockIdx.x == 0 && threadIdx.x == 0) a.scale[0] = s;
    const Recip d = make_recip(s);
    auto run = [&](auto fast) {
        for (;;) {
            for (int64_t i0 = first; i0 < a.H; i0 += NV * 1024) {
                if (i0 != first) begin(i0);
#pragma unroll
                for (int u = 0; u < NV; ++u) {
                    const f4 v = h[u] * r * gamma[u];
                    store_codes<CUT>(a, m, i0 + u * 1024, quantize4_t<decltype(fast)::value>(v[0], v[1], v[2], v[3], d));
                }
            }
            m -= gridDim.x;
            if (m < 0) break;
            begin(first);
        }
    };
    if (d.fast)
        run(std::true_type{});
    else
        run(std::false_type{});
}

constexpr int kParts = 4096;  // at most: partial maxima of a tensor

template <bool XB, int RES, int CUT>
hipError_t launch_t(const NormArgs &a, hipStream_t s) {
    const bool two = a.mode == kTensor;
    auto grid = [&](int64_t rows, int64_t most) {
        const int64_t n = (a.M + rows - 1) / rows;
        return (unsigned)(n < most ? n : most);
    };
    const int64_t most = two ? kParts : 1 << 20;
    unsigned n;
    // Threads by the row's length: as many as hold it in four groups each (a
    // wavefront a row of 4096 in 16 groups: 39 us for 4096 of them, against 30),
    // and the number of groups that just holds it: unused ones cost registers
    // and slots of the loads (4096 rows of 6144 in 3 groups of 512 threads 41
    // us, in 4 51; of 1536 in 2 of 256 13, in 4 17; of 300 in 2 of 64 5.2, in 4
    // 6.7).  Up to 256 rows do not fill the GPU: a row's own time counts, and
    // twice the threads with half the groups shorten it (256 rows of 4096, 512
    // threads 4.5 us, 256 threads 5.0; 512 rows 6.2 and 6.5, 4096 rows 29.5 and
    // 26.9; 64 rows of 8000, 1024 threads 5.2, 512 threads 5.5; from 256 rows on
    // equal).  Rows past 8192 take four groups of 1024 threads whatever their
    // length, and read what is past 16384 once more (4096 rows of 12288 in bf16
    // 120 us, 2.9 TB/s); fewer groups were not measured there.
    auto start = [&](auto tpr, auto nv, auto tail) {
        constexpr int TPR = decltype(tpr)::value, kThreads = TPR < 256 ? 256 : TPR;
        n = grid(kThreads / TPR, most);
        hipLaunchKernelGGL((k_rms_norm<XB, RES, CUT, TPR, decltype(nv)::value, decltype(tail)::value>), dim3(n),
                           dim3(kThreads), 0, s, a);
    };
    const std::integral_constant<int, 64> t64;
    const std::integral_constant<int, 256> t256;
    const std::integral_constant<int, 512> t512;
    const std::integral_constant<int, 1024> t1024;
    const std::integral_constant<int, 1> n1;
    const std::integral_constant<int, 2> n2;
    const std::integral_constant<int, 3> n3;
    const std::integral_constant<int, 4> n4;
    const std::false_type whole;
    const std::true_type tail;
    const int64_t q = (a.H + 255) / 256;  // groups of a wavefront
    if constexpr (CUT == kTiny)
        start(t64, n1, whole);
    else if (q <= 4)
        q == 1 ? start(t64, n1, whole) : q == 2 ? start(t64, n2, whole) : q == 3 ? start(t64, n3, whole) : start(t64, n4, whole);
    else if (q <= 8)
        start(t256, n2, whole);
    else if (q <= 16)
        a.M <= 256 ? start(t512, n2, whole) : q <= 12 ? start(t256, n3, whole) : start(t256, n4, whole);
    else if (q <= 24)
        start(t512, n3, whole);
    else if (q <= 32)
        a.M <= 256 ? start(t1024, n2, whole) : start(t512, n4, whole);
    else
        start(t1024, n4, tail);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess || !two) return err;
    auto encode = [&](auto nv) {
        hipLaunchKernelGGL((k_norm_encode<XB, RES, CUT, decltype(nv)::value>), dim3(grid(1, 2048)), dim3(256), 0, s, a, (int)n);
    };
    // a row in rounds of 256 threads x 1 to 4 groups, the fewest rounds and then
    // the fewest groups (4096 rows of 2048 in 2 27 us with the first pass, in 4 33)
    const int64_t rounds = (q + 15) / 16, groups = ((q + 3) / 4 + rounds - 1) / rounds;
    if constexpr (CUT == kTiny)
        encode(n1);
    else
        groups == 1 ? encode(n1) : groups == 2 ? encode(n2) : groups == 3 ? encode(n3) : encode(n4);
    return hipGetLastError();
}

template <bool XB, int RES>
hipError_t launch_t(const NormArgs &a, hipStream_t s) {
    if (a.H < 4) return launch_t<XB, RES, kTiny>(a, s);
    return a.H % 4 ? launch_t<XB, RES, kOdd>(a, s) : launch_t<XB, RES, kWhole>(a, s);
}

}  // namespace

int64_t rms_norm_workspace(int64_t M) { return 4 * (M + kParts); }

hipError_t launch_rms_norm(int64_t M, int64_t H, const void *x, bool x_bf16, int64_t ldx, const void *res,
                           void *res_out, bool res_bf16, int64_t ldr, int64_t ldro, const float *gamma, float eps,
                           uint8_t *y, int64_t ldy, int mode, float *scale, void *work, hipStream_t s) {
    uint32_t *part = static_cast<uint32_t *>(work);
    float *rstd = work ? reinterpret_cast<float *>(part) + kParts : nullptr;
    // one row's scale is its tensor's
    const NormArgs a{x,  res, res_out, gamma, y,   scale, rstd, part, M,
                     H,  ldx, ldr,     ldro,  ldy, eps,   mode == kTensor && M == 1 ? kRow : mode};
    const int r = !res ? kNoRes : res_bf16 ? kResBf16 : kResF32;
    if (x_bf16)
        return r == kNoRes ? launch_t<true, kNoRes>(a, s) : r == kResBf16 ? launch_t<true, kResBf16>(a, s)
                                                                          : launch_t<true, kResF32>(a, s);
    return r == kNoRes ? launch_t<false, kNoRes>(a, s) : r == kResBf16 ? launch_t<false, kResBf16>(a, s)
                                                                       : launch_t<false, kResF32>(a, s);
}

}  // namespace lcml
