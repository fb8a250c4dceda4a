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

// elements i .. i+3 of a row of H; zero past its end
template <bool BF16>
__device__ inline f4 load_row4(const void *p, int64_t i, int64_t H) {
    if (i + 4 <= H) return load4<BF16>(p, i);
    f4 v{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e)
        if (i + e < H) v[e] = load1<BF16>(p, i + e);
    return v;
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

// h of four elements of row m, rounded to the residual's type
template <bool XB, int RES>
__device__ inline f4 load_h(const NormArgs &a, int64_t m, int64_t i) {
    const char *xr = static_cast<const char *>(a.x) + m * a.ldx * (XB ? 2 : 4);
    f4 v = load_row4<XB>(xr, i, a.H);
    if constexpr (RES != kNoRes) {
        const char *rr = static_cast<const char *>(a.res) + m * a.ldr * (RES == kResBf16 ? 2 : 4);
        v += load_row4<RES == kResBf16>(rr, i, a.H);
        if constexpr (RES == kResBf16)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = widen(bf16_rne(v[e]));
    }
    return v;
}

template <int RES>
__device__ inline void store_h(const NormArgs &a, int64_t m, int64_t i, f4 h) {
    if constexpr (RES == kResBf16) {
        uint16_t *o = static_cast<uint16_t *>(a.res_out) + m * a.ldro + i;
        H4 q;
#pragma unroll
        for (int e = 0; e < 4; ++e) q.v[e] = (uint16_t)(f32_bits(h[e]) >> 16);
        if (i + 4 <= a.H)
            *reinterpret_cast<H4 *>(o) = q;
        else
            for (int e = 0; e < 4 && i + e < a.H; ++e) o[e] = q.v[e];
    } else if constexpr (RES == kResF32) {
        float *o = static_cast<float *>(a.res_out) + m * a.ldro + i;
        if (i + 4 <= a.H)
            *reinterpret_cast<F4 *>(o) = F4{{h[0], h[1], h[2], h[3]}};
        else
            for (int e = 0; e < 4 && i + e < a.H; ++e) o[e] = h[e];
    }
}

__device__ inline void store_codes(const NormArgs &a, int64_t m, int64_t i, uint32_t c) {
    uint8_t *o = a.y + m * a.ldy + i;
    if (i + 4 <= a.H)
        reinterpret_cast<C4 *>(o)->v = c;
    else
        for (int e = 0; e < 4 && i + e < a.H; ++e) o[e] = (uint8_t)(c >> (8 * e));
}

__device__ inline float abs_max4(float m, f4 v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float b = fabsf(v[e]);
        m = b > m ? b : m;  // false for NaN
    }
    return m;
}

// One row at a time; NV groups of four elements for each thread stay in
// registers.  Rows longer than THREADS * NV * 4 read their tail again.
template <bool XB, int RES, int THREADS, int NV>
__global__ __launch_bounds__(THREADS) void k_rms_norm(NormArgs a) {
    __shared__ float red[THREADS / 64];
    constexpr int64_t kHeld = (int64_t)THREADS * NV * 4;
    float tensor_max = 0.0f;
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        f4 h[NV];
        float ss = 0.0f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int64_t i = ((int64_t)u * THREADS + threadIdx.x) * 4;
            h[u] = i < a.H ? load_h<XB, RES>(a, m, i) : f4{0.f, 0.f, 0.f, 0.f};
        }
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int64_t i = ((int64_t)u * THREADS + threadIdx.x) * 4;
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(h[u][e], h[u][e], ss);
            if (RES != kNoRes && a.res_out && i < a.H) store_h<RES>(a, m, i, h[u]);
        }
        for (int64_t i = kHeld + threadIdx.x * 4; i < a.H; i += THREADS * 4) {
            const f4 v = load_h<XB, RES>(a, m, i);
#pragma unroll
            for (int e = 0; e < 4; ++e) ss = fmaf(v[e], v[e], ss);
        }
        ss = block_sum<THREADS>(ss, red);
        const float r = 1.0f / sqrtf(ss / (float)a.H + a.eps);
        auto norm = [&](f4 v, int64_t i) { return v * r * load_row4<false>(a.gamma, i, a.H); };
        float mx = 0.0f;
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int64_t i = ((int64_t)u * THREADS + threadIdx.x) * 4;
            if (i < a.H) h[u] = norm(h[u], i);
            mx = abs_max4(mx, h[u]);
        }
        float s;
        if (a.mode == kStatic) {
            s = a.scale[0];
        } else {
            for (int64_t i = kHeld + threadIdx.x * 4; i < a.H; i += THREADS * 4)
                mx = abs_max4(mx, norm(load_h<XB, RES>(a, m, i), i));
            if (a.mode == kTensor) {
                tensor_max = fmaxf(tensor_max, mx);
                if (threadIdx.x == 0) a.rstd[m] = r;
                // the tail's h, after its last reader in this row
                if (RES != kNoRes && a.res_out)
                    for (int64_t i = kHeld + threadIdx.x * 4; i < a.H; i += THREADS * 4)
                        store_h<RES>(a, m, i, load_h<XB, RES>(a, m, i));
                continue;
            }
            s = scale_from_amax_bits(f32_bits(block_max<THREADS>(mx, red)));
            if (threadIdx.x == 0) a.scale[m] = s;
        }
        const Recip d = make_recip(s);
#pragma unroll
        for (int u = 0; u < NV; ++u) {
            const int64_t i = ((int64_t)u * THREADS + threadIdx.x) * 4;
            const uint32_t c = quantize4(h[u][0], h[u][1], h[u][2], h[u][3], d);
            if (i < a.H) store_codes(a, m, i, c);
        }
        for (int64_t i = kHeld + threadIdx.x * 4; i < a.H; i += THREADS * 4) {
            const f4 t = load_h<XB, RES>(a, m, i);
            if (RES != kNoRes && a.res_out) store_h<RES>(a, m, i, t);
            const f4 v = norm(t, i);
            store_codes(a, m, i, quantize4(v[0], v[1], v[2], v[3], d));
        }
    }
    if (a.mode == kTensor) {
        const float b = block_max<THREADS>(tensor_max, red);
        if (threadIdx.x == 0) a.part[blockIdx.x] = f32_bits(b);
    }
}

// The second pass of one scale for the tensor: codes of h (the stored one, or
// x + residual again), from the rows' r and the partial maxima.
template <bool XB, int RES, int THREADS>
__global__ __launch_bounds__(THREADS) void k_norm_encode(NormArgs a, int npart) {
    __shared__ float red[THREADS / 64];
    const float s = scale_from_partials<THREADS>(a.part, npart, red);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.scale[0] = s;
    const Recip d = make_recip(s);
    for (int64_t m = blockIdx.x; m < a.M; m += gridDim.x) {
        const float r = a.rstd[m];
        for (int64_t i = threadIdx.x * 4; i < a.H; i += THREADS * 4) {
            f4 h;
            if (RES != kNoRes && a.res_out)
                h = load_row4<RES == kResBf16>(static_cast<const char *>(a.res_out) +
                                                   m * a.ldro * (RES == kResBf16 ? 2 : 4), i, a.H);
            else
                h = load_h<XB, RES>(a, m, i);
            const f4 v = h * r * load_row4<false>(a.gamma, i, a.H);
            store_codes(a, m, i, quantize4(v[0], v[1], v[2], v[3], d));
        }
    }
}

template <bool XB, int RES>
hipError_t launch_t(const NormArgs &a, hipStream_t s) {
    const bool two = a.mode == kTensor;
    const int64_t most = two ? kMaxAmaxPartials : 1 << 20;
    const unsigned grid = (unsigned)(a.M < most ? a.M : most);
    if (a.H <= 1024)
        hipLaunchKernelGGL((k_rms_norm<XB, RES, 64, 4>), dim3(grid), dim3(64), 0, s, a);
    else
        hipLaunchKernelGGL((k_rms_norm<XB, RES, 256, 4>), dim3(grid), dim3(256), 0, s, a);
    hipError_t err = hipGetLastError();
    if (err != hipSuccess || !two) return err;
    hipLaunchKernelGGL((k_norm_encode<XB, RES, 256>), dim3(grid), dim3(256), 0, s, a, (int)grid);
    return hipGetLastError();
}

}  // namespace

int64_t rms_norm_workspace(int64_t M) { return 4 * (M + kMaxAmaxPartials); }

hipError_t launch_rms_norm(int64_t M, int64_t H, const void *x, bool x_bf16, int64_t ldx, const void *res,
                           void *res_out, bool res_bf16, int64_t ldr, int64_t ldro, const float *gamma, float eps,
                           uint8_t *y, int64_t ldy, int mode, float *scale, void *work, hipStream_t s) {
    // one row's scale is its tensor's
    NormArgs a{x,   res, res_out, gamma, y,   scale, static_cast<float *>(work) + kMaxAmaxPartials, static_cast<uint32_t *>(work),
               M,   H,   ldx,     ldr,   ldro, ldy,  eps, mode == kTensor && M == 1 ? kRow : mode};
    const int r = !res ? kNoRes : res_bf16 ? kResBf16 : kResF32;
    if (x_bf16)
        return r == kNoRes ? launch_t<true, kNoRes>(a, s) : r == kResBf16 ? launch_t<true, kResBf16>(a, s)
                                                                          : launch_t<true, kResF32>(a, s);
    return r == kNoRes ? launch_t<false, kNoRes>(a, s) : r == kResBf16 ? launch_t<false, kResBf16>(a, s)
                                                                       : launch_t<false, kResF32>(a, s);
}

}  // namespace lcml
