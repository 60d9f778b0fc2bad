// Activations kept in 8 bits for the backward pass, and the experts' SwiGLU that writes and reads them.
//
// Format: each 32 consecutive values of a row share one scale byte b, the power of two 2^(b - 127) (255: NaN), and are signed 8-bit
// codes of at most 127 in magnitude. Codes [rows][cols], scales [rows][cols / 32]. With a block's largest magnitude m 2^k (1 <= m < 2) the
// scale is 2^(k - 6): a value is off by at most half of 2^(k - 6), by one whole where m 2^6 rounds to 128 and is held at 127.
#include "common.hpp"
#include "mx8.hpp"

#include "../../include/flashrt_moe.h"

namespace frt {

typedef uint32_t u4e4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4e2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef float f8_t __attribute__((ext_vector_type(8)));
typedef float f4_t __attribute__((ext_vector_type(4)));

// Eight values of a row as fp32, at the element's own alignment
__device__ __forceinline__ f8_t load8(const float* p) {
    const f4_t x = __builtin_bit_cast(f4_t, *reinterpret_cast<const u4e4_t*>(p)), y = __builtin_bit_cast(f4_t, *reinterpret_cast<const u4e4_t*>(p + 4));
    return __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T>
__device__ __forceinline__ f8_t load8(const T* p) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    return __builtin_convertvector(__builtin_bit_cast(v8, *reinterpret_cast<const u4e2_t*>(p)), f8_t);
}
__device__ __forceinline__ void store8(float* p, f8_t v) {
    *reinterpret_cast<u4e4_t*>(p) = __builtin_bit_cast(u4e4_t, __builtin_shufflevector(v, v, 0, 1, 2, 3));
    *reinterpret_cast<u4e4_t*>(p + 4) = __builtin_bit_cast(u4e4_t, __builtin_shufflevector(v, v, 4, 5, 6, 7));
}
template <typename T>
__device__ __forceinline__ void store8(T* p, f8_t v) {
    typedef T v8 __attribute__((ext_vector_type(8)));
    *reinterpret_cast<u4e2_t*>(p) = __builtin_bit_cast(u4e2_t, __builtin_convertvector(v, v8));
}
// Up to eight values of a row shorter than that (the others 0)
template <typename T>
__device__ __forceinline__ f8_t load_few(const T* p, int n) {
    f8_t v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? float(p[i]) : 0.0f;
    return v;
}
template <typename T>
__device__ __forceinline__ void store_few(T* p, f8_t v, int n) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (i < n) p[i] = T(v[i]);
}

// Codes and scale byte of a block of 32, of which each of four neighbouring lanes has eight values. The byte is the exponent field of
// the largest magnitude less 6, at least 0 (2^-127, all smaller blocks); x 2^-(k - 6) is an exact product (its low bits are lost only far
// below half a step) and is rounded to the nearest even integer. An infinity or a NaN (the exponent field 255) makes the block NaN, codes 0.
__device__ __forceinline__ u2_t encode8(f8_t v, uint32_t& byte) {
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = v[j];
        top = max(top, __builtin_bit_cast(uint32_t, f) & 0x7fffffffu);
    }
    top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), kDppXor1, 0xF, 0xF, true)));
    top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), kDppXor2, 0xF, 0xF, true)));
    const bool bad = top >= 0x7f800000u;
    byte = bad ? 255u : uint32_t(max(int(top >> 23) - 6, 0));
    const float inv = __builtin_bit_cast(float, (254u - min(byte, 248u)) << 23);   // 2^(127 - b)
    u2_t q = {0, 0};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int c = int(fminf(fmaxf(__builtin_rintf(v[j] * inv), -127.0f), 127.0f));
        q[j / 4] |= (uint32_t(c) & 255u) << (8 * (j % 4));
    }
    return bad ? u2_t{0, 0} : q;
}

// A row of 8-value pieces per thread index i: the row and the piece's first column
struct Place {
    uint32_t r;
    int c;
};
__device__ __forceinline__ Place place(uint32_t i, uint32_t per_row, const FastDiv& div) {
    const uint32_t r = div(i);
    return {r, int(i - r * per_row) * 8};
}

// A lane has eight values of a row, four lanes a block. Bound by HBM, with the inverse below (8192 x 2560 bf16 there and back, the codes in the last
// cache between them, 24 us).
template <typename T>
__global__ void __launch_bounds__(256) k_mx8_quantize(const T* __restrict__ x, int64_t ldx, uint32_t pieces, uint32_t per_row, FastDiv div,
                                                      u2_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;   // (pieces is a multiple of 4: whole quads stay or go)
    if (i >= pieces) return;
    const Place at = place(i, per_row, div);
    uint32_t b;
    codes[i] = encode8(load8(x + at.r * ldx + at.c), b);
    if ((i & 3) == 0) scales[i >> 2] = uint8_t(b);
}

template <typename T>
__global__ void __launch_bounds__(256) k_mx8_dequantize(const u2_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t pieces,
                                                        uint32_t per_row, FastDiv div, T* __restrict__ out, int64_t ldout) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const Place at = place(i, per_row, div);
    const u2_t q = codes[i];
    store8(out + at.r * ldout + at.c, mx8_values(q.x, q.y, mx8_scale(scales[i >> 2])));
}

// The sigmoid of g. 1 / (1 + exp(-g)) is 0 where exp overflows and NaN for a NaN; rows of 16 bits take the hardware's exponential and reciprocal
// (off by a few steps of fp32 and |g| more, far below a step of the row's type); the reciprocal is taken of a fourth, so that the subnormal s of
// gates below -87.3, which the hardware's would give as 0, is formed by the product.
template <typename T>
__device__ __forceinline__ float sigmoid(float g) {
    if constexpr (sizeof(T) == 4) return 1.0f / (1.0f + expf(-g));
    return 0.25f * __builtin_amdgcn_rcpf(0.25f * (1.0f + __expf(-g)));
}

// h = g s(g) u of rows z = g | u, eight values of each half per lane; KEEP: z in 8 bits too (ff a multiple of 32, so that four lanes hold
// whole blocks of both halves). Rows from *live on stay as they were. The last piece of a row of an odd width is moved back to
// end with it. Bound by HBM: 77824 rows of ff 640 in bf16 with the 8-bit copy, and the gradient below from it with h again, 161 us, 5.6 TB/s.
template <typename T, bool KEEP>
__global__ void __launch_bounds__(256) k_swiglu(const T* __restrict__ z, int64_t ldz, uint32_t pieces, uint32_t per_row, FastDiv div, int ff,
                                                const int32_t* __restrict__ live, uint32_t row0, T* __restrict__ h, int64_t ldh,
                                                u2_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    Place at = place(i, per_row, div);
    if (live && int64_t(row0) + at.r >= *live) return;
    if (at.c + 8 > ff) at.c = max(0, ff - 8);
    const T* const zr = z + at.r * ldz + at.c;
    const bool few = ff < 8;
    const f8_t g = few ? load_few(zr, ff) : load8(zr), u = few ? load_few(zr + ff, ff) : load8(zr + ff);
    f8_t o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = g[j] * sigmoid<T>(g[j]) * u[j];
    T* const hr = h + at.r * ldh + at.c;
    if (few)
        store_few(hr, o, ff);
    else
        store8(hr, o);
    if constexpr (KEEP) {
        const uint64_t p = uint64_t(at.r) * (2 * per_row) + at.c / 8;   // the piece of g in the codes
        uint32_t bg, bu;
        codes[p] = encode8(g, bg);
        codes[p + per_row] = encode8(u, bu);
        if ((i & 3) == 0) {
            scales[p / 4] = uint8_t(bg);
            scales[(p + per_row) / 4] = uint8_t(bu);
        }
    }
}

// dz of the same, from dh and z (or z in 8 bits), and h again where asked: dg = dh u s (1 + g (1 - s)), du = dh g s
template <typename T, bool KEPT>
__global__ void __launch_bounds__(256) k_swiglu_grad(const T* __restrict__ dh, int64_t lddh, const T* __restrict__ z, int64_t ldz,
                                                     const u2_t* __restrict__ codes, const uint8_t* __restrict__ scales, uint32_t pieces,
                                                     uint32_t per_row, FastDiv div, int ff, const int32_t* __restrict__ live, uint32_t row0,
                                                     T* __restrict__ dz, int64_t lddz, T* __restrict__ h, int64_t ldh) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    Place at = place(i, per_row, div);
    if (live && int64_t(row0) + at.r >= *live) return;
    if (at.c + 8 > ff) at.c = max(0, ff - 8);
    const bool few = ff < 8;
    f8_t g, u;
    if constexpr (KEPT) {
        const uint64_t p = uint64_t(at.r) * (2 * per_row) + at.c / 8;
        const u2_t qg = codes[p], qu = codes[p + per_row];
        g = mx8_values(qg.x, qg.y, mx8_scale(scales[p / 4]));
        u = mx8_values(qu.x, qu.y, mx8_scale(scales[(p + per_row) / 4]));
    } else {
        const T* const zr = z + at.r * ldz + at.c;
        g = few ? load_few(zr, ff) : load8(zr);
        u = few ? load_few(zr + ff, ff) : load8(zr + ff);
    }
    const T* const dr = dh + at.r * lddh + at.c;
    const f8_t d = few ? load_few(dr, ff) : load8(dr);
    f8_t dg, du, o;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float s = sigmoid<T>(g[j]), gs = g[j] * s;
        dg[j] = d[j] * u[j] * (s * (1.0f + g[j] * (1.0f - s)));
        du[j] = d[j] * gs;
        o[j] = gs * u[j];
    }
    T* const zo = dz + at.r * lddz + at.c;
    T* const hr = h + at.r * ldh + at.c;
    if (few) {
        store_few(zo, dg, ff);
        store_few(zo + ff, du, ff);
        if (h) store_few(hr, o, ff);
    } else {
        store8(zo, dg);
        store8(zo + ff, du);
        if (h) store8(hr, o);
    }
}

// Rows of one launch: fewer than 2^31 pieces of 8 values
static int64_t launch_rows(int64_t per_row) { return int64_t(0x7fffff00) / per_row > 0 ? int64_t(0x7fffff00) / per_row : 1; }

template <typename T>
static int quantize_t(const void* x, int64_t ldx, int64_t rows, int cols, void* codes, void* scales, hipStream_t stream) {
    const int64_t per_row = cols / 8, most = launch_rows(per_row);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * per_row);
        launch_timed("mx8_quantize", k_mx8_quantize<T>, dim3((pieces + 255) / 256), dim3(256), 0, stream, static_cast<const T*>(x) + r * ldx,
                     ldx, pieces, uint32_t(per_row), FastDiv(uint32_t(per_row)), static_cast<u2_t*>(codes) + r * per_row,
                     static_cast<uint8_t*>(scales) + r * (cols / 32));
        FRT_LAUNCHED("mx8_quantize");
    }
    return kOk;
}
template <typename T>
static int dequantize_t(const void* codes, const void* scales, int64_t rows, int cols, void* out, int64_t ldout, hipStream_t stream) {
    const int64_t per_row = cols / 8, most = launch_rows(per_row);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * per_row);
        launch_timed("mx8_dequantize", k_mx8_dequantize<T>, dim3((pieces + 255) / 256), dim3(256), 0, stream,
                     static_cast<const u2_t*>(codes) + r * per_row, static_cast<const uint8_t*>(scales) + r * (cols / 32), pieces,
                     uint32_t(per_row), FastDiv(uint32_t(per_row)), static_cast<T*>(out) + r * ldout, ldout);
        FRT_LAUNCHED("mx8_dequantize");
    }
    return kOk;
}
template <typename T>
static int swiglu_t(const void* z, int64_t ldz, int64_t rows, int ff, const int32_t* live, void* h, int64_t ldh, void* codes, void* scales,
                    hipStream_t stream) {
    const int64_t per_row = (int64_t(ff) + 7) / 8, most = launch_rows(per_row);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * per_row);
        auto go = [&](auto kernel) {
            launch_timed("moe_swiglu", kernel, dim3((pieces + 255) / 256), dim3(256), 0, stream, static_cast<const T*>(z) + r * ldz, ldz, pieces,
                         uint32_t(per_row), FastDiv(uint32_t(per_row)), ff, live, uint32_t(r), static_cast<T*>(h) + r * ldh, ldh,
                         codes ? static_cast<u2_t*>(codes) + r * 2 * per_row : nullptr, codes ? static_cast<uint8_t*>(scales) + r * (ff / 16) : nullptr);
        };
        if (codes)
            go(k_swiglu<T, true>);
        else
            go(k_swiglu<T, false>);
        FRT_LAUNCHED("moe_swiglu");
    }
    return kOk;
}
template <typename T>
static int swiglu_grad_t(const void* dh, int64_t lddh, const void* z, int64_t ldz, const void* codes, const void* scales, int64_t rows, int ff,
                         const int32_t* live, void* dz, int64_t lddz, void* h, int64_t ldh, hipStream_t stream) {
    const int64_t per_row = (int64_t(ff) + 7) / 8, most = launch_rows(per_row);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * per_row);
        auto go = [&](auto kernel) {
            launch_timed("moe_swiglu_grad", kernel, dim3((pieces + 255) / 256), dim3(256), 0, stream, static_cast<const T*>(dh) + r * lddh, lddh,
                         z ? static_cast<const T*>(z) + r * ldz : nullptr, ldz, codes ? static_cast<const u2_t*>(codes) + r * 2 * per_row : nullptr,
                         codes ? static_cast<const uint8_t*>(scales) + r * (ff / 16) : nullptr, pieces, uint32_t(per_row), FastDiv(uint32_t(per_row)),
                         ff, live, uint32_t(r), static_cast<T*>(dz) + r * lddz, lddz, h ? static_cast<T*>(h) + r * ldh : nullptr, ldh);
        };
        if (codes)
            go(k_swiglu_grad<T, true>);
        else
            go(k_swiglu_grad<T, false>);
        FRT_LAUNCHED("moe_swiglu_grad");
    }
    return kOk;
}

int mx8_quantize(int type, const void* x, int64_t ldx, int64_t rows, int cols, void* codes, void* scales, hipStream_t stream) {
    return FRT_BY_TYPE(type, quantize_t, x, ldx, rows, cols, codes, scales, stream);
}
int mx8_dequantize(int type, const void* codes, const void* scales, int64_t rows, int cols, void* out, int64_t ldout, hipStream_t stream) {
    return FRT_BY_TYPE(type, dequantize_t, codes, scales, rows, cols, out, ldout, stream);
}
int moe_swiglu(int type, const void* z, int64_t ldz, int64_t rows, int ff, const int32_t* live, void* h, int64_t ldh, void* codes,
               void* scales, hipStream_t stream) {
    return FRT_BY_TYPE(type, swiglu_t, z, ldz, rows, ff, live, h, ldh, codes, scales, stream);
}
int moe_swiglu_grad(int type, const void* dh, int64_t lddh, const void* z, int64_t ldz, const void* codes, const void* scales, int64_t rows,
                    int ff, const int32_t* live, void* dz, int64_t lddz, void* h, int64_t ldh, hipStream_t stream) {
    return FRT_BY_TYPE(type, swiglu_grad_t, dh, lddh, z, ldz, codes, scales, rows, ff, live, dz, lddz, h, ldh, stream);
}

}  // namespace frt
