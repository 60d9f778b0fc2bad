// Microscaled 4-bit floats: quantisation, and the grouped product of 4-bit operands on the matrix cores.
//
// Format: each 32 consecutive values of a row share one scale byte b, the power of two 2^(b - 127) (255: NaN), and are e2m1 codes
// (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6). Codes [rows][cols / 2], value 2 j in the low half of
// byte j; scales [rows][cols / 32]. This is the operand format of gfx950's scaled matrix instructions: a lane takes one block
// of 32 codes as 16 bytes and its scale as one byte.
#include "common.hpp"

#include "../../include/flashrt_moe.h"

namespace frt {

typedef uint32_t u4e4_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u4e2_t __attribute__((ext_vector_type(4), aligned(2)));
typedef float f4_t __attribute__((ext_vector_type(4)));
typedef float f8_t __attribute__((ext_vector_type(8)));
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef int i8_t __attribute__((ext_vector_type(8)));

// Eight values of a row as fp32, loaded at the element's own alignment
__device__ __forceinline__ f8_t load8(const float* p) {
    const u4e4_t a = *reinterpret_cast<const u4e4_t*>(p), b = *reinterpret_cast<const u4e4_t*>(p + 4);
    const f4_t x = __builtin_bit_cast(f4_t, a), y = __builtin_bit_cast(f4_t, b);
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

// The fp32 value of a scale byte (0: the subnormal 2^-127)
__device__ __forceinline__ float scale_value(uint32_t b) {
    return __builtin_bit_cast(float, b == 255u ? 0x7fc00000u : b ? b << 23 : 0x00400000u);
}

// ---------------------------------------------------------------- quantisation
// Four lanes to a block, eight values each. With amax = m 2^k (1 <= m < 2) the scale is 2^(k - 2), so the largest code's
// exponent is amax's; its byte k + 125 is the exponent field of amax less 2, at least 0 (2^-127, all smaller blocks). A value's
// code is x 2^-(k - 2), an exact product, rounded to nearest even by the conversion instruction, at most 6. A block with
// an infinity or a NaN (the exponent field 255 in the largest absolute bits) gets the NaN scale and zero codes.
template <typename T>
__global__ void __launch_bounds__(256) k_mx4_quantize(const T* __restrict__ x, int64_t ldx, uint32_t pieces, uint32_t per_row, FastDiv div,
                                                      uint32_t* __restrict__ codes, uint8_t* __restrict__ scales) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;   // (pieces is a multiple of 4: whole quads stay or go)
    if (i >= pieces) return;
    const uint32_t r = div(i);
    const f8_t v = load8(x + r * ldx + (i - r * per_row) * 8);
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float f = v[j];   // (a bit cast of a vector's element by itself takes the first one)
        top = max(top, __builtin_bit_cast(uint32_t, f) & 0x7fffffffu);
    }
    top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), kDppXor1, 0xF, 0xF, true)));
    top = max(top, uint32_t(__builtin_amdgcn_mov_dpp(int(top), kDppXor2, 0xF, 0xF, true)));
    const bool bad = top >= 0x7f800000u;
    const uint32_t b = bad ? 255u : uint32_t(max(int(top >> 23) - 2, 0));
    const float inv = __builtin_bit_cast(float, (254u - min(b, 252u)) << 23);   // 2^(127 - b)
    uint32_t q = 0;
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0] * inv, v[1] * inv, 1.0f, 0);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2] * inv, v[3] * inv, 1.0f, 1);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4] * inv, v[5] * inv, 1.0f, 2);
    q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6] * inv, v[7] * inv, 1.0f, 3);
    codes[i] = bad ? 0u : q;
    if ((i & 3) == 0) scales[i >> 2] = uint8_t(b);
}

template <typename T>
__global__ void __launch_bounds__(256) k_mx4_dequantize(const uint32_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                        uint32_t pieces, uint32_t per_row, FastDiv div, T* __restrict__ out, int64_t ldout) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= pieces) return;
    const uint32_t r = div(i);
    const uint32_t q = codes[i];
    const float s = scale_value(scales[i >> 2]);
    f8_t v;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t c = q >> (4 * j), m = c & 7u;
        // the e2m1 magnitude: 0, 0.5, then (1 + (m & 1) / 2) 2^(m / 2 - 1)
        const uint32_t bits = m < 2u ? (m ? 0x3f000000u : 0u) : ((m >> 1) + 126u) << 23 | (m & 1u) << 22;
        v[j] = __builtin_bit_cast(float, bits | (c & 8u) << 28) * s;
    }
    store8(out + r * ldout + (i - r * per_row) * 8, v);
}

// Rows of one launch: fewer than 2^31 pieces of 8 values
static int64_t launch_rows(int cols) { return (int64_t(0x7fffff00) / (cols / 8)) > 0 ? int64_t(0x7fffff00) / (cols / 8) : 1; }

template <typename T>
static int quantize_t(const void* x, int64_t ldx, int64_t rows, int cols, void* codes, void* scales, hipStream_t stream) {
    const int64_t most = launch_rows(cols);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * (cols / 8));
        launch_timed("mx4_quantize", k_mx4_quantize<T>, dim3((pieces + 255) / 256), dim3(256), 0, stream, static_cast<const T*>(x) + r * ldx,
                     ldx, pieces, uint32_t(cols / 8), FastDiv(cols / 8), static_cast<uint32_t*>(codes) + r * (cols / 8),
                     static_cast<uint8_t*>(scales) + r * (cols / 32));
        FRT_LAUNCHED("mx4_quantize");
    }
    return kOk;
}
template <typename T>
static int dequantize_t(const void* codes, const void* scales, int64_t rows, int cols, void* out, int64_t ldout, hipStream_t stream) {
    const int64_t most = launch_rows(cols);
    for (int64_t r = 0; r < rows; r += most) {
        const uint32_t pieces = uint32_t((rows - r < most ? rows - r : most) * (cols / 8));
        launch_timed("mx4_dequantize", k_mx4_dequantize<T>, dim3((pieces + 255) / 256), dim3(256), 0, stream,
                     static_cast<const uint32_t*>(codes) + r * (cols / 8), static_cast<const uint8_t*>(scales) + r * (cols / 32), pieces,
                     uint32_t(cols / 8), FastDiv(cols / 8), static_cast<T*>(out) + r * ldout, ldout);
        FRT_LAUNCHED("mx4_dequantize");
    }
    return kOk;
}

// ---------------------------------------------------------------- the grouped product
// A tile of a group's rows
struct RowTile {
    int g, row0, rows;   // rows 0: no such tile
};

// Tile `index` of the groups' rows cut into tiles of BM, found by one wave from bounds (no list in memory): each lane counts the
// tiles of its share of the groups, a scan over the lanes finds the lane, and that lane its group. Rows are clamped to
// [0, M), so that no bounds lead outside the operands.
template <int BM>
__device__ __forceinline__ RowTile find_tile(const int32_t* __restrict__ bounds, int E, int M, int index) {
    if (!bounds) return {0, index * BM, max(0, min(BM, M - index * BM))};
    const int lane = threadIdx.x & 63;
    const int per = (E + 63) / 64, e0 = min(lane * per, E), e1 = min(e0 + per, E);
    auto at = [&](int e) { return min(max(bounds[e], 0), M); };
    int n = 0;
    for (int e = e0; e < e1; ++e) n += max(0, at(e + 1) - at(e) + BM - 1) / BM;
    int incl = n;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o, 64);
        if (lane >= o) incl += y;
    }
    const uint64_t past = __ballot(incl > index);
    if (!past) return {0, 0, 0};
    const int owner = __builtin_ctzll(past);
    RowTile t{0, 0, 0};
    int left = index - (incl - n);
    if (lane == owner)
        for (int e = e0; e < e1; ++e) {
            const int lo = at(e), hi = at(e + 1), c = max(0, hi - lo + BM - 1) / BM;
            if (left < c) {
                t = {e, lo + left * BM, min(BM, hi - lo - left * BM)};
                break;
            }
            left -= c;
        }
    t.g = __builtin_amdgcn_readlane(t.g, owner);
    t.row0 = __builtin_amdgcn_readlane(t.row0, owner);
    t.rows = __builtin_amdgcn_readlane(t.rows, owner);
    return t;
}
// Tiles of BM rows that M rows in E groups have at most
static int64_t tiles_at_most(int64_t M, int64_t E, int BM, bool grouped) {
    const int64_t g = grouped ? (E < M ? E : M) : (M > 0 ? 1 : 0);   // groups with rows
    return (M - g) / BM + g;
}

struct Mx4Args {
    const uint8_t* aq;
    const uint8_t* as;
    int a_rows;
    const int32_t* rows;
    const uint8_t* wq;
    const uint8_t* ws;
    const int32_t* bounds;
    int E, M, N, C;
    void* out;
    int64_t ldout;
};

// A wave per 16 features x 16 rows: the weights as the A operand, so a lane's four results are consecutive features of one
// row. Lane l holds block 4 s + l / 16 of its feature and of its row in step s.
template <typename T>
__global__ void __launch_bounds__(256) k_mx4_rows(Mx4Args p, int ntile) {
    const int64_t unit = int64_t(blockIdx.x) * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63, j = lane & 15, g = lane >> 4;
    const RowTile t = find_tile<16>(p.bounds, p.E, p.M, int(unit / ntile));
    if (t.rows == 0) return;
    const int f0 = int(unit % ntile) * 16, nb = p.C / 32;
    int64_t a = -1;
    if (j < t.rows) {
        a = p.rows ? p.rows[t.row0 + j] : t.row0 + j;
        if (a < 0 || a >= p.a_rows) a = -1;
    }
    const bool fok = f0 + j < p.N;
    const int64_t w = (int64_t(t.g) * p.N + (fok ? f0 + j : 0)) * nb, x = (a < 0 ? 0 : a) * nb;
    f4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int b = 0; b < nb; b += 4) {
        i4_t wv = {0, 0, 0, 0}, xv = {0, 0, 0, 0};
        int wsc = 127, xsc = 127;
        if (b + g < nb) {
            if (fok) {
                wv = __builtin_bit_cast(i4_t, gld_u4(p.wq + (w + b + g) * 16));
                wsc = gld<uint8_t>(p.ws + w + b + g);
            }
            if (a >= 0) {
                xv = __builtin_bit_cast(i4_t, gld_u4(p.aq + (x + b + g) * 16));
                xsc = gld<uint8_t>(p.as + x + b + g);
            }
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(__builtin_shufflevector(wv, wv, 0, 1, 2, 3, -1, -1, -1, -1),
                                                               __builtin_shufflevector(xv, xv, 0, 1, 2, 3, -1, -1, -1, -1), acc, 4, 4, 0,
                                                               wsc, 0, xsc);
    }
    if (j < t.rows) {
        T* o = static_cast<T*>(p.out) + (t.row0 + j) * p.ldout + f0 + 4 * g;
        for (int i = 0; i < 4; ++i)
            if (f0 + 4 * g + i < p.N) o[i] = T(acc[i]);
    }
}

template <typename T>
static int product_t(const Mx4Args& p, hipStream_t stream) {
    const int ntile = (p.N + 15) / 16;
    const int64_t units = tiles_at_most(p.M, p.E, 16, p.bounds != nullptr) * ntile, wgs = (units + 3) / 4;
    if (wgs > 0x7fffffff) return set_error(kErrShape, "mx4_product: M=%d N=%d E=%d", p.M, p.N, p.E);
    launch_timed("mx4_product", k_mx4_rows<T>, dim3(uint32_t(wgs)), dim3(256), 0, stream, p, ntile);
    FRT_LAUNCHED("mx4_product");
    return kOk;
}

#define FRT_BY_TYPE(type, fn, ...)                                                            \
    ((type) == FRT_GGML_F32 ? fn<float>(__VA_ARGS__)                                          \
                            : (type) == FRT_GGML_F16 ? fn<_Float16>(__VA_ARGS__) : fn<__bf16>(__VA_ARGS__))
int mx4_quantize(int type, const void* x, int64_t ldx, int64_t rows, int cols, void* codes, void* scales, hipStream_t stream) {
    return FRT_BY_TYPE(type, quantize_t, x, ldx, rows, cols, codes, scales, stream);
}
int mx4_dequantize(int type, const void* codes, const void* scales, int64_t rows, int cols, void* out, int64_t ldout,
                   hipStream_t stream) {
    return FRT_BY_TYPE(type, dequantize_t, codes, scales, rows, cols, out, ldout, stream);
}
int mx4_product(const void* aq, const void* as, int a_rows, const int32_t* rows, const void* wq, const void* ws, const int32_t* bounds,
                int E, int M, int N, int C, void* out, int type, int64_t ldout, hipStream_t stream) {
    const Mx4Args p{static_cast<const uint8_t*>(aq), static_cast<const uint8_t*>(as), a_rows, rows, static_cast<const uint8_t*>(wq),
                    static_cast<const uint8_t*>(ws), bounds, E, M, N, C, out, ldout};
    return FRT_BY_TYPE(type, product_t, p, stream);
}

}  // namespace frt
