// Token rows in expert order and back, with their gradients: the sort of the (token, slot) pairs by expert with its inverse
// map, and the four moves between token rows [T][n] and sorted rows [T K][n].
//
//   sort            a stable counting sort of s = t K + k by ids[s]: bounds, tok_of, slot_of and the inverse row_of
//   permute         xs[row_of[s]] = x[s / K]
//   sum             y[t] = sum_k w[t, k] ys[row_of[t, k]] (moe_unpermute; without weights, moe_permute's gradient)
//   unpermute_grad  dys[row] = w[s] dy[t] and dw[s] = sum_j dy[t, j] ys[row, j], row = row_of[s]
// A slot with an id outside [0, E) has no row (row_of = -1): it takes no part in a sum, its dw is 0. Sums are fp32 with
// the slots in ascending k; 16-bit results are rounded once, to nearest even.
#include "common.hpp"

#include <type_traits>

#include "../../include/flashrt_moe.h"

namespace frt {

// 16 bytes of a row. Rows of an odd width start at any element, so the loads and stores are vectors of the element's own
// alignment (gfx950 takes any alignment in global memory).
typedef uint32_t Raw4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t Raw2 __attribute__((ext_vector_type(4), aligned(2)));
template <typename T>
struct Piece {
    static constexpr int V = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(V)));
    typedef std::conditional_t<sizeof(T) == 4, Raw4, Raw2> Raw;
    Vec v;
};

// Elements [c, c + V) of a row of n, zeros past its end
template <typename T>
__device__ __forceinline__ Piece<T> piece_load(const T* row, int c, int n) {
    Piece<T> p;
    if (c + Piece<T>::V <= n) {
        p.v = __builtin_bit_cast(typename Piece<T>::Vec, *reinterpret_cast<const typename Piece<T>::Raw*>(row + c));
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::V; ++i) p.v[i] = c + i < n ? row[c + i] : T(0.0f);
    }
    return p;
}
template <typename T>
__device__ __forceinline__ void piece_store(T* row, int c, int n, const Piece<T>& p) {
    if (c + Piece<T>::V <= n) {
        *reinterpret_cast<typename Piece<T>::Raw*>(row + c) = __builtin_bit_cast(typename Piece<T>::Raw, p.v);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::V; ++i)
            if (c + i < n) row[c + i] = p.v[i];
    }
}

// ---------------------------------------------------------------- the sort
constexpr int kSortE = 1024;       // experts at most (a thread each)
constexpr int kSortCopies = 16;    // histogram copies, one per lane of a row of 16 (and one per wave in the ranking)
constexpr int kSortGrid = 256;     // workgroups at most

// One launch, no workspace: every workgroup counts all ids itself (those before its own slots, then all of them) in an LDS
// histogram of 16 copies, one per lane of 16, so that a popular expert's atomics do not queue up behind each other; the scan of
// the totals over the experts gives the groups' first rows, and the workgroup ranks its own slots in batches of 1024, a wave of
// 64 at a time by ballots over the id bits (stable). Integer counts: the result does not depend on the atomics' order.
__global__ void __launch_bounds__(1024) k_sort(const int32_t* __restrict__ ids, int S, int K, int E, int id_bits, int batches,
                                               int32_t* __restrict__ bounds, int32_t* __restrict__ tok_of,
                                               int32_t* __restrict__ slot_of, int32_t* __restrict__ row_of) {
    extern __shared__ int32_t hist[];   // [E][16]
    __shared__ int s_base[kSortE];      // the next row of each expert for this workgroup's slots
    __shared__ int s_wave[16];
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const int s0 = min(int64_t(S), int64_t(blockIdx.x) * batches * 1024), s1 = min(int64_t(S), int64_t(s0) + batches * 1024);
    for (int i = tid; i < E * kSortCopies; i += 1024) hist[i] = 0;
    __syncthreads();
    auto count = [&](int lo, int hi) {
        for (int s = lo + tid; s < hi; s += 1024) {
            const int e = ids[s];
            if (unsigned(e) < unsigned(E)) atomicAdd(&hist[e * kSortCopies + (lane & 15)], 1);
        }
        __syncthreads();
        int sum = 0;
        if (tid < E)
            for (int c = 0; c < kSortCopies; ++c) sum += hist[tid * kSortCopies + ((c + tid) & 15)];
        return sum;
    };
    const int before = count(0, s0);
    __syncthreads();
    const int total = count(s0, S);
    // exclusive scan of the totals over the experts
    int incl = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int y = __shfl_up(incl, o, 64);
        if (lane >= o) incl += y;
    }
    if (lane == 63) s_wave[wave] = incl;
    __syncthreads();
    int first = incl - total;
    for (int w = 0; w < wave; ++w) first += s_wave[w];
    if (tid < E) {
        s_base[tid] = first + before;
        if (blockIdx.x == 0) {
            bounds[tid] = first;
            if (tid == E - 1) bounds[E] = first + total;
        }
    }
    const uint64_t lt = (lane == 0) ? 0ull : (~0ull >> (64 - lane));
    for (int b0 = s0; b0 < s1; b0 += 1024) {   // (uniform over the workgroup)
        const int s = b0 + tid;
        __syncthreads();   // (the histogram was read; s_base is written)
        for (int i = tid; i < E * kSortCopies; i += 1024) hist[i] = 0;
        __syncthreads();
        const int e0 = s < s1 ? ids[s] : -1;
        const bool valid = unsigned(e0) < unsigned(E);
        const int e = valid ? e0 : 0;
        uint64_t peers = __ballot(valid);
        for (int bit = 0; bit < id_bits; ++bit) {
            const bool on = (e >> bit) & 1;
            const uint64_t m = __ballot(on);
            peers &= on ? m : ~m;
        }
        const int rank = __popcll(peers & lt);
        if (valid && rank == 0) hist[e * kSortCopies + wave] = __popcll(peers);
        __syncthreads();
        if (tid < E) {   // each wave's first row of expert tid
            int run = s_base[tid];
            for (int w = 0; w < 16; ++w) {
                const int c = hist[tid * kSortCopies + w];
                hist[tid * kSortCopies + w] = run;
                run += c;
            }
            s_base[tid] = run;
        }
        __syncthreads();
        if (s < s1) {
            const int row = valid ? hist[e * kSortCopies + wave] + rank : -1;
            row_of[s] = row;
            if (valid) {
                tok_of[row] = s / K;
                slot_of[row] = s;
            }
        }
    }
}

int moe_sort(const int32_t* ids, int T, int K, int E, int32_t* bounds, int32_t* tok_of, int32_t* slot_of, int32_t* row_of,
             hipStream_t stream) {
    const int S = T * K;
    int id_bits = 1;
    while ((1 << id_bits) < E) ++id_bits;
    const int nb = S > 0 ? (S + 1023) / 1024 : 1;
    const int batches = (nb + kSortGrid - 1) / kSortGrid;
    launch_timed("moe_sort", k_sort, dim3((nb + batches - 1) / batches), dim3(1024), size_t(E) * kSortCopies * 4, stream, ids, S, K, E,
                 id_bits, batches, bounds, tok_of, slot_of, row_of);
    FRT_LAUNCHED("moe_sort");
    return kOk;
}

// ---------------------------------------------------------------- the moves
// A wave takes 64 pieces of 16 bytes of one token's row (a workgroup four such parts, of consecutive tokens where a row has fewer).

// The token's piece is read once and written to each of its rows.
template <typename T>
__global__ void __launch_bounds__(256) k_permute(const T* __restrict__ x, int64_t ldx, int n_tok, int K, int n, uint32_t parts, FastDiv div,
                                                 const int32_t* __restrict__ row_of, T* __restrict__ xs, int64_t ldxs) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = int(div(unit)), c = int((unit - t * parts) * 64 + (threadIdx.x & 63)) * V;
    if (t >= n_tok || c >= n) return;
    const unsigned S = unsigned(n_tok) * K;
    const Piece<T> p = piece_load(x + t * ldx, c, n);
    for (int k = 0; k < K; ++k) {
        const int row = row_of[size_t(t) * K + k];
        if (unsigned(row) < S) piece_store(xs + row * ldxs, c, n, p);
    }
}

// The pieces of a token's rows summed in fp32, ascending k.
template <typename T, bool WTS>
__global__ void __launch_bounds__(256) k_sum_rows(const T* __restrict__ ys, int64_t ldys, int n_tok, int K, int n, uint32_t parts, FastDiv div,
                                                  const int32_t* __restrict__ row_of, const float* __restrict__ wts,
                                                  T* __restrict__ y, int64_t ldy) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = int(div(unit)), c = int((unit - t * parts) * 64 + (threadIdx.x & 63)) * V;
    if (t >= n_tok || c >= n) return;
    const unsigned S = unsigned(n_tok) * K;
    float acc[V] = {};
    for (int k = 0; k < K; ++k) {
        const int row = row_of[size_t(t) * K + k];
        if (unsigned(row) >= S) continue;
        const Piece<T> p = piece_load(ys + row * ldys, c, n);
        const float w = WTS ? wts[size_t(t) * K + k] : 1.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) acc[i] = WTS ? fmaf(w, float(p.v[i]), acc[i]) : acc[i] + float(p.v[i]);
    }
    Piece<T> o;
#pragma unroll
    for (int i = 0; i < V; ++i) o.v[i] = T(acc[i]);
    piece_store(y + t * ldy, c, n, o);
}

// A wave per slot: its row of dys, and the dot product of dy and ys, each lane's terms in ascending order and the
// lanes' sums as a pairwise tree.
template <typename T>
__global__ void __launch_bounds__(256) k_unpermute_grad(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ ys, int64_t ldys,
                                                        int n_tok, int K, int n, FastDiv div, const int32_t* __restrict__ row_of,
                                                        const float* __restrict__ wts, T* __restrict__ dys, int64_t lddys,
                                                        float* __restrict__ dwts) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t s = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const unsigned S = unsigned(n_tok) * K;
    if (s >= S) return;
    const int row = row_of[s];
    float dot = 0.0f;
    if (unsigned(row) < S) {
        const float w = wts[s];
        const T* g = dy + div(s) * lddy;
        for (int c = lane * V; c < n; c += 64 * V) {
            const Piece<T> a = piece_load(g, c, n), b = piece_load(ys + row * ldys, c, n);
            Piece<T> o;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                o.v[i] = T(w * float(a.v[i]));
                dot = fmaf(float(a.v[i]), float(b.v[i]), dot);
            }
            piece_store(dys + row * lddys, c, n, o);
        }
    }
    dot = wave_sum_tree(dot);
    if (lane == 0) dwts[s] = dot;
}

// the waves of a token's row
template <typename T>
static uint32_t row_parts(int n) { return (uint32_t(n) + 1024 / sizeof(T) - 1) / (1024 / sizeof(T)); }
// workgroups of four waves; false where the units would not fit 31 bits (rows of 2^31 KiB in all)
static bool grid_of(int64_t units, dim3* g) {
    if (units > 0x7ffffff0) return false;
    *g = dim3(uint32_t((units + 3) / 4));
    return true;
}

template <typename T>
static int permute_t(const void* x, int64_t ldx, int n_tok, int K, int n, const int32_t* row_of, void* xs, int64_t ldxs, hipStream_t stream) {
    const uint32_t parts = row_parts<T>(n);
    dim3 g;
    if (!grid_of(int64_t(n_tok) * parts, &g)) return set_error(kErrShape, "moe_permute: T=%d n=%d", n_tok, n);
    launch_timed("moe_permute", k_permute<T>, g, dim3(256), 0, stream, static_cast<const T*>(x), ldx, n_tok, K, n, parts, FastDiv(parts), row_of,
                 static_cast<T*>(xs), ldxs);
    FRT_LAUNCHED("moe_permute");
    return kOk;
}
template <typename T>
static int sum_rows_t(const void* ys, int64_t ldys, int n_tok, int K, int n, const int32_t* row_of, const float* wts, void* y, int64_t ldy,
                      hipStream_t stream) {
    const uint32_t parts = row_parts<T>(n);
    dim3 g;
    if (!grid_of(int64_t(n_tok) * parts, &g)) return set_error(kErrShape, "moe_unpermute: T=%d n=%d", n_tok, n);
    if (wts)
        launch_timed("moe_unpermute", k_sum_rows<T, true>, g, dim3(256), 0, stream, static_cast<const T*>(ys), ldys, n_tok, K, n, parts,
                     FastDiv(parts), row_of, wts, static_cast<T*>(y), ldy);
    else
        launch_timed("moe_permute_grad", k_sum_rows<T, false>, g, dim3(256), 0, stream, static_cast<const T*>(ys), ldys, n_tok, K, n, parts,
                     FastDiv(parts), row_of, wts, static_cast<T*>(y), ldy);
    FRT_LAUNCHED("moe_unpermute");
    return kOk;
}
template <typename T>
static int unpermute_grad_t(const void* dy, int64_t lddy, const void* ys, int64_t ldys, int n_tok, int K, int n, const int32_t* row_of,
                            const float* wts, void* dys, int64_t lddys, float* dwts, hipStream_t stream) {
    dim3 g;
    if (!grid_of(int64_t(n_tok) * K, &g)) return set_error(kErrShape, "moe_unpermute_grad: T=%d K=%d", n_tok, K);
    launch_timed("moe_unpermute_grad", k_unpermute_grad<T>, g, dim3(256), 0, stream, static_cast<const T*>(dy), lddy,
                 static_cast<const T*>(ys), ldys, n_tok, K, n, FastDiv(K), row_of, wts, static_cast<T*>(dys), lddys, dwts);
    FRT_LAUNCHED("moe_unpermute_grad");
    return kOk;
}

#define FRT_BY_TYPE(type, fn, ...)                                                            \
    ((type) == FRT_GGML_F32 ? fn<float>(__VA_ARGS__)                                          \
                            : (type) == FRT_GGML_F16 ? fn<_Float16>(__VA_ARGS__) : fn<__bf16>(__VA_ARGS__))
int moe_permute(int type, const void* x, int64_t ldx, int T, int K, int n, const int32_t* row_of, void* xs, int64_t ldxs,
                hipStream_t stream) {
    return FRT_BY_TYPE(type, permute_t, x, ldx, T, K, n, row_of, xs, ldxs, stream);
}
int moe_sum_rows(int type, const void* ys, int64_t ldys, int T, int K, int n, const int32_t* row_of, const float* wts, void* y,
                 int64_t ldy, hipStream_t stream) {
    return FRT_BY_TYPE(type, sum_rows_t, ys, ldys, T, K, n, row_of, wts, y, ldy, stream);
}
int moe_unpermute_grad(int type, const void* dy, int64_t lddy, const void* ys, int64_t ldys, int T, int K, int n, const int32_t* row_of,
                       const float* wts, void* dys, int64_t lddys, float* dwts, hipStream_t stream) {
    return FRT_BY_TYPE(type, unpermute_grad_t, dy, lddy, ys, ldys, T, K, n, row_of, wts, dys, lddys, dwts, stream);
}

}  // namespace frt
