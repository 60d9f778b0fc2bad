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

// The piece of a row of n that begins at c < n. A row's last piece is moved back to end with the row (two lanes then hold, and
// store, the same values); a row shorter than a piece is taken by elements, zeros past its end.
template <typename T>
__device__ __forceinline__ int piece_at(int c, int n) { return max(0, min(c, n - Piece<T>::V)); }
template <typename T>
__device__ __forceinline__ Piece<T> piece_load(const T* row, int c, int n) {
    Piece<T> p;
    if (n >= Piece<T>::V) {
        p.v = __builtin_bit_cast(typename Piece<T>::Vec, *reinterpret_cast<const typename Piece<T>::Raw*>(row + piece_at<T>(c, n)));
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::V; ++i) p.v[i] = i < n ? row[i] : T(0.0f);
    }
    return p;
}
template <typename T>
__device__ __forceinline__ void piece_store(T* row, int c, int n, const Piece<T>& p) {
    if (n >= Piece<T>::V) {
        *reinterpret_cast<typename Piece<T>::Raw*>(row + piece_at<T>(c, n)) = __builtin_bit_cast(typename Piece<T>::Raw, p.v);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T>::V; ++i)
            if (i < n) row[i] = p.v[i];
    }
}

// ---------------------------------------------------------------- the sort
constexpr int kSortE = 1024;       // experts at most (a thread each)
constexpr int kSortCopies = 16;    // histogram copies, one per lane of a row of 16 (and one per wave in the ranking)
constexpr int kSortGrid = 256;     // workgroups at most

// Up to 64 slots (a decode step): every wave has all ids, one per lane. A group's first row is the number of ids below it, a slot's
// row the number of ids that sort before it: no histogram, scan or barrier. One token's 10 slots, launches back to back, 2.4 us (8.2 with
// the kernel below).
__global__ void __launch_bounds__(1024) k_sort_few(const int32_t* __restrict__ ids, int S, int K, int E, int32_t* __restrict__ bounds,
                                                   int32_t* __restrict__ tok_of, int32_t* __restrict__ slot_of,
                                                   int32_t* __restrict__ row_of) {
    const int tid = threadIdx.x, lane = tid & 63;
    int id = lane < S ? ids[lane] : -1;
    if (unsigned(id) >= unsigned(E)) id = 0x7fffffff;
    int below = 0, row = 0;
    for (int s = 0; s < S; ++s) {
        const int e = __builtin_amdgcn_readlane(id, s);
        below += e < tid;
        row += e < id || (e == id && s < lane);
    }
    const int live = __popcll(__ballot(id < E));
    if (tid < E) bounds[tid] = below;
    if (tid == 0) bounds[E] = live;
    if (tid < S) {
        const bool valid = id < E;
        row_of[tid] = valid ? row : -1;
        if (valid) {
            tok_of[row] = tid / K;
            slot_of[row] = tid;
        }
    }
}

// One launch, no workspace: every workgroup counts all ids itself, in two LDS histograms (the slots before its own, and the
// others) of 16 copies, one per lane of 16, so that a popular expert's atomics do not queue up behind each other; the scan of
// the totals over the experts gives the groups' first rows, and the workgroup ranks its own slots in batches of 1024, a wave of
// 64 at a time by ballots over the id bits (stable). Integer counts: the result does not depend on the atomics' order. The
// counting reads 16 ids per thread at once and spends three instructions on an id: ids outside are counted in a bin of their own,
// and the histogram is the wave's choice (81920 slots of 512 experts, launches back to back, 11.8 us, of which 4.9 are the LDS atomics,
// about 8 clocks per 64 ids; with two passes and a branch per id 13.7, reading one by one 22.4; a launch alone in a trace takes 13.2).
// One launch instead of the dispatch's four costs each workgroup the whole list, 328 KB from L2 at 81920 slots, so the time grows
// with the list, bound by the atomics; the dispatch stays behind it (us, this and the dispatch: 2048 slots 7.4 / 10.3, 20480 9.0 / 19.2,
// 81920 11.5 / 25.3, 2^18 21 / 44, 2^20 61 / 139, 2^23 430 / 966, 2^26 3863 / 10898).
// ONE: a single batch, whose ranking counts it.
template <bool ONE>
__global__ void __launch_bounds__(1024) k_sort(const int32_t* __restrict__ ids, int S, int K, int E, int id_bits, int batches,
                                               int32_t* __restrict__ bounds, int32_t* __restrict__ tok_of,
                                               int32_t* __restrict__ slot_of, int32_t* __restrict__ row_of) {
    // [E + 1][16], the last for ids outside; twice unless ONE: of the slots before the workgroup's own, and of the others
    extern __shared__ int32_t hist[];
    __shared__ int s_base[kSortE];      // the next row of each expert for this workgroup's slots
    __shared__ int s_wave[16];
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
    const int s0 = min(int64_t(S), int64_t(blockIdx.x) * batches * 1024), s1 = min(int64_t(S), int64_t(s0) + batches * 1024);
    auto clear = [&](int n) {
        for (int i = tid; i < n; i += 1024) hist[i] = 0;
        __syncthreads();
    };
    const int one = (E + 1) * kSortCopies;   // a histogram
    auto sum = [&](const int32_t* h) {       // of expert tid's copies
        int n = 0;
        if (tid < E)
#pragma unroll
            for (int c = 0; c < kSortCopies; ++c) n += h[tid * kSortCopies + ((c + tid) & 15)];
        return n;
    };
    auto count = [&]() {   // all ids
        // a wave's ids are all before s0, a multiple of 1024, or none
        auto add = [&](uint32_t e, int32_t* h) { atomicAdd(h + min(e, uint32_t(E)) * kSortCopies, 1); };
        int32_t* const mine = hist + (lane & 15);
        int64_t s = 0;   // (past 2^31 after the last step of a list near that length)
        for (; s + 16384 <= S; s += 16384) {
            Raw4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const Raw4*>(ids + s + (i * 1024 + tid) * 4);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int32_t* const h = mine + (s + (i * 1024 + wave * 64) * 4 < s0 ? 0 : one);
#pragma unroll
                for (int k = 0; k < 4; ++k) add(v[i][k], h);
            }
        }
        uint32_t v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = s + i * 1024 + tid < S ? ids[s + i * 1024 + tid] : -1;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (s + i * 1024 < S) add(v[i], mine + (s + i * 1024 < s0 ? 0 : one));
        __syncthreads();
    };
    // the first row of expert tid's group, from its rows
    auto starts = [&](int total) {
        const int incl = wave_scan(total);
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        int first = incl - total;
        for (int w = 0; w < wave; ++w) first += s_wave[w];
        if (tid < E && blockIdx.x == 0) {
            bounds[tid] = first;
            if (tid == E - 1) bounds[E] = first + total;
        }
        return first;
    };
    clear(ONE ? one : 2 * one);
    if (!ONE) {
        count();
        const int before = sum(hist), first = starts(before + sum(hist + one));
        if (tid < E) s_base[tid] = first + before;
        clear(one);   // (read before the barrier in starts)
    }
    const uint64_t lt = (lane == 0) ? 0ull : (~0ull >> (64 - lane));
    for (int64_t b0 = s0; b0 < s1; b0 += 1024) {   // (uniform over the workgroup)
        const int64_t s = b0 + tid;
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
        auto at = [&](int ex, int w) { return ex * kSortCopies + ((w + ex) & 15); };   // (turned by the expert: other banks)
        if (valid && rank == 0) hist[at(e, wave)] = __popcll(peers);
        __syncthreads();
        int run = 0;
        if (ONE)
            run = starts(sum(hist));
        else if (tid < E)
            run = s_base[tid];
        if (tid < E) {   // each wave's first row of expert tid
#pragma unroll
            for (int w = 0; w < 16; ++w) {
                const int c = hist[at(tid, w)];
                hist[at(tid, w)] = run;
                run += c;
            }
            if (!ONE) s_base[tid] = run;
        }
        __syncthreads();
        if (s < s1) {
            const int row = valid ? hist[at(e, wave)] + rank : -1;
            row_of[s] = row;
            if (valid) {
                tok_of[row] = int(s) / K;
                slot_of[row] = int(s);
            }
        }
        if (b0 + 1024 < s1) {
            __syncthreads();
            clear(one);
        }
    }
}

int moe_sort(const int32_t* ids, int T, int K, int E, int32_t* bounds, int32_t* tok_of, int32_t* slot_of, int32_t* row_of,
             hipStream_t stream) {
    const int S = T * K;
    if (S <= 64) {
        launch_timed("moe_sort", k_sort_few, dim3(1), dim3(1024), 0, stream, ids, S, K, E, bounds, tok_of, slot_of, row_of);
        FRT_LAUNCHED("moe_sort");
        return kOk;
    }
    int id_bits = 1;
    while ((1 << id_bits) < E) ++id_bits;
    const int nb = int((int64_t(S) + 1023) / 1024);
    const int batches = (nb + kSortGrid - 1) / kSortGrid;
    const size_t lds = size_t(E + 1) * kSortCopies * (nb == 1 ? 4 : 8);
    const auto kernel = nb == 1 ? k_sort<true> : k_sort<false>;
    if (lds + 8192 > 65536)
        FRT_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, int(lds)));
    launch_timed("moe_sort", kernel, dim3((nb + batches - 1) / batches), dim3(1024),
                 lds, stream, ids, S, K, E, id_bits, batches, bounds, tok_of, slot_of, row_of);
    FRT_LAUNCHED("moe_sort");
    return kOk;
}

// ---------------------------------------------------------------- the moves
// A wave takes 64 pieces of 16 bytes of one token's row (a workgroup four such parts, of consecutive tokens where a row has fewer).
// All four are bound by HBM: 8192 tokens of 2560 bf16 values and their 81920 sorted rows 92 us to permute (5.0 TB/s; a large copy
// reaches 4.8 to 5.1), 91 us to sum, 179 us for the weighted sum's gradient (4.9); short calls by one trip to memory and the
// launch (one token of ten slots 2.8 to 3.8 us).

// The token's piece is read once and written to each of its rows.
template <typename T>
__global__ void __launch_bounds__(256) k_permute(const T* __restrict__ x, int64_t ldx, int n_tok, int K, int n, uint32_t parts, FastDiv div,
                                                 const int32_t* __restrict__ row_of, T* __restrict__ xs, int64_t ldxs) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t unit = wide_block() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = int(div(unit)), c = int((unit - t * parts) * 64 + (threadIdx.x & 63)) * V;
    if (t >= n_tok || c >= n) return;
    const unsigned S = unsigned(n_tok) * K;
    const Piece<T> p = piece_load(x + t * ldx, c, n);
    for (int k = 0; k < K; ++k) {
        const int row = row_of[size_t(t) * K + k];
        if (unsigned(row) < S) piece_store(xs + row * ldxs, c, n, p);
    }
}

// The pieces of a token's rows summed in fp32, ascending k; four rows' loads are in flight together.
template <typename T, bool WTS>
__global__ void __launch_bounds__(256) k_sum_rows(const T* __restrict__ ys, int64_t ldys, int n_tok, int K, int n, uint32_t parts, FastDiv div,
                                                  const int32_t* __restrict__ row_of, const float* __restrict__ wts,
                                                  T* __restrict__ y, int64_t ldy) {
    constexpr int V = 16 / sizeof(T);
    const uint32_t unit = wide_block() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = int(div(unit)), c = int((unit - t * parts) * 64 + (threadIdx.x & 63)) * V;
    if (t >= n_tok || c >= n) return;
    const unsigned S = unsigned(n_tok) * K;
    const size_t s0 = size_t(t) * K;
    float acc[V] = {};
    const uint32_t slots = K;   // (k0 passes 2^31 after the last step where K is near it)
    for (uint32_t k0 = 0; k0 < slots; k0 += 4) {
        int row[4];
        Piece<T> p[4];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) row[k] = row_of[s0 + min(k0 + k, slots - 1)];
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (k0 + k < slots && unsigned(row[k]) < S) p[k] = piece_load(ys + row[k] * ldys, c, n);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (k0 + k < slots && unsigned(row[k]) < S) {
                const float w = WTS ? wts[s0 + k0 + k] : 1.0f;
#pragma unroll
                for (int i = 0; i < V; ++i) acc[i] = WTS ? fmaf(w, float(p[k].v[i]), acc[i]) : acc[i] + float(p[k].v[i]);
            }
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
    const uint32_t s = wide_block() * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const unsigned S = unsigned(n_tok) * K;
    if (s >= S) return;
    const int row = row_of[s];
    float dot = 0.0f;
    if (unsigned(row) < S) {
        const float w = wts[s];
        const T* g = dy + div(s) * lddy;
        const T* y = ys + row * ldys;
        T* const d = dys + row * lddys;
        for (int c0 = lane * V; c0 < n; c0 += 2 * 64 * V) {   // two pieces of both in flight
            const int c1 = c0 + 64 * V;
            const bool two = c1 < n;
            Piece<T> a[2], b[2];
            a[0] = piece_load(g, c0, n);
            b[0] = piece_load(y, c0, n);
            if (two) {
                a[1] = piece_load(g, c1, n);
                b[1] = piece_load(y, c1, n);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (k == 1 && !two) break;
                const int c = k ? c1 : c0, again = c - piece_at<T>(c, n);   // the first `again` are the lane's before, too
                Piece<T> o;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    o.v[i] = T(w * float(a[k].v[i]));
                    dot = i >= again ? fmaf(float(a[k].v[i]), float(b[k].v[i]), dot) : dot;
                }
                piece_store(d, c, n, o);
            }
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
    if (units > 0x7fffffff) return false;
    *g = wide_grid(uint32_t((units + 3) / 4));
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
