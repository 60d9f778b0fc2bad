// Tiles of the rows of groups (the sorted rows of the experts), found by a wave from the groups' bounds.
#pragma once

#include "common.hpp"

namespace frt {

// A tile of a group's rows
struct RowTile {
    int g, row0, rows;   // rows 0: no such tile
    bool only;           // the group's only one
};

// The tile that which(number of tiles) names, of the groups' rows cut into tiles of BM, found by one wave from bounds (no list in
// memory): each lane counts the tiles of 8 neighbouring groups, whose loads are in flight together (one trip to memory for up to
// 512 groups), a scan over the lanes finds the lane, and that lane its group. Rows are clamped to [0, M), so that no bounds lead
// outside the operands.
template <int BM, typename Which>
__device__ __forceinline__ RowTile find_tile(const int32_t* __restrict__ bounds, int E, int M, Which which) {
    if (!bounds) {
        const int index = which((M + BM - 1) / BM);
        return {0, index * BM, index < 0 ? 0 : max(0, min(BM, M - index * BM)), M <= BM};
    }
    const int lane = threadIdx.x & 63;
    int at[9], n = 0, incl = 0, total = 0;
    auto block = [&](int e0) {   // groups e0 + 8 lane ..: their first rows, their tiles, and the tiles up to the lane
#pragma unroll
        for (int i = 0; i < 9; ++i) at[i] = gld<int>(bounds + min(e0 + 8 * lane + i, E));
        n = 0;
#pragma unroll
        for (int i = 0; i < 9; ++i) at[i] = min(max(at[i], 0), M);
#pragma unroll
        for (int i = 0; i < 8; ++i) n += max(0, at[i + 1] - at[i] + BM - 1) / BM;
        incl = wave_scan(n);
    };
    for (int e0 = 0; e0 < E; e0 += 512) {
        block(e0);
        total += __builtin_amdgcn_readlane(incl, 63);
    }
    int index = which(total), e0 = 0;
    if (index < 0 || index >= total) return {0, 0, 0, false};
    if (E > 512) {   // (the last block is in the registers: from the first one again)
        for (; e0 < E; e0 += 512) {
            block(e0);
            const int here = __builtin_amdgcn_readlane(incl, 63);
            if (index < here) break;
            index -= here;
        }
        if (e0 >= E) return {0, 0, 0, false};
    }
    const int owner = __builtin_ctzll(__ballot(incl > index));
    int left = index - (incl - n), g = 0, row0 = 0, rows = 0, of = 0;   // (of use in that lane)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = max(0, at[i + 1] - at[i] + BM - 1) / BM;
        if (left >= 0 && left < c) {
            g = e0 + 8 * lane + i;
            row0 = at[i] + left * BM;
            rows = min(BM, at[i + 1] - row0);
            of = c;
        }
        left -= c;
    }
    return {__builtin_amdgcn_readlane(g, owner), __builtin_amdgcn_readlane(row0, owner), __builtin_amdgcn_readlane(rows, owner),
            __builtin_amdgcn_readlane(of, owner) == 1};
}
// The group of rank r by size, largest first (equal ones in any fixed order), of up to 512 groups, by one wave: the rank's size bit by bit, each bit by
// counting the groups that have at least that many rows.
__device__ __forceinline__ int group_by_size(const int32_t* __restrict__ bounds, int E, int M, int rank) {
    const int lane = threadIdx.x & 63;
    int at[9], rows[8];
#pragma unroll
    for (int i = 0; i < 9; ++i) at[i] = gld<int>(bounds + min(8 * lane + i, E));
#pragma unroll
    for (int i = 0; i < 9; ++i) at[i] = min(max(at[i], 0), M);
#pragma unroll
    for (int i = 0; i < 8; ++i) rows[i] = 8 * lane + i < E ? max(0, at[i + 1] - at[i]) : -1;
    auto count = [&](int least) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) n += __popcll(__ballot(rows[i] >= least));
        return n;
    };
    int size = 0;
    for (int bit = 31 - __builtin_clz(M | 1); bit >= 0; --bit)
        if (count(size | 1 << bit) > rank) size |= 1 << bit;
    int left = rank - count(size + 1);   // of the groups of that size
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        uint64_t same = __ballot(rows[i] == size);
        const int n = __popcll(same);
        if (left < n) {
            for (; left > 0; --left) same &= same - 1;
            return 8 * __builtin_ctzll(same) + i;
        }
        left -= n;
    }
    return 0;   // (rank is below E)
}
// Tiles of BM rows that M rows in E groups have at most
inline int64_t tiles_at_most(int64_t M, int64_t E, int BM, bool grouped) {
    const int64_t g = grouped ? (E < M ? E : M) : (M > 0 ? 1 : 0);   // groups with rows
    return (M - g) / BM + g;
}

}  // namespace frt
