// gk_group.cuh -- ragged groups on the device: the offsets of a grouped product made safe, and
// the tile schedule that every role of a persistent kernel walks.
//
// A grouped call splits `rows` rows into groups by a device array off[0 .. groups]: group g is
// the rows off[g] <= i < off[g + 1]. The host never reads it. Whatever the array holds, the
// kernels use its running maximum clamped to [0, rows], so no group reaches outside the buffers
// and no row belongs to two groups; an array that had to be changed sets GK_DEV_BAD_OFFSETS in
// the device status word.
#pragma once

#include <stdint.h>

#include "gk_sm100.cuh"

namespace gk {

constexpr int MAX_GROUPS = 1024;

// Shared-memory tables of a grouped kernel (int each): off[groups + 1], tile0[groups + 1].
constexpr int GROUP_TABLE_INTS = MAX_GROUPS + 1;

// The sanitised offsets into shared memory `off`, and into `acc` the running sums of
// f(rows of the group) (acc[0] = 0). All threads of the block call it (two block barriers
// inside); offsets == nullptr means `groups` equal groups of rows / groups rows.
template <typename F>
__device__ __forceinline__ void load_groups(const int32_t* offsets, int groups, int rows, int* off,
                                            int* acc, unsigned int* status, F f) {
    if (offsets) {
        for (int i = threadIdx.x; i <= groups; i += blockDim.x) off[i] = offsets[i];
    } else {
        const int per = rows / groups;
        for (int i = threadIdx.x; i <= groups; i += blockDim.x) off[i] = i * per;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        int carry = 0, sum = 0;  // the maximum so far, and the sum over the groups so far
        bool bad = false;
        for (int base = 0; base <= groups; base += 32) {
            const int i = base + lane;
            const int raw = i <= groups ? off[i] : 0;
            int v = min(max(raw, 0), rows);
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, v, d);
                if (lane >= d) v = max(v, u);
            }
            v = max(v, carry);
            if (i <= groups && v != raw) bad = true;
            int prev = __shfl_up_sync(0xffffffffu, v, 1);
            if (lane == 0) prev = carry;
            // group i - 1 ends at v; its share is added to acc[i]
            int s = (i >= 1 && i <= groups) ? f(v - prev) : 0;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, s, d);
                if (lane >= d) s += u;
            }
            s += sum;
            if (i <= groups) {
                off[i] = v;
                acc[i] = s;
            }
            carry = __shfl_sync(0xffffffffu, v, 31);
            sum = __shfl_sync(0xffffffffu, s, 31);
        }
        if (__any_sync(0xffffffffu, bad) && lane == 0 && status) atomicOr(status, GK_DEV_BAD_OFFSETS);
    }
    __syncthreads();
}

// Running sums of f(rows of the group) over sanitised offsets, by one warp: acc[0 .. groups].
template <typename F>
__device__ __forceinline__ void sum_groups(const int* off, int groups, int* acc, F f) {
    const int lane = threadIdx.x & 31;
    int sum = 0;
    for (int base = 0; base < groups; base += 32) {
        const int i = base + lane;
        int s = i < groups ? f(off[i + 1] - off[i]) : 0;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int u = __shfl_up_sync(0xffffffffu, s, d);
            if (lane >= d) s += u;
        }
        s += sum;
        if (i < groups) acc[i + 1] = s;
        sum = __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) acc[0] = 0;
}

// Walks one block's tiles t = first, first + step, ... of a group schedule. Inside a group the
// tiles run in bands of BAND tiles of the q side, q fastest: the blocks that work at one time
// share the p operand's tiles, and the band's q operand stays in L2.
struct GroupWalk {
    static constexpr int BAND = 16;
    const int* off;
    const int* tile0;
    int g, t, total, step;

    __device__ __forceinline__ GroupWalk(const int* off_, const int* tile0_, int groups, int first,
                                         int step_)
        : off(off_), tile0(tile0_), g(0), t(first - step_), total(tile0_[groups]), step(step_) {}

    // The next tile: its group and its tile indices on the two sides (tiles_p tiles on the p
    // side; the group has tiles / tiles_p tiles on the q side).
    __device__ __forceinline__ bool next(int tiles_p, int& tp, int& tq) {
        t += step;
        if (t >= total) return false;
        locate(t, tiles_p, tp, tq);
        return true;
    }

    // The group and the indices of tile i; i does not fall from call to call.
    __device__ __forceinline__ void locate(int i, int tiles_p, int& tp, int& tq) {
        while (i >= tile0[g + 1]) ++g;
        const int r = i - tile0[g];
        const int nq = (tile0[g + 1] - tile0[g]) / tiles_p;
        const int band = r / (BAND * tiles_p);
        const int rr = r - band * BAND * tiles_p;
        const int h = min(BAND, nq - band * BAND);
        tp = rr / h;
        tq = band * BAND + rr - tp * h;
    }
};

}  // namespace gk
