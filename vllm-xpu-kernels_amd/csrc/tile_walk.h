// The tiles that the workgroups of a launch take, in order (plain C++: a test follows them on the host).
#pragma once

namespace mi355 {

// Every step-th tile of [t, end).  Workgroups are dealt round-robin to the 8 XCDs: XCD i takes a
// contiguous range of tiles, in bands of 4 tiles of q, so that the tiles that run together on an
// XCD share rows of both operands in its L2.
struct XcdWalk {
  int t, end, step;
  __host__ __device__ __forceinline__ XcdWalk(int total, int block, int blocks) {
    const int per = (total + 7) / 8;
    const int xcd = block & 7;
    step = blocks >> 3;
    end = (xcd + 1) * per < total ? (xcd + 1) * per : total;
    t = xcd * per + (block >> 3);
  }
  __host__ __device__ __forceinline__ bool more() const { return t + step < end; }
  __host__ __device__ __forceinline__ void next() { t += step; }
};

// The tiles of the second of two products in one launch, behind the workgroup's XcdWalk over the
// first.  The workgroups of an XCD that get one tile of the first less than the others (`light`,
// its last ones) take `extra` (1 at least) tiles of the second first: `pre` of them `pre_step`
// apart, then, as all do, every step-th from `main` on.
struct SecondWalk {
  int t, end, step, pre, pre_step, main;
  __host__ __device__ __forceinline__ SecondWalk(int first, int second, int extra, int block, int blocks) {
    const int each = blocks >> 3, lane = block >> 3;
    const XcdWalk all(second, block, blocks);
    const int heavy = (first + 7) / 8 % each, light = each - heavy;
    const int base = all.t - lane;
    const bool early = lane >= heavy;
    main = base + light * extra + lane;
    t = early ? base + lane - heavy : main;
    end = all.end;
    step = each;
    pre = early ? extra : 0;
    pre_step = light;
  }
  __host__ __device__ __forceinline__ int after() const { return pre > 1 ? t + pre_step : pre ? main : t + step; }
  __host__ __device__ __forceinline__ bool more() const { return after() < end; }
  __host__ __device__ __forceinline__ void next() {
    t = after();
    pre = pre ? pre - 1 : 0;
  }
};

}  // namespace mi355
