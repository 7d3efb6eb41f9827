// voxel_windows.h -- the rows of a sparse tensor by the windows of a grid (voxel_windows.hip), as voxel_attention.h reads them.
#pragma once

#include "coord.h"

namespace sessd {

struct WindowGrid {
    int shape[3];  // z,y,x
    int window[3];
    int shift[3];
    int count[3];  // windows
    uint64_t over[3];  // 2^64 / window, rounded up; 0 for windows of one cell
    size_t windows() const { return (size_t)count[0] * count[1] * count[2]; }
};

constexpr size_t kMostWindows = 1 << 22;
constexpr int kItemRows = 64;  // queries of a work item
// Rows of a window: up to kTinyRows it is listed as a whole, beyond it has items, beyond kShortRows they are the long ones
constexpr int kTinyRows = 32, kShortRows = 128;

// Words of WindowIndex::head.  Four ranges that window_base takes stand one after the other;
// kHeadRows: voxel_num as the list was made, which later readers go by (rows that it does not name have no places)
enum { kHeadStatus = 0, kHeadPlaces, kHeadLong, kHeadShort, kHeadTiny, kHeadOutside, kHeadRows, kHeadWords = 64 };

// What a layer's workspace holds.  The list comes first: its place follows from max_voxels and the number of windows alone, which layers
// on the same windows share.
struct WindowIndex {
    int32_t* head;
    int32_t* order;  // places 0 .. places - 1: rows by windows, a window's rows ascending; behind them the rows outside the grid
    float4* cell;    // of a place: its voxel, x,y,z from the window's first one on
    int4* items;     // first place of a window, its rows, first of up to kItemRows queries among them; long windows from the front on,
    int32_t items_cap;  // short ones from the back
    int2* tiny;      // first place and rows of a tiny window
    int2* span;      // of a place: first place and rows of its window (few rows)
    // while the list is made
    int2* ticket;    // of a row: its window (-1 = outside), its place among the window's rows (of its chunk)
    uint16_t* chunk_count;  // [chunks][windows]: rows
    int32_t* chunk_base;    // [chunks][windows]: the first one's place
    int32_t* list;          // the same by tickets that are given out by chance
    int32_t* count;
    int32_t* base;
    int32_t max_voxels;
    size_t bytes;
};

WindowIndex carve_windows(void* workspace, int max_voxels, size_t windows);
// Tensors of up to so many rows have spans in place of items
constexpr int kFewRows = 4096;
// coors, voxel_num -> the list; every word that is read has been written before
int launch_windows(const int32_t* coors, const int32_t* voxel_num, const WindowGrid& g, const WindowIndex& w, hipStream_t stream);

#ifdef __HIPCC__
// the window that a cell lies in on an axis: n / window, exact for n * window < 2^64
__device__ __forceinline__ int window_on_axis(const WindowGrid& g, int axis, int n) {
    const uint64_t m = g.over[axis];
    const uint64_t q = ((uint64_t)(uint32_t)n * (uint32_t)(m >> 32) + ((uint64_t)(uint32_t)n * (uint32_t)m >> 32)) >> 32;
    return m ? (int)q : n;
}
// window of a row's voxel, -1 = outside the grid
__device__ __forceinline__ int window_of(const int4 c, const WindowGrid& g) {  // (b,z,y,x)
    if (c.x != 0 || c.y < 0 || c.y >= g.shape[0] || c.z < 0 || c.z >= g.shape[1] || c.w < 0 || c.w >= g.shape[2]) return -1;
    return (window_on_axis(g, 0, c.y + g.shift[0]) * g.count[1] + window_on_axis(g, 1, c.z + g.shift[1])) * g.count[2] + window_on_axis(g, 2, c.w + g.shift[2]);
}
// a voxel of the grid from its window's first cell on: x,y,z
__device__ __forceinline__ float4 cell_of(const int4 c, const WindowGrid& g) {
    const int z = c.y + g.shift[0], y = c.z + g.shift[1], x = c.w + g.shift[2];
    return make_float4((float)(x - window_on_axis(g, 2, x) * g.window[2]), (float)(y - window_on_axis(g, 1, y) * g.window[1]),
                       (float)(z - window_on_axis(g, 0, z) * g.window[0]), 0.f);
}

__device__ __forceinline__ int4 long_item(const WindowIndex& w, int i) { return w.items[i]; }
__device__ __forceinline__ int4 short_item(const WindowIndex& w, int i) { return w.items[w.items_cap - 1 - i]; }
#endif

}  // namespace sessd
