// voxel_windows.h -- the rows of a sparse tensor by the windows of a grid (voxel_windows.hip), as voxel_attention.h reads them.
#pragma once

#include "coord.h"

namespace sessd {

struct WindowGrid {
    int shape[3];  // z,y,x
    int window[3];
    int shift[3];
    int count[3];  // windows
    size_t windows() const { return (size_t)count[0] * count[1] * count[2]; }
};

constexpr size_t kMostWindows = 1 << 22;
constexpr int kItemRows = 64;  // queries of a work item

// Words of WindowIndex::head
enum { kHeadStatus = 0, kHeadPlaces, kHeadLong, kHeadShort, kHeadOutside, kHeadWords = 64 };

// What a layer's workspace holds.  The list comes first: its place follows from max_voxels and the number of windows alone, which layers
// on the same windows share.
struct WindowIndex {
    int32_t* head;
    int32_t* order;  // places 0 .. places - 1: rows by windows, a window's rows ascending; behind them the rows outside the grid
    float4* cell;    // of a place: its voxel, x,y,z
    int4* items;     // first place of a window, its rows, first of up to kItemRows queries among them; long windows from the front on,
    int32_t items_cap;  // short ones from the back
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
// coors, voxel_num -> the list; every word that is read has been written before
int launch_windows(const int32_t* coors, const int32_t* voxel_num, const WindowGrid& g, const WindowIndex& w, hipStream_t stream);

#ifdef __HIPCC__
__device__ __forceinline__ int4 window_item(const WindowIndex& w, int i, int longs) { return w.items[i < longs ? i : w.items_cap - 1 - (i - longs)]; }
#endif

}  // namespace sessd
