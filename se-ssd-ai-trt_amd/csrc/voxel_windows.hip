// voxel_windows.hip -- the rows of a sparse tensor, which come in the order in which their voxels were met, by the windows of a grid.
//
// A window's rows are listed ascending, so that the order of a row's sums does not depend on chance; where a window's rows begin does.
//
//   window_count   1 024 rows a workgroup: each row's place among its window's rows of the chunk, and the chunk's counts for all windows.
//                  A wave finds the lanes that share a window with ballots over the window's bits; then the waves add their counts one
//                  after the other, in LDS
//   window_base    a thread for each window: its rows over all chunks, its place in the list, each chunk's place in it, its work items
//   window_place   rows into the list
//
// No atomics in the first pass: all of a near window's rows would ask at one address, 24 ns each (627 rows of 16 000 in one window: 15 us).
// Tensors of up to kFewRows rows take one launch instead of three, which is what bounds a call on few rows (the host takes 3.4 us for a launch):
//
//   window_few     kFewOwn rows a workgroup, and the windows of all rows in its LDS: a row's place is the number of rows with smaller windows and of
//                  those with the same one in front of it.  (Comparisons bound it: 2 000 rows 12 us with 64 rows a workgroup, 6 with 16, 5 with 8)
//
// Where a larger tensor has more windows than LDS holds counts for (kMostCounted), windows are small, and where it has more than 2^20 rows, tickets
// are given out by atomics:
//
//   window_ticket, window_base, window_scatter, window_rank    the last puts a window's rows in ascending order
#include "fill.h"
#include "voxel_windows.h"

namespace sessd {

namespace {

constexpr int kBlock = 256;
constexpr int kChunk = 1024;
constexpr int kFewOwn = 8;
constexpr int kMostCounted = 32768;  // windows: 64 KB of 16-bit counts

constexpr int kMostCountedRows = 1 << 20;  // 1 024 chunks, whose counts a thread adds up
bool counts(int max_voxels, size_t windows) { return windows <= kMostCounted && max_voxels <= kMostCountedRows; }

size_t counted_windows(size_t windows) { return (windows + 7) / 8 * 8; }

__global__ void __launch_bounds__(kChunk)
window_count(const int32_t* __restrict__ coors, const int32_t* __restrict__ voxel_num, WindowGrid g, int windows, int bits, WindowIndex w) {
    extern __shared__ uint4 s_count4[];
    uint16_t* s_count = reinterpret_cast<uint16_t*>(s_count4);
    const int row = blockIdx.x * kChunk + threadIdx.x, wave = threadIdx.x >> 6;
    int4 c = make_int4(-1, 0, 0, 0);
    if (row < w.max_voxels) c = reinterpret_cast<const int4*>(coors)[row];
    for (int i = threadIdx.x; i < windows / 8; i += kChunk) s_count4[i] = make_uint4(0, 0, 0, 0);
    const int n = clamp_rows(voxel_num, w.max_voxels);
    if (blockIdx.x == 0 && threadIdx.x < kHeadWords) w.head[threadIdx.x] = threadIdx.x == kHeadRows ? n : 0;
    if ((int)blockIdx.x * kChunk >= n) return;
    const int key = row < n ? window_of(c, g) : -1;
    uint64_t same = __ballot(key >= 0);
    for (int b = 0; b < bits; ++b) {
        const bool mine = (key >> b) & 1;
        const uint64_t set = __ballot(mine);
        same &= mine ? set : ~set;
    }
    const int rank = (int)rank_in_wave(same), group = (int)__popcll(same);
    const int left = (n - (int)blockIdx.x * kChunk + 63) / 64, waves = left < kChunk / 64 ? left : kChunk / 64;
    int before = 0;
    __syncthreads();
    for (int i = 0; i < waves; ++i) {
        if (wave == i && key >= 0) {
            before = s_count[key];
            if (rank == group - 1) s_count[key] = (uint16_t)(before + group);
        }
        __syncthreads();
    }
    if (row < n) w.ticket[row] = make_int2(key, before + rank);
    uint4* dst = reinterpret_cast<uint4*>(w.chunk_count + (size_t)blockIdx.x * windows);
    for (int i = threadIdx.x; i < windows / 8; i += kChunk) dst[i] = s_count4[i];
}

constexpr int kTaken = 4;  // ranges that window_base takes: places, long items, short items, tiny windows

// Windows of a workgroup of window_base.  A workgroup takes its ranges with one atomic each, 8 ns apiece where all ask at one address: 250 000 windows
// 34 us with an atomic for each wave, 5 us with one for 1 024 windows.  Where chunks are to be added up, smaller workgroups reach more of the card.
constexpr int kBaseCounted = 256, kBaseTicketed = 1024;

template <bool CHUNKED, int BLOCK>
__global__ void __launch_bounds__(BLOCK)
window_base(const int32_t* __restrict__ voxel_num, int windows, WindowIndex w) {
    constexpr int kWaves = BLOCK / 64;
    __shared__ int32_t s_sum[kWaves][kTaken], s_from[kTaken];
    const int i = blockIdx.x * BLOCK + threadIdx.x, wave = threadIdx.x >> 6;
    const int chunks = CHUNKED ? (clamp_rows(voxel_num, w.max_voxels) + kChunk - 1) / kChunk : 0;
    int rows = 0;
    if (i < windows) {
        if constexpr (CHUNKED) {
#pragma unroll 8
            for (int c = 0; c < chunks; ++c) rows += w.chunk_count[(size_t)c * windows + i];
        } else {
            rows = w.count[i];
        }
    }
    const int items = rows > kTinyRows ? (rows + kItemRows - 1) / kItemRows : 0;
    const bool is_long = rows > kShortRows, is_tiny = rows > 0 && rows <= kTinyRows;
    const int mine[kTaken] = {rows, is_long ? items : 0, is_long ? 0 : items, is_tiny ? 1 : 0};
    int at[kTaken];
#pragma unroll
    for (int k = 0; k < kTaken; ++k) {
        const int upto = (int)wave_scan((uint32_t)mine[k]);
        at[k] = upto - mine[k];
        if (lane_id() == 63) s_sum[wave][k] = upto;
    }
    __syncthreads();
    if (threadIdx.x < kTaken) {
        int all = 0;
#pragma unroll
        for (int v = 0; v < kWaves; ++v) {
            const int sum = s_sum[v][threadIdx.x];
            s_sum[v][threadIdx.x] = all;
            all += sum;
        }
        s_from[threadIdx.x] = all ? atomicAdd(&w.head[kHeadPlaces + threadIdx.x], all) : 0;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kTaken; ++k) at[k] += s_sum[wave][k] + s_from[k];
    const int base = at[0], front = at[1], back = at[2], tiny = at[3];
    if (!rows) return;
    if constexpr (CHUNKED) {
        int next = base;
#pragma unroll 8
        for (int c = 0; c < chunks; ++c) {
            w.chunk_base[(size_t)c * windows + i] = next;
            next += w.chunk_count[(size_t)c * windows + i];
        }
    } else {
        w.base[i] = base;
    }
    if (is_tiny) w.tiny[tiny] = make_int2(base, rows);
    for (int k = 0; k < items; ++k) w.items[is_long ? front + k : w.items_cap - 1 - (back + k)] = make_int4(base, rows, k * kItemRows, 0);
}

__device__ __forceinline__ void set_place(const WindowIndex& w, const WindowGrid& g, int place, int row, const int4 c) {
    w.order[place] = row;
    w.cell[place] = cell_of(c, g);
}
__device__ __forceinline__ void set_outside(const WindowIndex& w, int n, int row) {
    w.order[n - 1 - atomicAdd(&w.head[kHeadOutside], 1)] = row;
    atomicOr(&w.head[kHeadStatus], SESSD_STATUS_BAD_COORD);
}

__global__ void __launch_bounds__(kBlock)
window_place(const int32_t* __restrict__ coors, const int32_t* __restrict__ voxel_num, WindowGrid g, int windows, WindowIndex w) {
    const int row = blockIdx.x * kBlock + threadIdx.x;
    if (row >= w.max_voxels) return;
    const int4 c = reinterpret_cast<const int4*>(coors)[row];
    const int n = clamp_rows(voxel_num, w.max_voxels);
    if (row >= n) return;
    const int2 t = w.ticket[row];
    if (t.x >= 0) set_place(w, g, w.chunk_base[(size_t)(row / kChunk) * windows + t.x] + t.y, row, c);
    else set_outside(w, n, row);
}

__global__ void __launch_bounds__(1024)
window_few(const int32_t* __restrict__ coors, const int32_t* __restrict__ voxel_num, WindowGrid g, WindowIndex w) {
    constexpr int kOutside = 0x7fffffff;                  // behind all windows
    __shared__ __align__(16) int32_t s_key[kFewRows];
    __shared__ int32_t s_sum[16][3][kFewOwn];
    __shared__ int32_t s_outside;
    const int tid = threadIdx.x, wave = tid >> 6, mine_at = tid % kFewOwn, own = blockIdx.x * kFewOwn + mine_at;
    const int n = clamp_rows(voxel_num, w.max_voxels), end = (n + 63) / 64 * 64;
    if (tid == 0) s_outside = 0;
    __syncthreads();
    int outside = 0;
    for (int i = tid; i < end; i += 1024) {
        const int key = i < n ? window_of(reinterpret_cast<const int4*>(coors)[i], g) : -1;
        s_key[i] = key < 0 ? kOutside : key;
        outside += i < n && key < 0 ? 1 : 0;
    }
    if (blockIdx.x == 0 && outside) atomicAdd(&s_outside, outside);
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) {
        w.head[kHeadStatus] = s_outside ? SESSD_STATUS_BAD_COORD : 0;
        w.head[kHeadPlaces] = n - s_outside;
        w.head[kHeadRows] = n;
    }
    if ((int)blockIdx.x * kFewOwn >= n) return;
    // (the rows between n and end are behind all others: smaller than none, equal to those outside, in front of none)
    const int mine = own < n ? s_key[own] : kOutside;
    int sum[3] = {0, 0, 0};                               // smaller ones, the same, those of them in front
    for (int i = tid / kFewOwn * 4; i < end; i += 1024 / kFewOwn * 4) {
        const int4 k = *reinterpret_cast<const int4*>(s_key + i);
        sum[0] += (k.x < mine) + (k.y < mine) + (k.z < mine) + (k.w < mine);
        const int e0 = k.x == mine, e1 = k.y == mine, e2 = k.z == mine, e3 = k.w == mine;
        sum[1] += e0 + e1 + e2 + e3;
        sum[2] += (i < own ? e0 : 0) + (i + 1 < own ? e1 : 0) + (i + 2 < own ? e2 : 0) + (i + 3 < own ? e3 : 0);
    }
#pragma unroll
    for (int c = 0; c < 3; ++c) {
#pragma unroll
        for (int d = kFewOwn; d < 64; d *= 2) sum[c] += __shfl_xor(sum[c], d);
        if ((tid & 63) < kFewOwn) s_sum[wave][c][mine_at] = sum[c];
    }
    __syncthreads();
    if (tid >= kFewOwn || own >= n) return;
    int less = 0, same = 0, before = 0;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        less += s_sum[i][0][mine_at];
        same += s_sum[i][1][mine_at];
        before += s_sum[i][2][mine_at];
    }
    const int place = less + before;
    w.order[place] = own;
    if (mine == kOutside) return;
    w.cell[place] = cell_of(reinterpret_cast<const int4*>(coors)[own], g);
    w.span[place] = make_int2(less, same);
}

__global__ void __launch_bounds__(kBlock)
window_ticket(const int32_t* __restrict__ coors, const int32_t* __restrict__ voxel_num, WindowGrid g, WindowIndex w) {
    const int row = blockIdx.x * kBlock + threadIdx.x;
    const int n = clamp_rows(voxel_num, w.max_voxels);
    if (row == 0) w.head[kHeadRows] = n;
    if (row >= n) return;
    const int key = window_of(reinterpret_cast<const int4*>(coors)[row], g);
    if (key < 0) set_outside(w, n, row);
    w.ticket[row] = make_int2(key, key < 0 ? 0 : atomicAdd(&w.count[key], 1));
}

__global__ void __launch_bounds__(kBlock)
window_scatter(const int32_t* __restrict__ voxel_num, WindowIndex w) {
    const int row = blockIdx.x * kBlock + threadIdx.x;
    if (row >= clamp_rows(voxel_num, w.max_voxels)) return;
    const int2 t = w.ticket[row];
    if (t.x >= 0) w.list[w.base[t.x] + t.y] = row;
}

__global__ void __launch_bounds__(kBlock)
window_rank(const int32_t* __restrict__ coors, WindowGrid g, WindowIndex w) {
    const int p = blockIdx.x * kBlock + threadIdx.x;
    if (p >= w.head[kHeadPlaces]) return;
    const int row = w.list[p], key = w.ticket[row].x;
    const int start = w.base[key], rows = w.count[key];
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < rows; ++i) rank += w.list[start + i] < row ? 1 : 0;
    set_place(w, g, start + rank, row, reinterpret_cast<const int4*>(coors)[row]);
}

}  // namespace

WindowIndex carve_windows(void* workspace, int max_voxels, size_t windows) {
    const bool few = max_voxels <= kFewRows, counted = !few && counts(max_voxels, windows), ticketed = !few && !counted;
    const size_t rows = (size_t)max_voxels, listed = few ? 0 : rows, chunks = (listed + kChunk - 1) / kChunk;
    WorkspaceCarver c(workspace);
    WindowIndex w;
    w.max_voxels = max_voxels;
    w.items_cap = (int32_t)(rows / (kTinyRows + 1) + rows / kItemRows) + 1;  // (windows that have items, and whole items)
    w.head = c.take<int32_t>(kHeadWords);
    w.order = c.take<int32_t>(rows);
    w.cell = c.take<float4>(rows);
    w.span = c.take<int2>(few ? rows : 0);
    w.items = c.take<int4>(few ? 0 : (size_t)w.items_cap);
    w.tiny = c.take<int2>(listed < windows ? listed : windows);
    w.ticket = c.take<int2>(listed);
    w.chunk_count = c.take<uint16_t>(counted ? chunks * counted_windows(windows) : 0);
    w.chunk_base = c.take<int32_t>(counted ? chunks * counted_windows(windows) : 0);
    w.list = c.take<int32_t>(ticketed ? rows : 0);
    w.count = c.take<int32_t>(ticketed ? windows : 0);
    w.base = c.take<int32_t>(ticketed ? windows : 0);
    w.bytes = c.total();
    return w;
}

int launch_windows(const int32_t* coors, const int32_t* voxel_num, const WindowGrid& g, const WindowIndex& w, hipStream_t stream) {
    const dim3 rows((unsigned)ceil_div(w.max_voxels, kBlock)), block(kBlock);
    if (w.max_voxels <= kFewRows) {
        hipLaunchKernelGGL(window_few, dim3((unsigned)ceil_div(w.max_voxels, kFewOwn)), dim3(1024), 0, stream, coors, voxel_num, g, w);
    } else if (counts(w.max_voxels, g.windows())) {
        const int windows = (int)counted_windows(g.windows());
        int bits = 0;
        while (((size_t)1 << bits) < g.windows()) ++bits;
        hipLaunchKernelGGL(window_count, dim3((unsigned)ceil_div(w.max_voxels, kChunk)), dim3(kChunk), (size_t)windows * sizeof(uint16_t), stream, coors,
                           voxel_num, g, windows, bits, w);
        hipLaunchKernelGGL((window_base<true, kBaseCounted>), dim3((unsigned)ceil_div(windows, kBaseCounted)), dim3(kBaseCounted), 0, stream, voxel_num,
                           windows, w);
        hipLaunchKernelGGL(window_place, rows, block, 0, stream, coors, voxel_num, g, windows, w);
    } else {
        const int windows = (int)g.windows();
        FillArgs f;
        f.add(w.head, kHeadWords, 0);
        f.add(w.count, (uint64_t)windows, 0);
        SESSD_TRY(launch_fill(f, stream));
        hipLaunchKernelGGL(window_ticket, rows, block, 0, stream, coors, voxel_num, g, w);
        hipLaunchKernelGGL((window_base<false, kBaseTicketed>), dim3((unsigned)ceil_div(windows, kBaseTicketed)), dim3(kBaseTicketed), 0, stream, voxel_num,
                           windows, w);
        hipLaunchKernelGGL(window_scatter, rows, block, 0, stream, voxel_num, w);
        hipLaunchKernelGGL(window_rank, rows, block, 0, stream, coors, g, w);
    }
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

}  // namespace sessd
