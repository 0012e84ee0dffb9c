// A pool of resident scenes in pages (gfx950): block tables from lengths, slot maps from tables, rows moved through a map.
//
// A finished batch stands in HBM with a length per scene that only the device knows (r3d_batch_t.n_out).  These kernels
// give every scene its blocks, number the points of the scenes a training step asks for and move the points, without a
// word to the host.  All of it is copying and prefix sums: the large calls are bound by HBM, the small ones by the launch.
// Measured: tables of 256 scenes x 74 blocks 10 us (two launches), of 23 201 scenes 29; the map of 30.7 million points (38 million slots)
// 81 us, 461 MB written at 5.7 TB/s; 480 000 rows of 20 bytes taken in 6.3 us, 7.7 million put in 86 us, 5.3 TB/s.
#include "r3d_host.hpp"
#include "r3d_map_core.hpp"

namespace {
using namespace r3d;

constexpr int kGroup = 256;          // rows of a table per workgroup (and per partial sum)

// Sum over the 256 threads of a workgroup; every thread gets it.  `s` holds 4 words; ends with the words free for re-use.
__device__ __forceinline__ int64_t group_sum(int64_t v, int64_t *s) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  v = s[0] + s[1] + s[2] + s[3];
  __syncthreads();
  return v;
}

// Inclusive sum over the threads before and including this one.
__device__ __forceinline__ int64_t group_scan(int64_t v, int64_t *s) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  if (lane == 63) s[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) v += s[w];
  __syncthreads();
  return v;
}

struct TablesArgs {
  const int32_t *lengths, *tables, *held, *free_blocks, *n_free;
  int32_t *tables_out, *held_out, *free_out, *n_free_out, *status;
  int64_t n_rows, n_blocks;
  int32_t block, most;
  int64_t *part;        // [2][groups] blocks given back / asked for by the rows of a group
  int32_t groups;
};

struct RowWant {
  int32_t have, want;   // blocks before, blocks after if served
  bool fits;
};

__device__ __forceinline__ RowWant row_want(const TablesArgs &a, int64_t row) {
  RowWant w{0, 0, true};
  if (row >= a.n_rows) return w;
  const int64_t len = a.lengths[row], held = a.held[row], bs = a.block;
  int64_t have = held > 0 ? (held + bs - 1) / bs : 0;
  w.have = (int32_t)(have > a.most ? a.most : have);      // (never beyond the table, whatever `held` says)
  const int64_t need = len > 0 ? (len + bs - 1) / bs : 0;
  w.fits = len >= 0 && need <= a.most;
  w.want = w.fits ? (int32_t)need : w.have;
  return w;
}

// What every group of rows gives back and asks for.
__global__ __launch_bounds__(kGroup) void k_tables_count(TablesArgs a) {
  __shared__ int64_t s[4];
  const RowWant w = row_want(a, (int64_t)blockIdx.x * kGroup + threadIdx.x);
  const int64_t back = group_sum(w.have > w.want ? w.have - w.want : 0, s);
  const int64_t grow = group_sum(w.want > w.have ? w.want - w.have : 0, s);
  if (threadIdx.x == 0) {
    a.part[blockIdx.x] = back;
    a.part[a.groups + blockIdx.x] = grow;
  }
}

struct Sums {
  int64_t back_before, back_all, grow_before;
};
__device__ __forceinline__ Sums sums_before(const TablesArgs &a, int group, int64_t *s) {
  if (a.groups == 1) {      // (no launch for the sums of a single group)
    const RowWant w = row_want(a, threadIdx.x);
    return Sums{0, group_sum(w.have > w.want ? w.have - w.want : 0, s), 0};
  }
  int64_t before = 0, all = 0, grow = 0;
  for (int g = threadIdx.x; g < a.groups; g += kGroup) {
    const int64_t b = a.part[g];
    all += b;
    if (g < group) {
      before += b;
      grow += a.part[a.groups + g];
    }
  }
  Sums r;
  r.back_before = group_sum(before, s);
  r.back_all = group_sum(all, s);
  r.grow_before = group_sum(grow, s);
  return r;
}

__device__ __forceinline__ int64_t clamp_free(const TablesArgs &a) {
  const int64_t n = a.n_free[0];
  return n < 0 ? 0 : n > a.n_blocks ? a.n_blocks : n;
}

// The free stack with the blocks that rows give back on its end (rows in order, blocks in order).  Two jobs that share
// the launch: workgroup g copies its part of the stack, and pushes what the rows of group g give back.
__global__ __launch_bounds__(kGroup) void k_tables_release(TablesArgs a) {
  __shared__ int64_t s[4];
  const int group = blockIdx.x;
  const int64_t row = (int64_t)group * kGroup + threadIdx.x;
  const RowWant w = group < a.groups ? row_want(a, row) : RowWant{0, 0, true};
  const Sums sum = sums_before(a, group, s);
  if (blockIdx.x == 0 && threadIdx.x == 0 && a.status) *a.status = 0;      // (k_tables_write adds what it finds)
  const int64_t n_free = clamp_free(a), n_all = n_free + sum.back_all;
  for (int64_t i = (int64_t)blockIdx.x * kGroup + threadIdx.x; i < a.n_blocks; i += (int64_t)gridDim.x * kGroup)
    if (i < n_free || i >= n_all) a.free_out[i] = i < n_free ? a.free_blocks[i] : -1;
  if (group >= a.groups) return;
  const int32_t back = w.have > w.want ? w.have - w.want : 0;
  const int64_t mine = n_free + sum.back_before + group_scan(back, s) - back;
  // a wave's rows that give something back, four at a time, 64 of their blocks each time
  const int lane = threadIdx.x & 63;
  uint64_t rows = __ballot(back > 0);
  while (rows) {
    int64_t at[4];
    const int32_t *from[4];
    int n[4], most = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int r = rows ? __builtin_ctzll(rows) : 0;
      n[k] = rows ? __shfl(back, r) : 0;
      at[k] = __shfl(mine, r);
      from[k] = a.tables + (row - lane + r) * a.most + __shfl(w.want, r);
      most = n[k] > most ? n[k] : most;
      rows &= rows - 1;
    }
    for (int c = lane; c < most; c += 64) {
      int32_t v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = c < n[k] ? from[k][c] : 0;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (c < n[k] && at[k] + c < a.n_blocks) a.free_out[at[k] + c] = v[k];
    }
  }
}

// The new tables.  A growing row pops its blocks from the end of the stack; the cell that takes an entry is the only one
// that touches it, and leaves -1 there.  Every workgroup takes a slice of a group's rows (gridDim.y slices).
__global__ __launch_bounds__(kGroup) void k_tables_write(TablesArgs a) {
  __shared__ int64_t s[4];
  __shared__ int64_t s_number[kGroup];     // number of the row's first new block among all that are handed out
  __shared__ int32_t s_have[kGroup], s_want[kGroup];
  const int group = blockIdx.x;
  const Sums sum = sums_before(a, group, s);
  int64_t n_all = clamp_free(a) + sum.back_all;
  const bool odd = n_all > a.n_blocks;      // a block is both free and held: the caller's tables contradict each other
  if (odd) n_all = a.n_blocks;
  const int64_t row = (int64_t)group * kGroup + threadIdx.x;
  const RowWant w = row_want(a, row);
  const int32_t grow = w.want > w.have ? w.want - w.have : 0;
  const int64_t run = sum.grow_before + group_scan(grow, s);
  const bool served = grow == 0 || run <= n_all;
  s_number[threadIdx.x] = run - grow;
  s_have[threadIdx.x] = w.have;
  s_want[threadIdx.x] = served ? w.want : w.have;
  const int64_t taken = sum.grow_before + group_sum(served ? grow : 0, s);    // (served rows of a group are a prefix of it)
  const int64_t asked = sum.grow_before + group_sum(grow, s);
  const int64_t refused = group_sum(row < a.n_rows && !(served && w.fits) ? 1 : 0, s);
  if (blockIdx.y == 0) {
    if (row < a.n_rows) a.held_out[row] = w.fits && served ? a.lengths[row] : a.held[row];
    if (threadIdx.x == 0) {
      // the totals: written by the group in which the stack runs out, else by the last one
      if (sum.grow_before <= n_all && (asked > n_all || group == a.groups - 1)) a.n_free_out[0] = (int32_t)(n_all - taken);
      if (a.status && (refused || odd)) atomicOr(reinterpret_cast<unsigned int *>(a.status), (unsigned)R3D_S_CAPACITY);
    }
  }
  __syncthreads();
  const int64_t rows = min((int64_t)kGroup, a.n_rows - (int64_t)group * kGroup);
  const int64_t cells = rows * a.most, first = (int64_t)group * kGroup * a.most;
  const bool few = cells <= UINT32_MAX;
  for (int64_t i = (int64_t)blockIdx.y * kGroup + threadIdx.x; i < cells; i += (int64_t)gridDim.y * kGroup) {
    const int r = few ? (int)((unsigned)i / (unsigned)a.most) : (int)(i / a.most), c = (int)(i - (int64_t)r * a.most);
    int32_t v = -1;
    if (c < s_want[r]) {
      if (c < s_have[r]) {
        v = a.tables[first + i];
      } else {
        const int64_t at = n_all - 1 - (s_number[r] + (c - s_have[r]));
        v = a.free_out[at];
        a.free_out[at] = -1;
      }
    }
    a.tables_out[first + i] = v;
  }
}

// ---- slot maps -------------------------------------------------------------------------------------------------------
struct MapArgs {
  const int32_t *lengths, *tables, *rows;
  int64_t n_lengths, n_seq, capacity;
  int32_t block, most, shift;      // shift: log2(block) where block is a power of two, else -1
  int64_t *offsets, *slots;
  int32_t *sequence;
};

__device__ __forceinline__ int64_t seq_row(const MapArgs &a, int64_t i) { return a.rows ? a.rows[i] : i; }

// Points of sequence i: 0 for a row that is not there or a negative length, never more than the row's table has room for.
__device__ __forceinline__ int64_t seq_length(const MapArgs &a, int64_t i) {
  const int64_t row = seq_row(a, i);
  if (row < 0 || row >= a.n_lengths) return 0;
  const int64_t len = a.lengths[row], room = (int64_t)a.most * a.block;
  return len < 0 ? 0 : len > room ? room : len;
}

// Exclusive sums of the lengths, one workgroup: every thread takes a run of sequences.
__global__ __launch_bounds__(1024) void k_map_offsets(MapArgs a) {
  __shared__ int64_t s_wave[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t each = (a.n_seq + 1023) / 1024, lo = min(each * threadIdx.x, a.n_seq), hi = min(lo + each, a.n_seq);
  int64_t mine = 0;
  for (int64_t i = lo; i < hi; ++i) mine += seq_length(a, i);
  int64_t run = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  if (lane == 63) s_wave[wave] = run;
  __syncthreads();
  for (int w = 0; w < wave; ++w) run += s_wave[w];
  int64_t at = run - mine;
  for (int64_t i = lo; i < hi; ++i) {
    a.offsets[i] = at;
    at += seq_length(a, i);
  }
  if (threadIdx.x == 1023) a.offsets[a.n_seq] = run;
}

// kSums: the offsets are made here, by every workgroup for itself (n_seq <= kMapLds), and there is no k_map_offsets before.
template <bool kSums>
__global__ __launch_bounds__(256) void k_map_slots(MapArgs a) {
  __shared__ int64_t s_off[kMapLds + 1];
  const int64_t first = (int64_t)blockIdx.x * kMapTokens, last = min(first + kMapTokens, a.capacity);
  MapPart part{0, 0, false};
  int64_t total;
  if constexpr (kSums) {
    static_assert(kMapLds == 512, "two sequences a thread");
    __shared__ int64_t s[4];
    const int64_t i = threadIdx.x * 2, l0 = i < a.n_seq ? seq_length(a, i) : 0, l1 = i + 1 < a.n_seq ? seq_length(a, i + 1) : 0;
    const int64_t run = group_scan(l0 + l1, s);
    if (i < a.n_seq) s_off[i] = run - l0 - l1;
    if (i + 1 < a.n_seq) s_off[i + 1] = run - l1;
    if (threadIdx.x == 255) s_off[a.n_seq] = run;
    __syncthreads();
    if (blockIdx.x == 0)
      for (int64_t k = threadIdx.x; k <= a.n_seq; k += 256) a.offsets[k] = s_off[k];
    total = s_off[a.n_seq];
    part = MapPart{0, a.n_seq, true};
  } else {
    total = a.offsets[a.n_seq];
  }
  const int64_t stop = min(last, total);      // tokens beyond the capacity are left out: what is looked up here ends before them
  if (!kSums && first < stop) {
    // the sequences this part of the tokens touches; short ranges are searched in LDS from then on
    part = map_part(a.offsets, a.n_seq, first, stop);
    if (part.near)
      for (int64_t i = threadIdx.x; i <= part.hi - part.lo; i += 256) s_off[i] = a.offsets[part.lo + i];
  }
  __syncthreads();
  // a thread's tokens two by two, so that the lanes of a store lie in one line: 1 KB of slots, 512 bytes of numbers
  const int64_t t0 = first + threadIdx.x * 2;
  int64_t slot[kMapAhead][2];
  int32_t seq[kMapAhead][2];
  map_walk(a, s_off, part, t0, stop, slot, seq);
#pragma unroll
  for (int u = 0; u < kMapAhead; ++u) {
    const int64_t t = t0 + u * 512;
    if (t + 2 <= last) {
      *reinterpret_cast<longlong2 *>(a.slots + t) = make_longlong2(slot[u][0], slot[u][1]);
      *reinterpret_cast<int2 *>(a.sequence + t) = make_int2(seq[u][0], seq[u][1]);
    } else if (t < last) {
      a.slots[t] = slot[u][0];
      a.sequence[t] = seq[u][0];
    }
  }
}

// ---- rows through maps --------------------------------------------------------------------------------------------------
struct RowsArgs {
  r3d_rows_t a[R3D_MAX_ROW_ARRAYS];
  int32_t n_arrays, unit[R3D_MAX_ROW_ARRAYS];      // unit: bytes of one load (16, 8, 4, 2, 1)
  const int64_t *src_slots, *dst_slots;
  int64_t n, n_src, n_dst;
};

template <class U>
__device__ __forceinline__ void move_unit(const r3d_rows_t &a, int64_t from, int64_t to, int64_t u, bool zero) {
  U v{};
  if (!zero) v = *reinterpret_cast<const U *>(static_cast<const char *>(a.src) + from * a.src_stride + u * (int64_t)sizeof(U));
  *reinterpret_cast<U *>(static_cast<char *>(a.dst) + to * a.dst_stride + u * (int64_t)sizeof(U)) = v;
}

__device__ __forceinline__ void move_any(const RowsArgs &g, int k, int64_t from, int64_t to, int64_t u, bool zero) {
  switch (g.unit[k]) {
    case 16: move_unit<uint4>(g.a[k], from, to, u, zero); break;
    case 8: move_unit<uint2>(g.a[k], from, to, u, zero); break;
    case 4: move_unit<uint32_t>(g.a[k], from, to, u, zero); break;
    case 2: move_unit<uint16_t>(g.a[k], from, to, u, zero); break;
    default: move_unit<uint8_t>(g.a[k], from, to, u, zero); break;
  }
}

// Where row t comes from and goes to: false when it is left out (no destination); `zero`: it has no source.
__device__ __forceinline__ bool row_ends(const RowsArgs &g, int64_t t, int64_t &from, int64_t &to, bool &zero) {
  from = g.src_slots ? g.src_slots[t] : t;
  to = g.dst_slots ? g.dst_slots[t] : t;
  zero = from < 0 || from >= g.n_src;
  // a take (no destination map) fills a row without a source with zeros; a put leaves its destination as it was
  return to >= 0 && to < g.n_dst && !(zero && g.dst_slots);
}

// Rows of one unit in every array (a point's 16 bytes, its label): a thread per row, neighbouring rows by neighbouring lanes --
// the points of a block lie in a line, so both sides are whole cache lines.  (Two or four rows a thread: 88 and 91 us for the put above, with
// one 86: nothing waits but HBM.)
__global__ __launch_bounds__(256) void k_rows_thin(RowsArgs g) {
  for (int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x; t < g.n; t += (int64_t)gridDim.x * 256) {
    int64_t from, to;
    bool zero;
    if (!row_ends(g, t, from, to, zero)) continue;
    for (int k = 0; k < g.n_arrays; ++k) move_any(g, k, from, to, 0, zero);
  }
}

// Rows of any width: the units of the rows in one line, a thread per unit; gridDim.y arrays.
__global__ __launch_bounds__(256) void k_rows_wide(RowsArgs g) {
  const int k = blockIdx.y;
  const int64_t units = g.a[k].row_bytes / g.unit[k], all = g.n * units;
  for (int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x; e < all; e += (int64_t)gridDim.x * 256) {
    const int64_t t = e / units;
    int64_t from, to;
    bool zero;
    if (!row_ends(g, t, from, to, zero)) continue;
    move_any(g, k, from, to, e - t * units, zero);
  }
}

int64_t groups_of(int64_t n_rows) { return (n_rows + kGroup - 1) / kGroup; }
}  // namespace

extern "C" size_t r3d_block_tables_workspace_bytes(int64_t n_rows) {
  if (n_rows <= 0 || n_rows > R3D_MAX_SCENES) return 0;
  return align_up((size_t)groups_of(n_rows) * 2 * sizeof(int64_t));
}

extern "C" int r3d_block_tables(const int32_t *lengths, int64_t n_rows, int32_t block_size, int32_t max_blocks, const int32_t *tables,
                                const int32_t *held, const int32_t *free_blocks, int64_t n_blocks, const int32_t *n_free,
                                int32_t *tables_out, int32_t *held_out, int32_t *free_out, int32_t *n_free_out, int32_t *status,
                                void *workspace, size_t workspace_bytes, void *stream) {
  if (!lengths || !tables || !held || !free_blocks || !n_free || !tables_out || !held_out || !free_out || !n_free_out || !workspace)
    return fail(R3D_E_ARG, "block_tables: null pointer");
  if (n_rows <= 0 || n_rows > R3D_MAX_SCENES || block_size <= 0 || max_blocks <= 0 || n_blocks <= 0 || n_blocks > INT32_MAX ||
      (int64_t)max_blocks * block_size > INT32_MAX || n_rows * (int64_t)max_blocks > (1ll << 40))
    return fail(R3D_E_ARG, "block_tables: bad size");
  if (tables == tables_out || held == held_out || free_blocks == free_out || n_free == n_free_out)
    return fail(R3D_E_ARG, "block_tables: an output is its input");
  if (!aligned(workspace, 8)) return fail(R3D_E_ARG, "block_tables: workspace must be 8-byte aligned");
  if (workspace_bytes < r3d_block_tables_workspace_bytes(n_rows)) return fail(R3D_E_WORKSPACE, "block_tables: workspace too small");
  hipStream_t st = static_cast<hipStream_t>(stream);
  TablesArgs a{lengths, tables, held, free_blocks, n_free, tables_out, held_out, free_out, n_free_out, status, n_rows, n_blocks,
               block_size, max_blocks, static_cast<int64_t *>(workspace), (int32_t)groups_of(n_rows)};
  if (a.groups > 1) hipLaunchKernelGGL(k_tables_count, dim3(a.groups), dim3(kGroup), 0, st, a);
  const int copies = blocks_for(n_blocks, kGroup * 8, 1024);
  hipLaunchKernelGGL(k_tables_release, dim3(a.groups > copies ? a.groups : copies), dim3(kGroup), 0, st, a);
  // slices: two cells a thread (256 x 74: 7.8 us with eight, 6.0 with two), four workgroups a CU at most (23 201 x 74: 11 us, with
  // 3400 workgroups, each of which sums the groups before it, 20)
  const int64_t cells = (n_rows < kGroup ? n_rows : kGroup) * max_blocks;
  int slices = blocks_for(cells, kGroup * 2, 1024);
  while (slices > 1 && (int64_t)slices * a.groups > 1024) slices /= 2;
  hipLaunchKernelGGL(k_tables_write, dim3(a.groups, slices), dim3(kGroup), 0, st, a);
  R3D_LAUNCHED("block_tables kernels");
  return R3D_OK;
}

extern "C" int r3d_slot_map(const int32_t *lengths, int64_t n_lengths, const int32_t *tables, int32_t block_size, int32_t max_blocks,
                            const int32_t *rows, int64_t n_seq, int64_t capacity, int64_t *offsets, int64_t *slots,
                            int32_t *sequence, void *stream) {
  if (!lengths || !offsets || !slots || !sequence) return fail(R3D_E_ARG, "slot_map: null pointer");
  if (n_lengths <= 0 || n_lengths > INT32_MAX || n_seq < 0 || n_seq > R3D_MAX_SCENES || (!rows && n_seq > n_lengths) || capacity < 0 ||
      block_size <= 0 || (tables && max_blocks <= 0) || capacity > (1ll << 40) ||
      (tables && (int64_t)max_blocks * block_size > INT32_MAX))
    return fail(R3D_E_ARG, "slot_map: bad size");
  if (!aligned(slots, 16) || !aligned(sequence, 16) || !aligned(offsets, 8))
    return fail(R3D_E_ARG, "slot_map: slots and sequence must be 16-byte aligned, offsets 8");
  hipStream_t st = static_cast<hipStream_t>(stream);
  MapArgs a{lengths, tables, rows, n_lengths, n_seq, capacity, block_size, tables ? max_blocks : 1, -1, offsets, slots, sequence};
  if ((block_size & (block_size - 1)) == 0) a.shift = __builtin_ctz((unsigned)block_size);
  // few sequences: one launch, in which every workgroup makes the sums (256 scenes, 38 million slots: one microsecond less
  // than without, and 5 and a launch of k_map_offsets; 8 scenes, 64 000 points: 6.3 us)
  const int64_t blocks = (capacity + kMapTokens - 1) / kMapTokens;
  if (blocks > 0 && n_seq <= kMapLds) {
    hipLaunchKernelGGL(k_map_slots<true>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  } else {
    hipLaunchKernelGGL(k_map_offsets, dim3(1), dim3(1024), 0, st, a);
    if (blocks > 0) hipLaunchKernelGGL(k_map_slots<false>, dim3((unsigned)blocks), dim3(256), 0, st, a);
  }
  R3D_LAUNCHED("slot_map kernels");
  return R3D_OK;
}

extern "C" int r3d_move_rows(const r3d_rows_t *arrays, int32_t n_arrays, const int64_t *src_slots, const int64_t *dst_slots, int64_t n,
                             int64_t n_src, int64_t n_dst, void *stream) {
  if (!arrays || n_arrays <= 0 || n_arrays > R3D_MAX_ROW_ARRAYS || n < 0 || n_src < 0 || n_dst < 0 || n > (1ll << 40))
    return fail(R3D_E_ARG, "move_rows: bad argument");
  if (!aligned(src_slots, 8) || !aligned(dst_slots, 8)) return fail(R3D_E_ARG, "move_rows: slots must be 8-byte aligned");
  if ((!src_slots && n > n_src) || (!dst_slots && n > n_dst)) return fail(R3D_E_ARG, "move_rows: more rows than the side without a map has");
  RowsArgs g{};
  g.n_arrays = n_arrays;
  g.src_slots = src_slots;
  g.dst_slots = dst_slots;
  g.n = n;
  g.n_src = n_src;
  g.n_dst = n_dst;
  bool thin = true;
  int64_t most = 0;
  for (int k = 0; k < n_arrays; ++k) {
    const r3d_rows_t &r = arrays[k];
    if (!r.src || !r.dst || r.row_bytes <= 0 || r.src_stride < 0 || r.dst_stride < r.row_bytes || r.row_bytes > (1ll << 30))
      return fail(R3D_E_ARG, "move_rows: bad array");
    g.a[k] = r;
    const uint64_t all = reinterpret_cast<uintptr_t>(r.src) | reinterpret_cast<uintptr_t>(r.dst) | (uint64_t)r.row_bytes |
                         (uint64_t)r.src_stride | (uint64_t)r.dst_stride;
    int unit = 16;
    while (all & (unit - 1)) unit /= 2;
    g.unit[k] = unit;
    thin = thin && r.row_bytes == unit;
    if (r.row_bytes / unit > most) most = r.row_bytes / unit;
  }
  if (n == 0) return R3D_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (thin)
    hipLaunchKernelGGL(k_rows_thin, dim3(blocks_for(n, 256, 1 << 16)), dim3(256), 0, st, g);
  else
    hipLaunchKernelGGL(k_rows_wide, dim3(blocks_for(n * most, 256, 1 << 16), n_arrays), dim3(256), 0, st, g);
  R3D_LAUNCHED("move_rows kernel");
  return R3D_OK;
}
