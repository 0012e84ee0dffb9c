// The index arithmetic of a slot map (r3d_pool.hip), apart from the kernel around it: what a workgroup looks up and what its threads
// read.  Templates over the arrays, so that a build for the host can run it with every index checked (tests/test_slot_map_host.py).
#pragma once

#include <cstdint>

#ifdef __HIPCC__
#define R3D_MAP_INLINE __device__ __forceinline__
#else
#define R3D_MAP_INLINE inline
#endif

namespace r3d {

// kMapAhead: pairs of tokens of a thread.  All of a workgroup's are on their way together (38 million slots: 86 us in two turns of four
// pairs, 81 in one of four, 81 in one of eight, 99 in one of two).
constexpr int kMapLds = 512, kMapAhead = 4, kMapTokens = kMapAhead * 512;

// Last sequence i in [lo, hi) with off[i - base] <= t, i.e. the one token t falls in (empty sequences are passed over).
template <class Offsets>
R3D_MAP_INLINE int64_t find_sequence(const Offsets &off, int64_t base, int64_t lo, int64_t hi, int64_t t) {
  while (hi - lo > 1) {
    const int64_t mid = (lo + hi) >> 1;
    if (off[mid - base] <= t) lo = mid; else hi = mid;
  }
  return lo;
}

struct MapPart {      // the sequences [lo, hi) that the tokens of a workgroup fall in; near: their offsets fit LDS
  int64_t lo, hi;
  bool near;
};

// Of the tokens [first, stop), first < stop <= offsets[n_seq].
template <class Offsets>
R3D_MAP_INLINE MapPart map_part(const Offsets &offsets, int64_t n_seq, int64_t first, int64_t stop) {
  MapPart p;
  p.lo = find_sequence(offsets, 0, 0, n_seq, first);
  p.hi = find_sequence(offsets, 0, p.lo, n_seq, stop - 1) + 1;
  p.near = p.hi - p.lo <= kMapLds;
  return p;
}

// The slots and sequences of a thread's tokens t0 + 512 u + {0, 1}, -1 from `stop` on.  near_off: offsets[lo .. hi], where near.
template <class Args, class Near>
R3D_MAP_INLINE void map_walk(const Args &a, const Near &near_off, MapPart part, int64_t t0, int64_t stop, int64_t (&slot)[kMapAhead][2],
                             int32_t (&seq)[kMapAhead][2]) {
  int64_t i = -1, start = 0, end = t0, row = 0;      // the sequence that a token before this one fell in
#ifdef __HIPCC__
#pragma unroll
#endif
  for (int u = 0; u < kMapAhead; ++u) {
    int64_t blk = 0, in = -1, page = 0;
#ifdef __HIPCC__
#pragma unroll
#endif
    for (int j = 0; j < 2; ++j) {
      const int64_t t = t0 + u * 512 + j;
      slot[u][j] = -1;
      seq[u][j] = -1;
      if (t >= stop) continue;
      if (t >= end) {                      // the next sequence that has points
        const int64_t from = i < 0 ? part.lo : i + 1;
        i = part.near ? find_sequence(near_off, part.lo, from, part.hi, t) : find_sequence(a.offsets, 0, from, a.n_seq, t);
        start = part.near ? near_off[i - part.lo] : a.offsets[i];
        end = part.near ? near_off[i - part.lo + 1] : a.offsets[i + 1];
        row = a.rows ? a.rows[i] : i;
        in = -1;
      }
      if (in < 0) {
        const int64_t at = t - start;
        blk = a.shift >= 0 ? at >> a.shift : (int64_t)((uint32_t)at / (uint32_t)a.block);
        in = at - blk * a.block;
        page = a.tables ? a.tables[row * a.most + blk] : row;
      } else if (++in == a.block) {
        in = 0;
        page = a.tables ? a.tables[row * a.most + ++blk] : row;
      }
      slot[u][j] = page < 0 ? -1 : page * a.block + in;
      seq[u][j] = (int32_t)i;
    }
  }
}

}  // namespace r3d
