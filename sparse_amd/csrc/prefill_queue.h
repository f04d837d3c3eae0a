// The tile queues of a prefill-size FFN call (swiglu_prefill_merged.hip says how they are ordered): layout of the
// workspace, and the device code that builds them, for a launch of its own or beside other work.
#pragma once

#include "common.h"
#include "prefill_tiles.h"

namespace sparse {

struct PfxMapArgs {
  const int32_t* expert_slot;
  const int32_t* seg_offsets;
  sparse_hip_seglist segs;
  int32_t* hdr;            // per launch (gate/up, down) 16 ints: first entry [8], entries [8]
  PfTile* map_gu;          // entry 0 of each map is the idle entry
  PfTile* map_dn;
  int32_t nt_gu, nt_dn;    // column tiles of a routed expert
  int32_t nts_gu, nts_dn;  // column tiles of the shared expert (0: none)
  int32_t mts_gu, mts_dn;  // row tiles of the shared expert
  int32_t T;               // tokens (rows of the shared expert)
  int32_t cap_gu, cap_dn;  // entries in each map
  int32_t tile_rows;       // rows per tile, kPfBM or fewer
  int32_t shared_rows;     // ... of the shared expert's gate/up tiles
};

// Share x of n items cut into kPfXcds contiguous shares starts here.
__device__ __forceinline__ int pfx_start(int n, int x) { return static_cast<int>(static_cast<int64_t>(n) * x / kPfXcds); }   // (a shift)
__device__ __forceinline__ int pfx_share_of(int n, int i) {
  int x = min(kPfXcds - 1, static_cast<int>(static_cast<float>(i) * kPfXcds / static_cast<float>(max(n, 1))));   // within one; the loops settle it
  while (x + 1 < kPfXcds && pfx_start(n, x + 1) <= i) ++x;
  while (x > 0 && pfx_start(n, x) > i) --x;
  return x;
}
// Queue x of a launch with R routed and S shared tiles: its share of the shared tiles, then its share
// of the routed ones (the shared expert's down tiles are the long ones, so they go first).
__device__ __forceinline__ int pfx_queue_base(int R, int S, int x) { return 1 + pfx_start(S, x) + pfx_start(R, x); }

// One workgroup of 256 threads, number b of nt_gu + nt_dn + 2, of the queue build.  Workgroups [0, nt_gu) and
// [nt_gu, nt_gu + nt_dn): one per routed column tile of the two launches -- segment s -> its row-tile count, scan,
// then thread s writes the entries of (segment s, this column tile, row tile 0 ..), routed order (segment, column
// tile, row tile).  The two last workgroups write the shared expert's entries (column tile, row tile) and the queue
// headers of their launch.
__device__ __forceinline__ void prefill_queue_block(const PfxMapArgs& a, const int b) {
  static_assert(SPARSE_HIP_MAX_EXPERTS <= 256, "one thread per segment");
  const int tid = threadIdx.x;
  int nseg = a.segs.n;
  if (a.segs.eids_dev != nullptr) nseg = min(nseg, a.segs.count_dev[0]);
  int mt = 0, slot = 0, r0 = 0, rows = 0;
  if (tid < nseg) {
    const int e = (a.segs.eids_dev != nullptr) ? a.segs.eids_dev[tid] : a.segs.eids[tid];
    r0 = a.seg_offsets[e];
    rows = a.seg_offsets[e + 1] - r0;
    mt = (rows + a.tile_rows - 1) / a.tile_rows;
    slot = (a.segs.eids_dev != nullptr) ? (a.expert_slot != nullptr ? a.expert_slot[e] : e) : a.segs.slots[tid];
  }
  // inclusive scan: within the wavefronts, then over their totals
  int scan = mt;
  for (int off = 1; off < 64; off <<= 1) {
    const int v = __shfl_up(scan, off);
    if ((tid & 63) >= off) scan += v;
  }
  __shared__ int32_t s_total[4];
  if ((tid & 63) == 63) s_total[tid >> 6] = scan;
  __syncthreads();
  for (int w = 0; w < (tid >> 6); ++w) scan += s_total[w];
  const int total_mt = s_total[0] + s_total[1] + s_total[2] + s_total[3];
  if (b < a.nt_gu + a.nt_dn) {
    const int which = b < a.nt_gu ? 0 : 1;
    const int bn = which == 0 ? b : b - a.nt_gu;
    PfTile* map = which == 0 ? a.map_gu : a.map_dn;
    const int nt = which == 0 ? a.nt_gu : a.nt_dn;
    const int cap = which == 0 ? a.cap_gu : a.cap_dn;
    const int R = total_mt * nt, S = which == 0 ? a.mts_gu * a.nts_gu : a.mts_dn * a.nts_dn;
    if (mt > 0) {
      const int g0 = (scan - mt) * nt + bn * mt;
      for (int bm = 0; bm < mt; ++bm) {
        const int g = g0 + bm;
        const int x = pfx_share_of(R, g);
        const int pos = pfx_queue_base(R, S, x) + (pfx_start(S, x + 1) - pfx_start(S, x)) + (g - pfx_start(R, x));
        if (pos < cap) map[pos] = PfTile{slot, r0 + bm * a.tile_rows, min(a.tile_rows, rows - bm * a.tile_rows), bn};
      }
    }
    return;
  }
  const int which = b - (a.nt_gu + a.nt_dn);
  PfTile* map = which == 0 ? a.map_gu : a.map_dn;
  const int nt = which == 0 ? a.nt_gu : a.nt_dn;
  const int cap = which == 0 ? a.cap_gu : a.cap_dn;
  const int mts = which == 0 ? a.mts_gu : a.mts_dn, rows_s = which == 0 ? a.shared_rows : a.tile_rows;
  const int R = total_mt * nt, S = mts * (which == 0 ? a.nts_gu : a.nts_dn);
  // The shared expert's tiles.  Where the tile grid divides evenly, XCD x takes a block of it -- a quarter
  // of the row tiles by half of the column tiles -- and walks the block down its rows first, so that the
  // 64 workgroups an XCD runs at a time cover about 8 x 8 tiles: each activation row tile and each weight
  // tile is then fetched into that L2 once per 8 users.  (Column by column over all row tiles, an XCD reads
  // the whole activation matrix, four times its L2, once per column tile.)  Otherwise: contiguous shares
  // of the (column tile, row tile) order.
  const int nts = which == 0 ? a.nts_gu : a.nts_dn;
  const bool blocked = mts % 4 == 0 && nts % 2 == 0 && nts > 0;
  const int RG = mts / 4, per_xcd = S / kPfXcds;
  for (int h = tid; h < S; h += 256) {
    int bn, bm, x, local;
    if (blocked) {
      x = h / per_xcd;
      local = h - x * per_xcd;
      bm = (x & 3) * RG + local % RG;
      bn = (x >> 2) * (nts / 2) + local / RG;
    } else {
      bn = h / mts;
      bm = h - bn * mts;
      x = pfx_share_of(S, h);
      local = h - pfx_start(S, x);
    }
    const int pos = pfx_queue_base(R, S, x) + local;
    if (pos < cap) map[pos] = PfTile{-1, bm * rows_s, min(rows_s, a.T - bm * rows_s), bn};
  }
  if (tid == 0) map[0] = PfTile{0, 0, 0, 0};
  if (tid < kPfXcds) {
    int32_t* hdr = a.hdr + which * 16;
    hdr[tid] = pfx_queue_base(R, S, tid);
    hdr[kPfXcds + tid] = (pfx_start(S, tid + 1) - pfx_start(S, tid)) + (pfx_start(R, tid + 1) - pfx_start(R, tid));
  }
}

inline int pfx_max_mtiles(int Ttok, int K, int nseg, int tile_rows) { return (Ttok * K + tile_rows - 1) / tile_rows + nseg; }

struct PfxLayout {
  int nt_gu, nt_dn, nts_gu, nts_dn, mts_gu, mts_dn, cap_gu, cap_dn;
};
inline PfxLayout pfx_layout(int Ttok, int K, int nseg, int H, int I, int Is, int tile_rows, int down_columns, int shared_rows) {
  PfxLayout l;
  l.nt_gu = (I + kPfBR / 2 - 1) / (kPfBR / 2);
  l.nt_dn = (H + down_columns - 1) / down_columns;
  l.nts_gu = Is > 0 ? (Is + kPfBR / 2 - 1) / (kPfBR / 2) : 0;
  l.nts_dn = Is > 0 ? l.nt_dn : 0;
  l.mts_gu = Is > 0 ? (Ttok + shared_rows - 1) / shared_rows : 0;
  l.mts_dn = Is > 0 ? (Ttok + tile_rows - 1) / tile_rows : 0;
  const int mt = nseg > 0 ? pfx_max_mtiles(Ttok, K, nseg, tile_rows) : 0;
  l.cap_gu = 1 + mt * l.nt_gu + l.mts_gu * l.nts_gu;
  l.cap_dn = 1 + mt * l.nt_dn + l.mts_dn * l.nts_dn;
  return l;
}

constexpr size_t kPfWsHeader = 256;   // two launches x 16 ints, padded

inline size_t prefill_queue_ws_bytes(int Ttok, int K, int nseg, int H, int I, int Is, int tile_rows = kPfBM,
                                     int down_columns = kPfBR, int shared_rows = kPfBM) {
  const PfxLayout l = pfx_layout(Ttok, K, nseg, H, I, Is, tile_rows, down_columns, shared_rows);
  return kPfWsHeader + (static_cast<size_t>(l.cap_gu) + l.cap_dn) * sizeof(PfTile);
}

// The arguments that build both launches' queues of a call in `tile_ws` (prefill_queue_ws_bytes), and where
// they will be.
inline PfQueues prefill_queue_args(const int32_t* expert_slot, const int32_t* seg_offsets, const sparse_hip_seglist& segs,
                                   int Ttok, int K, int H, int I, int Is, void* tile_ws, PfxMapArgs* args,
                                   int tile_rows = kPfBM, int down_columns = kPfBR, int shared_rows = kPfBM) {
  const PfxLayout l = pfx_layout(Ttok, K, segs.n, H, I, Is, tile_rows, down_columns, shared_rows);
  int32_t* hdr = static_cast<int32_t*>(tile_ws);
  PfTile* map_gu = reinterpret_cast<PfTile*>(static_cast<uint8_t*>(tile_ws) + kPfWsHeader);
  PfTile* map_dn = map_gu + l.cap_gu;
  PfxMapArgs m = {};
  m.expert_slot = expert_slot;
  m.seg_offsets = seg_offsets;
  m.segs = segs;
  m.hdr = hdr;
  m.map_gu = map_gu;
  m.map_dn = map_dn;
  m.nt_gu = l.nt_gu;
  m.nt_dn = l.nt_dn;
  m.nts_gu = l.nts_gu;
  m.nts_dn = l.nts_dn;
  m.mts_gu = l.mts_gu;
  m.mts_dn = l.mts_dn;
  m.T = Ttok;
  m.cap_gu = l.cap_gu;
  m.cap_dn = l.cap_dn;
  m.tile_rows = tile_rows;
  m.shared_rows = shared_rows;
  *args = m;
  return PfQueues{hdr, map_gu, map_dn, l.cap_gu, l.cap_dn};
}

}  // namespace sparse
