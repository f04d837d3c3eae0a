// C ABI of the block-scaled 8-bit operators: argument checks and the order of launches.
#include <atomic>

#include "fp8.h"
#include "prefill_queue.h"

namespace sparse {

static inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
// Which kernels serve more than kF8FewRows rows: 0 by size, 1 the streaming ones, 2 the tiles.
static std::atomic<int> g_path{0};

constexpr int kF8MaxDim = 1 << 16;          // the tile kernel keeps a scale byte per row and block in LDS
constexpr int kF8MaxOut = 1 << 28;          // columns of a product
constexpr int64_t kF8MaxRows = 1ll << 28;   // flat rows: the division by topk is a 32-bit multiply
constexpr int kF8StreamRows = 1 << 20;      // the streaming kernel's grid has a row of workgroups for every 32 rows

// The streaming kernel reads the weights once for every 32 rows; the tile kernel reads them once or twice in all,
// but starts slowly (5 us, then 0.25 us a 128-wide slab while few tiles are there to overlap).  Measured on both
// sides of the border, streaming / tiles:
//   linear  2048 x 5632: 32 rows 10.4 / 11.2 us, 64 rows 13.3 / 11.5;  4096 x 4096: 48 rows 14.8 / 15.4, 64 rows 17.1 / 15.4
//           1000 x 1418: 192 rows 9.2 / 9.7, 333 rows 11.9 / 10.2;  512 x 1024: 192 rows 7.3 / 7.6, 333 rows 8.6 / 7.7
//           5632 x 2048: 64 rows 12.3 / 18.4, 192 rows 26.7 / 19.7;  256 x 256: 512 rows 6.3 / 7.0, 1024 rows 7.5 / 7.1
//   experts 60 of 1408 x 2048, 4 a token, shared 5632: 32 tokens 80.8 / 99.6 us, 48 tokens 104 / 104, 64 tokens 113 / 107
//           16 of 704 x 1024, 3 a token: 64 tokens 20.8 / 24.8, 96 tokens 23.4 / 25.0, 128 tokens 25.9 / 25.3
//           8 of 704 x 2048, 2 a token, shared 1408: 64 tokens 25.8 / 27.5, 96 tokens 34.3 / 28.1
//           64 of 256 x 512, 6 a token: 32 tokens 18.7 / 20.2, 48 tokens 20.4 / 20.1, 64 tokens 21.3 / 20.3
static bool linear_tiles(int T, int N) {
  const int path = g_path.load(std::memory_order_relaxed);
  if (T <= kF8FewRows || path == 1) return false;
  return path == 2 || T > kF8StreamRows || static_cast<int64_t>(T) * N > 256000;
}
// (The routed experts decide, all of them, so that a layer whose experts are executed in several calls, or apart
// from the shared one, takes the same kernels in each.)
static bool ffn_tiles(int T, int K, int E, int H, int I) {
  const int path = g_path.load(std::memory_order_relaxed);
  if (T <= kF8FewRows || path == 1) return false;
  // work of the rows against a fixed cost and one for the weights
  const double size = static_cast<double>(H) * I;
  return path == 2 || T > kF8StreamRows || static_cast<double>(T) * K * (size + 1.0e6) > 3.6e8 + 2.5 * size * E;
}

// Rows per tile: the fewest of 32, 64, 128 with which the call's tiles (of 256 columns) still fit on the device
// together, two on a compute unit.  A launch of fewer tiles than that is as long as its longest tile, and one of 32
// rows takes half the time of one of 128; more tiles than that cost what the weights' second reading costs.  Tiles
// of 32 rows are then cut to 128 columns (f8_tile_columns).
static int tile_rows(int64_t rows, int segments, int column_tiles) {
  for (int r = 32; r < kPfBM; r *= 2)
    if ((rows / r + segments) * column_tiles <= 512) return r;
  return kPfBM;
}
static int ffn_tile_rows(int T, int K, int E, int H, int I) {
  // half of the segments' last tiles are half empty; gate/up has the more tiles where it has fewer columns
  const int nt_gu = (I + kPfBR / 2 - 1) / (kPfBR / 2), nt_dn = (H + kPfBR - 1) / kPfBR;
  return tile_rows(static_cast<int64_t>(T) * K, E / 2, nt_gu > nt_dn ? nt_gu : nt_dn);
}

// Rows of the shared expert's gate/up tiles: higher ones, beside routed tiles that leave less room.  128 tokens, 4 of 60
// experts of 1408 x 2048 and a shared one of 5632: 176 tiles of 32 rows behind 600 routed ones 128 us, 88 of 64 116.
static int ffn_shared_rows(int T, int K, int E, int I, int Is, int rows) {
  const int64_t routed = (static_cast<int64_t>(T) * K / rows + E / 2) * ((I + kPfBR / 2 - 1) / (kPfBR / 2));
  while (rows < kPfBM && routed + static_cast<int64_t>((T + rows - 1) / rows) * ((Is + kPfBR / 2 - 1) / (kPfBR / 2)) > 512) rows *= 2;
  return rows;
}

static inline size_t up256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

// A workspace handed out front to back in 256-byte steps; with a null base it only counts.
struct Carve {
  uint8_t* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base == nullptr ? nullptr : base + used;
    used += up256(bytes);
    return p;
  }
};

struct F8Rows {
  uint8_t *values, *scales;
};
static F8Rows take_rows(Carve& c, int64_t rows, int K) {
  F8Rows r;
  r.values = static_cast<uint8_t*>(c.take(static_cast<size_t>(rows) * f8_padded(K)));
  r.scales = static_cast<uint8_t*>(c.take(static_cast<size_t>(rows) * f8_blocks(K)));
  return r;
}

struct LinearWs {
  F8Rows x;
  size_t bytes;
};
static LinearWs linear_ws(void* ws, int T, int K) {
  Carve c{static_cast<uint8_t*>(ws)};
  LinearWs w = {};
  if (T > kF8FewRows) w.x = take_rows(c, T, K);
  w.bytes = c.used;
  return w;
}

struct FfnWs {
  F8Rows x, h, sh;
  float *hf, *shf;    // few rows: the intermediate before it is quantised
  void* tiles;        // many rows: the tile queues
  size_t bytes;
};
static FfnWs ffn_ws(void* ws, int T, int K, int E, int nseg, int H, int I, int Is) {
  Carve c{static_cast<uint8_t*>(ws)};
  FfnWs w = {};
  const int64_t rows = nseg > 0 ? static_cast<int64_t>(T) * K : 0;
  const bool tiles = ffn_tiles(T, K, E, H, I);
  if (T > kF8FewRows) {
    if (tiles) w.x.values = static_cast<uint8_t*>(c.take(static_cast<size_t>(T) * f8_padded(H) * sizeof(uint16_t)));
    else w.x = take_rows(c, T, H);
    w.h = take_rows(c, rows, I);
    if (Is > 0) w.sh = take_rows(c, T, Is);
  }
  if (tiles) {
    const int rows_per_tile = ffn_tile_rows(T, K, E, H, I);
    w.tiles = c.take(prefill_queue_ws_bytes(T, K, nseg, H, I, Is, rows_per_tile, f8_tile_columns(rows_per_tile),
                                            ffn_shared_rows(T, K, E, I, Is, rows_per_tile)));
  } else {
    w.hf = static_cast<float*>(c.take(static_cast<size_t>(rows) * I * sizeof(float)));
    if (Is > 0) w.shf = static_cast<float*>(c.take(static_cast<size_t>(T) * Is * sizeof(float)));
  }
  w.bytes = c.used;
  return w;
}

static int check_matrix(const char* fn, const char* name, const sparse_hip_fp8_matrix* m, int rows, int cols) {
  SP_REQUIRE(m->rows == rows && m->cols == cols, "%s: %s is [%d,%d], must be [%d,%d]", fn, name, m->rows, m->cols, rows, cols);
  SP_REQUIRE(m->values_dev && m->scales_dev, "%s: %s has a NULL pointer", fn, name);
  SP_REQUIRE(aligned16(m->values_dev), "%s: %s values must be 16-byte aligned", fn, name);
  return SPARSE_HIP_OK;
}

}  // namespace sparse

using namespace sparse;

extern "C" {

int sparse_hip_fp8_path(int which) {
  SP_REQUIRE(which >= 0 && which <= 2, "fp8_path: %d outside [0,2]", which);
  return g_path.exchange(which);
}

int sparse_hip_fp8_quantize(const void* x_dev, int dtype, int T, int K, void* values_dev, void* scales_dev, void* stream) {
  SP_REQUIRE(valid_dtype(dtype), "fp8_quantize: unknown dtype %d", dtype);
  SP_REQUIRE(T >= 0 && K >= 1 && K <= kF8MaxDim, "fp8_quantize: T=%d, K=%d outside [0,..] x [1,%d]", T, K, kF8MaxDim);
  if (T == 0) return SPARSE_HIP_OK;
  SP_REQUIRE(x_dev && values_dev && scales_dev, "fp8_quantize: NULL pointer");
  SP_REQUIRE(aligned16(values_dev), "fp8_quantize: values must be 16-byte aligned");
  return f8_quantize({x_dev, T, K, values_dev, scales_dev}, {}, dtype, as_stream(stream));
}

size_t sparse_hip_fp8_linear_ws_bytes(int T, int K) {
  if (T <= 0 || K <= 0 || K > kF8MaxDim) return 0;
  return linear_ws(nullptr, T, K).bytes;
}

int sparse_hip_fp8_linear(const void* x_dev, const void* xq_dev, const void* xs_dev, int dtype, int T,
                          const sparse_hip_fp8_matrix* weight, int pow2_scales, void* out_dev, void* ws_dev, void* stream) {
  SP_REQUIRE(is_16bit(dtype), "fp8_linear: activations must be bf16 or fp16, got dtype %d", dtype);
  SP_REQUIRE(weight != nullptr, "fp8_linear: NULL weight");
  SP_REQUIRE(weight->rows >= 1 && weight->rows <= kF8MaxOut && weight->cols >= 1 && weight->cols <= kF8MaxDim,
             "fp8_linear: weight is [%d,%d], must be in [1,%d] x [1,%d]", weight->rows, weight->cols, kF8MaxOut, kF8MaxDim);
  int rc = check_matrix("fp8_linear", "weight", weight, weight->rows, weight->cols);
  if (rc != SPARSE_HIP_OK) return rc;
  SP_REQUIRE(T >= 0 && T <= kF8MaxRows, "fp8_linear: T=%d outside [0,%d]", T, static_cast<int>(kF8MaxRows));
  if (T == 0) return SPARSE_HIP_OK;
  SP_REQUIRE((x_dev != nullptr) != (xq_dev != nullptr), "fp8_linear: give x or its 8-bit rows");
  SP_REQUIRE(out_dev != nullptr, "fp8_linear: NULL output");
  hipStream_t st = as_stream(stream);
  F8Product p = {};
  int source = kF8From8;
  if (x_dev == nullptr) {
    SP_REQUIRE(xs_dev != nullptr && aligned16(xq_dev), "fp8_linear: 8-bit rows need scales and 16-byte alignment");
    p.act_s = static_cast<const uint8_t*>(xq_dev);
    p.act_ss = static_cast<const uint8_t*>(xs_dev);
  } else if (T > kF8FewRows) {
    SP_REQUIRE(ws_dev != nullptr && aligned16(ws_dev), "fp8_linear: workspace is NULL or not 16-byte aligned");
    const LinearWs w = linear_ws(ws_dev, T, weight->cols);
    rc = f8_quantize({x_dev, T, weight->cols, w.x.values, w.x.scales}, {}, dtype, st);
    if (rc != SPARSE_HIP_OK) return rc;
    p.act_s = w.x.values;
    p.act_ss = w.x.scales;
  } else {
    source = kF8From16;
    p.act_s = static_cast<const uint8_t*>(x_dev);
  }
  p.w0 = static_cast<const uint8_t*>(weight->values_dev);
  p.s0 = weight->scales_dev;
  p.w1 = p.w0;
  p.s1 = p.s0;
  p.out_s = out_dev;
  p.Ks = weight->cols;
  p.Ns = weight->rows;
  p.T = T;
  p.dtype = dtype;
  p.pow2 = pow2_scales;
  if (T <= kF8FewRows) return f8_few(p, source, false, false, true, st);
  if (!linear_tiles(T, weight->rows)) return f8_rows(p, false, false, true, st);
  return f8_tile_linear(p, tile_rows(T, 0, (weight->rows + kPfBR - 1) / kPfBR), st);
}

size_t sparse_hip_fp8_slot_bytes(int H, int I) {
  if (H <= 0 || I <= 0 || H > kF8MaxDim || I > kF8MaxDim) return 0;
  return f8_slot(H, I).bytes;
}

size_t sparse_hip_fp8_moe_ffn_ws_bytes(int T, int K, int num_experts, int num_segments, int H, int I, int Is) {
  if (T <= 0 || K <= 0 || K > SPARSE_HIP_MAX_TOPK || static_cast<int64_t>(T) * K >= kF8MaxRows) return 0;
  if (num_experts <= 0 || num_experts > SPARSE_HIP_MAX_EXPERTS || num_segments < 0 || num_segments > SPARSE_HIP_MAX_EXPERTS) return 0;
  if (H <= 0 || H > kF8MaxDim || I <= 0 || I > kF8MaxDim || Is < 0 || Is > kF8MaxDim) return 0;
  return ffn_ws(nullptr, T, K, num_experts, num_segments, H, I, Is).bytes;
}

int sparse_hip_fp8_moe_ffn(const sparse_hip_experts* experts, const void* x_dev, const void* topv_dev,
                           const int32_t* perm_dev, const int32_t* seg_offsets_dev, const sparse_hip_seglist* segs,
                           int T, int K, void* parts_dev, const sparse_hip_fp8_matrix* shared_gate_w,
                           const sparse_hip_fp8_matrix* shared_up_w, const sparse_hip_fp8_matrix* shared_down_w,
                           const void* shared_gate_dev, int pow2_scales, void* shared_dev, void* ws_dev, void* stream) {
  static const char fn[] = "fp8_moe_ffn";
  SP_REQUIRE(experts != nullptr && segs != nullptr, "%s: NULL descriptor", fn);
  const int H = experts->hidden, I = experts->inter, E = experts->num_experts, dtype = experts->dtype;
  SP_REQUIRE(is_16bit(dtype), "%s: activations must be bf16 or fp16, got dtype %d", fn, dtype);
  SP_REQUIRE(E >= 1 && E <= SPARSE_HIP_MAX_EXPERTS, "%s: E=%d outside [1,%d]", fn, E, SPARSE_HIP_MAX_EXPERTS);
  SP_REQUIRE(H > 0 && H % 64 == 0 && H <= kF8MaxDim, "%s: H=%d must be a positive multiple of 64", fn, H);
  SP_REQUIRE(I > 0 && I % 64 == 0 && I <= kF8MaxDim, "%s: I=%d must be a positive multiple of 64", fn, I);
  SP_REQUIRE(T >= 1 && K >= 1 && K <= SPARSE_HIP_MAX_TOPK, "%s: T=%d, K=%d outside [1,..] x [1,%d]", fn, T, K, SPARSE_HIP_MAX_TOPK);
  SP_REQUIRE(static_cast<int64_t>(T) * K < kF8MaxRows, "%s: T=%d, K=%d: too many rows", fn, T, K);
  SP_REQUIRE(static_cast<uint64_t>(T) * f8_padded(H) < (1ull << 32), "%s: T=%d rows of %d: too large for 32-bit offsets", fn, T, H);
  SP_REQUIRE(segs->n >= 0 && segs->n <= SPARSE_HIP_MAX_EXPERTS, "%s: segment count %d outside [0,%d]", fn, segs->n, SPARSE_HIP_MAX_EXPERTS);
  const F8Slot slot = f8_slot(H, I);
  const bool routed = segs->n > 0, shared = shared_down_w != nullptr;
  SP_REQUIRE(x_dev != nullptr, "%s: NULL x", fn);
  if (routed) {
    SP_REQUIRE(experts->slab_dev != nullptr && aligned16(experts->slab_dev), "%s: weight slab is NULL or not 16-byte aligned", fn);
    SP_REQUIRE(experts->slot_stride >= slot.bytes && experts->slot_stride % 16 == 0, "%s: slot_stride=%llu too small or not 16-byte aligned", fn,
               static_cast<unsigned long long>(experts->slot_stride));
    SP_REQUIRE(topv_dev && perm_dev && seg_offsets_dev && parts_dev, "%s: NULL pointer", fn);
    SP_REQUIRE(aligned16(parts_dev), "%s: parts must be 16-byte aligned", fn);
    if (segs->eids_dev != nullptr) {
      SP_REQUIRE(segs->count_dev != nullptr, "%s: a device segment list needs a count", fn);
      SP_REQUIRE(segs->n <= E, "%s: a device segment list of up to %d, there are %d experts", fn, segs->n, E);
    } else {
      bool seen[SPARSE_HIP_MAX_EXPERTS] = {};     // (the workspace has room for each segment's tiles once)
      for (int i = 0; i < segs->n; ++i) {
        SP_REQUIRE(segs->eids[i] >= 0 && segs->eids[i] < E && segs->slots[i] >= 0, "%s: segment %d names expert %d in slot %d", fn, i,
                   static_cast<int>(segs->eids[i]), static_cast<int>(segs->slots[i]));
        SP_REQUIRE(!seen[segs->eids[i]], "%s: expert %d is listed twice", fn, static_cast<int>(segs->eids[i]));
        seen[segs->eids[i]] = true;
      }
    }
  }
  int Is = 0;
  if (shared) {
    SP_REQUIRE(shared_gate_w && shared_up_w && shared_dev, "%s: NULL shared-expert pointer", fn);
    Is = shared_down_w->cols;
    SP_REQUIRE(Is > 0 && Is % 64 == 0 && Is <= kF8MaxDim, "%s: Is=%d must be a positive multiple of 64", fn, Is);
    int rc = check_matrix(fn, "shared gate_proj", shared_gate_w, Is, H);
    if (rc == SPARSE_HIP_OK) rc = check_matrix(fn, "shared up_proj", shared_up_w, Is, H);
    if (rc == SPARSE_HIP_OK) rc = check_matrix(fn, "shared down_proj", shared_down_w, H, Is);
    if (rc != SPARSE_HIP_OK) return rc;
    SP_REQUIRE(aligned16(shared_dev), "%s: shared output must be 16-byte aligned", fn);
  }
  if (!routed && !shared) return SPARSE_HIP_OK;
  SP_REQUIRE(ws_dev != nullptr && aligned16(ws_dev), "%s: workspace is NULL or not 16-byte aligned", fn);
  hipStream_t st = as_stream(stream);
  const FfnWs w = ffn_ws(ws_dev, T, K, E, segs->n, H, I, Is);

  // One or two tokens: rows are quantised inside the products.  More: in launches of their own, beside products
  // that stream weights; beside the tiles x only, as gate/up quantises the intermediate in its epilogue.
  const bool few = T <= kF8FewRows, tiles = ffn_tiles(T, K, E, H, I);
  const int rows_per_tile = tiles ? ffn_tile_rows(T, K, E, H, I) : 0;
  int rc = SPARSE_HIP_OK;
  PfQueues queues = {};
  if (tiles) {
    PfxMapArgs queue_args;
    queues = prefill_queue_args(experts->expert_slot_dev, seg_offsets_dev, *segs, T, K, H, I, Is, w.tiles, &queue_args,
                                rows_per_tile, f8_tile_columns(rows_per_tile),
                                ffn_shared_rows(T, K, E, I, Is, rows_per_tile));
    rc = f8_quantize_and_queue({x_dev, T, H, w.x.values, nullptr}, dtype, queue_args, st);
  } else if (!few) {
    rc = f8_quantize({x_dev, T, H, w.x.values, w.x.scales}, {}, dtype, st);
  }
  if (rc != SPARSE_HIP_OK) return rc;
  F8Product p = {};
  p.slab = static_cast<const uint8_t*>(experts->slab_dev);
  p.slot_stride = experts->slot_stride;
  p.expert_slot = experts->expert_slot_dev;
  p.perm = perm_dev;
  p.seg_offsets = seg_offsets_dev;
  p.topv = topv_dev;
  p.topk = K;
  p.T = T;
  p.dtype = dtype;
  p.pow2 = pow2_scales;
  p.segs = *segs;
  // gate and up: x -> h
  p.off0 = 0;
  p.off1 = slot.up;
  p.soff0 = slot.sgate;
  p.soff1 = slot.sup;
  p.act_r = p.act_s = few ? static_cast<const uint8_t*>(x_dev) : w.x.values;
  p.act_rs = p.act_ss = w.x.scales;
  p.gather = 1;
  p.out_r = w.hf;
  p.Kr = H;
  p.Nr = I;
  if (shared) {
    p.w0 = static_cast<const uint8_t*>(shared_gate_w->values_dev);
    p.w1 = static_cast<const uint8_t*>(shared_up_w->values_dev);
    p.s0 = shared_gate_w->scales_dev;
    p.s1 = shared_up_w->scales_dev;
    p.out_s = w.shf;
    p.Ks = H;
    p.Ns = Is;
  }
  if (tiles) {
    rc = f8_tile_gateup(p, queues, w.h.values, w.h.scales, w.sh.values, w.sh.scales, st);
  } else if (few) {
    rc = f8_few(p, kF8From16, true, routed, shared, st);
  } else {
    rc = f8_rows(p, true, routed, shared, st);
    if (rc == SPARSE_HIP_OK)
      rc = f8_quantize({w.hf, routed ? static_cast<int64_t>(T) * K : 0, I, w.h.values, w.h.scales},
                       {w.shf, shared ? T : 0, Is, w.sh.values, w.sh.scales}, SPARSE_HIP_F32, st);
  }
  if (rc != SPARSE_HIP_OK) return rc;
  // down: h -> rows times their route weight (shared expert: times sigmoid of its gate)
  p.off0 = p.off1 = slot.down;
  p.soff0 = p.soff1 = slot.sdown;
  p.act_r = few ? reinterpret_cast<const uint8_t*>(w.hf) : w.h.values;
  p.act_rs = w.h.scales;
  p.gather = 0;
  p.out_r = parts_dev;
  p.Kr = I;
  p.Nr = H;
  if (shared) {
    p.w0 = p.w1 = static_cast<const uint8_t*>(shared_down_w->values_dev);
    p.s0 = p.s1 = shared_down_w->scales_dev;
    p.act_s = few ? reinterpret_cast<const uint8_t*>(w.shf) : w.sh.values;
    p.act_ss = w.sh.scales;
    p.gate_s = shared_gate_dev;
    p.out_s = shared_dev;
    p.Ks = Is;
    p.Ns = H;
  }
  if (tiles) return f8_tile_down(p, queues, rows_per_tile, st);
  return few ? f8_few(p, kF8From32, false, routed, shared, st) : f8_rows(p, false, routed, shared, st);
}

}  // extern "C"
