// Host-side planning of a decode call: argument checks, the workspace
// layout and the launch shape. Plain C++ with no HIP dependency, so that
// the same code is also compiled for the CPU with the address and
// undefined-behaviour sanitizers (tests/plan_sanitize.cpp).
//
// All size arithmetic is done in 64 bits and checked: a call whose
// workspace would not fit in 2^62 bytes is rejected (workspace_bytes
// returns 0 for it), so no size can wrap around to a small value.
#pragma once

#include <stddef.h>
#include <stdint.h>
#include <stdio.h>

#include "triton_mla.h"

namespace tmla {

constexpr int kTileTokens = 64;                   // planning unit (one page at page_size 64)
// Balanced partition with straddling ranges: tiles charged for the start of
// each sequence in a worker's range (its segment's start-up and finalize)
#ifndef TMLA_SEG_COST_TILES
#define TMLA_SEG_COST_TILES 2
#endif
constexpr int kSegCostTiles = TMLA_SEG_COST_TILES;
constexpr size_t kFusedCounterBytes = 256 * 1024;  // the single launch's counter block
constexpr int64_t kMaxWorkspaceBytes = (int64_t)1 << 62;

inline thread_local char g_err[512] = "no error";

inline int fail(int code, const char* msg) {
  snprintf(g_err, sizeof(g_err), "%s", msg);
  return code;
}

// Workgroups per worker along the heads (32, 64 or 128 heads each).
inline int64_t head_blocks(int32_t heads) {
  const int64_t per = heads <= 32 ? 32 : heads <= 64 ? 64 : 128;
  return ((int64_t)heads + per - 1) / per;
}

// Partial slots of a call: batch * num_splits (uniform) or num_workers +
// batch (balanced).
inline int64_t partial_slots(int32_t batch, int32_t splits, int32_t workers) {
  return splits > 0 ? (int64_t)batch * splits : (int64_t)workers + batch;
}

// Workspace of a call: partial rows [slots, H, dv] (input dtype) at offset 0,
// their base-2 lse [slots, H] (float) after them, and the fused merge's int32
// counters m_count and m_done [batch, head blocks] and flags m_flag [slots,
// head blocks] at the start of a block of fixed size (kFusedCounterBytes)
// anchored at the END of the caller's buffer (its size rounded down to 256
// bytes). Every call reserves the whole block, so no call's partials reach
// it, whatever the shapes of the calls that share the buffer: the block is
// zero-filled once, and every single launch leaves its counters at zero
// again. A call whose counters exceed the block runs as two kernels.
struct WsLayout {
  size_t o, l, part_end;  // byte offsets: partial rows, lse, end of both
  size_t cnt_bytes;       // counter block (a multiple of 256)
  size_t total;           // part_end + cnt_bytes: the bytes the call needs; 0 if too large
};

inline WsLayout ws_layout(int32_t batch, int32_t heads, int32_t dv, int32_t splits, int32_t workers) {
  WsLayout w{0, 0, 0, kFusedCounterBytes, 0};
  const int64_t slots = partial_slots(batch, splits, workers);
  if (slots < 0 || heads < 0 || dv < 0) return w;
  // rows = slots * heads, each dv * 2 bytes, all below 2^62
  if (heads > 0 && slots > kMaxWorkspaceBytes / heads) return w;
  const int64_t rows = slots * heads;
  if (rows > 0 && (int64_t)dv * 2 > kMaxWorkspaceBytes / rows) return w;
  const int64_t o_bytes = rows * dv * 2, l_bytes = rows * 4;
  auto al = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  const int64_t total = al(o_bytes) + al(l_bytes) + (int64_t)kFusedCounterBytes;
  if (total > kMaxWorkspaceBytes) return w;
  w.o = 0;
  w.l = (size_t)al(o_bytes);
  w.part_end = w.l + (size_t)al(l_bytes);
  w.total = w.part_end + w.cnt_bytes;
  return w;
}

// 0 for invalid or too large arguments
inline size_t workspace_bytes(int32_t batch, int32_t heads, int32_t dv, int32_t splits, int32_t workers) {
  if (batch < 0 || heads <= 0 || dv < 0) return 0;
  return ws_layout(batch, heads, dv, splits, workers).total;
}

// Bytes of the fused merge's counters and flags of a call whose grid has gy
// workgroups along the heads.
inline int64_t fused_counter_bytes(int32_t batch, int64_t gy, int32_t splits, int32_t workers) {
  return (2 * (int64_t)batch + partial_slots(batch, splits, workers)) * gy * 4;
}

// Workgroups along the workers: all of them for uniform splits; for the
// balanced partition no more than the 64-token tiles the call can hold
// (block-table width or dense capacity: capacity_tokens per sequence), since
// workers past them never get a range. At least 1, at most INT32_MAX.
inline int64_t worker_grid(int32_t batch, int32_t num_splits, int32_t num_workers, int64_t capacity_tokens) {
  if (num_splits > 0) {
    const int64_t w = (int64_t)batch * num_splits;
    return w < 1 ? 1 : (w > INT32_MAX ? INT32_MAX : w);
  }
  const int64_t cap = capacity_tokens > 0 ? capacity_tokens : 0;
  const int64_t tiles_per_seq = cap / kTileTokens + (cap % kTileTokens != 0);
  // batch * tiles_per_seq, saturated
  const int64_t tile_bound =
      batch > 0 && tiles_per_seq > INT64_MAX / batch ? INT64_MAX : (int64_t)(batch > 0 ? batch : 0) * tiles_per_seq;
  const int64_t w = tile_bound < num_workers ? tile_bound : num_workers;
  return w < 1 ? 1 : w;
}

// Launch shape of a decode call: blocks of 32 heads per workgroup (1, 2 or 4)
// and the grid, and whether the single launch merges in-kernel.
struct LaunchPlan {
  int nhb;
  int64_t grid_x, grid_y;
  bool fused;
};

// capacity_tokens: tokens the block table (or dense cache) can hold per
// sequence; mode as in decode_launch (1: the single launch if it fits);
// cus: compute units of the device.
inline LaunchPlan plan_launch(int32_t batch, int32_t num_heads, int32_t num_splits, int32_t num_workers,
                              int64_t capacity_tokens, size_t mid_o_bytes, int mode, int cus) {
  LaunchPlan p;
  p.nhb = num_heads <= 32 ? 1 : num_heads <= 64 ? 2 : 4;
  // When the busy workgroups would leave compute units idle, fewer heads per
  // workgroup (more, shorter workgroups: less Q to load, less MFMA work per
  // sub-tile, smaller partial rows) use them. (Halving keeps grid.x * grid.y
  // within the compute units, so it never takes a call off the single launch.)
  const int64_t heads = num_heads > 0 ? num_heads : 1;
  p.grid_x = worker_grid(batch, num_splits, num_workers, capacity_tokens);
  while (p.nhb > 1 && p.grid_x * ((heads + 16 * p.nhb - 1) / (16 * p.nhb)) <= cus) p.nhb /= 2;
  const int64_t heads_per_wg = 32 * p.nhb;
  p.grid_y = (heads + heads_per_wg - 1) / heads_per_wg;
  // The fused merge: one workgroup per compute unit at most (the kernel's LDS
  // use admits one), so that siblings normally run side by side; its
  // counters (per sequence and per slot, for each workgroup along the heads)
  // fit the workspace's counter block.
  p.fused = mode == 1 && p.grid_x * p.grid_y <= cus && mid_o_bytes < (size_t)INT32_MAX &&
            fused_counter_bytes(batch, p.grid_y, num_splits, num_workers) <= (int64_t)kFusedCounterBytes;
  return p;
}

// Launch shape of a call that runs the 16-head-group kernel (workgroups of
// 16 heads along grid.y); the single launch under the conditions of
// plan_launch.
inline LaunchPlan plan_launch_g16(int32_t batch, int32_t num_heads, int32_t num_splits, int32_t num_workers,
                                  int64_t capacity_tokens, size_t mid_o_bytes, int mode, int cus) {
  LaunchPlan p;
  p.nhb = 0;
  p.grid_x = worker_grid(batch, num_splits, num_workers, capacity_tokens);
  p.grid_y = ((int64_t)(num_heads > 0 ? num_heads : 1) + 15) / 16;
  p.fused = mode == 1 && p.grid_x * p.grid_y <= cus && mid_o_bytes < (size_t)INT32_MAX &&
            fused_counter_bytes(batch, p.grid_y, num_splits, num_workers) <= (int64_t)kFusedCounterBytes;
  return p;
}

// fp8 cache: up to this many heads the 16-head-group kernel runs (its
// workgroups stream the cache on their own); above, where pages are a power of
// two of whole 32-token sub-tiles with one scale each (or for the cache), the
// 16-bit kernel with the cache widened once per workgroup into its ring
#ifndef TMLA_FP8_GROUP_HEADS
#define TMLA_FP8_GROUP_HEADS 16
#endif
constexpr int kFp8GroupHeads = TMLA_FP8_GROUP_HEADS;
inline bool fp8_ring(int32_t heads, bool paged, int32_t page_size, int64_t scale_s1) {
  return heads > kFp8GroupHeads && paged && page_size > 0 && page_size % 32 == 0 &&
         (page_size & (page_size - 1)) == 0 && scale_s1 == 0;
}

struct Common {
  int32_t batch, heads, dv, dr, dtype, splits, workers;
};

inline int check_common(const Common& c, const void* workspace, size_t ws_bytes) {
  if (c.batch < 0 || c.heads <= 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "batch must be >= 0 and num_heads > 0");
  if (c.dtype != TMLA_BF16 && c.dtype != TMLA_FP16) return fail(TMLA_ERR_INVALID_ARGUMENT, "dtype must be TMLA_BF16 or TMLA_FP16");
  if (c.splits < 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_splits must be >= 0");
  if (c.splits == 0 && c.workers <= 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_workers must be > 0 when num_splits == 0");
  if (c.splits > 0 && (int64_t)c.batch * c.splits > INT32_MAX) return fail(TMLA_ERR_INVALID_ARGUMENT, "batch * num_splits overflows");
  if (c.dv != 512) return fail(TMLA_ERR_UNSUPPORTED, "head_dim_v must be 512");
  const size_t need = workspace_bytes(c.batch, c.heads, c.dv, c.splits, c.workers);
  if (need == 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "the call's workspace would exceed 2^62 bytes");
  if (workspace == nullptr || ws_bytes < need)
    return fail(TMLA_ERR_WORKSPACE_TOO_SMALL, "workspace is missing or smaller than tmla_workspace_bytes()");
  return TMLA_OK;
}

// ---------------------------------------------------------------------------
// The generic decode: head dims and element types outside the specialised
// kernels (any power-of-two head_dim_v in [16, 1024] and rope_dim in
// [16, 256]; bf16, fp16 or fp32), with the reference's uniform splits and
// float32 partials [batch, heads, splits, dv] plus their base-2 lse
// [batch, heads, splits].
// ---------------------------------------------------------------------------
constexpr int kGenHeads = 16;                   // heads per workgroup (4 per wave)
constexpr int kGenSmallLds = 64 * 1024;         // two workgroups per compute unit
constexpr int kGenLargeLds = 152 * 1024;        // one
constexpr int kGenProbBytes = 4 * 64 * 4 * 4;   // probabilities: [waves][tokens][4 heads] float
constexpr int kGenMaxSplits = 65535;            // grid.y of the partial kernel
constexpr int kGenMaxBatchHeads = 65535;        // grid.z of the partial kernel, grid.y of the merge

inline bool pow2_between(int64_t x, int64_t lo, int64_t hi) { return x >= lo && x <= hi && (x & (x - 1)) == 0; }
inline int elem_bytes(int32_t dtype) { return dtype == TMLA_FP32 ? 4 : 2; }

struct GenericPlan {
  int lds;    // LDS bytes of the kernel form (kGenSmallLds or kGenLargeLds)
  int tile;   // tokens staged per step: a power of two in [1, 64]
  int pitch;  // LDS bytes per staged row: the row plus 16 bytes of padding
};

// LDS of a workgroup: Q of its heads in float (64 * D bytes), the
// probabilities, and `tile` rows. The small form when it holds at least 16
// rows. Valid for dims accepted by check_generic (D <= 1280: the large form
// holds at least 8 fp32 rows beside Q).
inline GenericPlan generic_plan(int32_t dv, int32_t dr, int32_t dtype) {
  const int64_t d = (int64_t)dv + dr;
  GenericPlan p;
  p.pitch = (int)(d * elem_bytes(dtype) + 16);
  auto tile_in = [&](int lds) {
    const int64_t room = lds - 64 * d - kGenProbBytes;
    int t = 64;
    while (t > 0 && (int64_t)t * p.pitch > room) t >>= 1;
    return t;
  };
  const int small = tile_in(kGenSmallLds);
  if (small >= 16) {
    p.lds = kGenSmallLds;
    p.tile = small;
  } else {
    p.lds = kGenLargeLds;
    p.tile = tile_in(kGenLargeLds);
  }
  return p;
}

// The matrix-core form of the generic decode (bf16 / fp16, head_dim_v <= 512,
// D = head_dim_v + rope_dim <= 576): workgroups of 4 waves x 16 heads over
// 32-token steps. LDS: the rows (32 x (2D + 16) bytes), the value dims
// transposed ([dv][32 tokens], 80-byte rows), the probabilities (4 waves x
// 16 heads x 80 bytes) and Q (64 heads x (2D + 16) bytes) (the 16-byte
// paddings are kGenRowPad and kGenMP - 64). 0 when the form
// does not apply; else the LDS form (kGenMfmaSmallLds: two workgroups per
// compute unit, or kGenMfmaLargeLds).
constexpr int kGenMfmaTokens = 32;
constexpr int kGenMfmaHeads = 64;
// padding bytes of the staged rows and of the transposed rows (bank spread)
#ifndef TMLA_GEN_ROW_PAD
#define TMLA_GEN_ROW_PAD 16
#endif
#ifndef TMLA_GEN_MP_PAD
#define TMLA_GEN_MP_PAD 16
#endif
constexpr int kGenRowPad = TMLA_GEN_ROW_PAD;
constexpr int kGenMP = 2 * kGenMfmaTokens + TMLA_GEN_MP_PAD;
constexpr int kGenMfmaSmallLds = 78 * 1024;
constexpr int kGenMfmaLargeLds = 156 * 1024;

inline int64_t generic_mfma_lds_need(int32_t dv, int32_t dr) {
  const int64_t d = (int64_t)dv + dr;
  return kGenMfmaTokens * (2 * d + kGenRowPad) + (int64_t)dv * kGenMP + 4 * 16 * kGenMP +
         kGenMfmaHeads * (2 * d + kGenRowPad);
}

inline int generic_mfma_form(int32_t dv, int32_t dr, int32_t dtype) {
  if (dtype != TMLA_BF16 && dtype != TMLA_FP16) return 0;
  if (dv > 512 || (int64_t)dv + dr > 576) return 0;
  const int64_t need = generic_mfma_lds_need(dv, dr);
  return need <= kGenMfmaSmallLds ? kGenMfmaSmallLds : (need <= kGenMfmaLargeLds ? kGenMfmaLargeLds : 0);
}

// The matrix-core kernels of other dims and float32 (mla_decode_dims.hip):
// rows whose latent part is whole 128-byte blocks and whose rope part is at
// most one, read in 16-byte pieces.
inline bool dims_form(int32_t dv, int32_t dr) {
  return (dv == 64 || dv == 128 || dv == 256 || dv == 512) && (dr == 16 || dr == 32 || dr == 64);
}
// Heads per workgroup: 128 (32 per wave) in 16 bits; 16 or 32 in float32.
inline int32_t dims_heads_per_workgroup(int32_t dtype, int32_t heads) {
  return dtype != TMLA_FP32 ? 128 : heads <= 16 ? 16 : 32;
}
// Workers of the balanced partition: the workgroups that are resident at
// once (one per compute unit by their LDS; two in float32 up to 256 value
// dims), shared by the workgroups along the heads.
inline int32_t dims_workers(int32_t dv, int32_t dtype, int32_t heads, int32_t cus) {
  const int64_t per = dims_heads_per_workgroup(dtype, heads);
  const int64_t gy = ((int64_t)heads + per - 1) / per;
  const int64_t resident = (int64_t)cus * (dtype == TMLA_FP32 && dv <= 256 ? 2 : 1);
  return (int32_t)(resident / gy > 0 ? resident / gy : 1);
}
// Lengths of a generic call are cut to the cache's capacity and to this, so
// that a token index up to 128 past a sequence's end stays below 2^31.
constexpr int32_t kMaxGenericLen = INT32_MAX - 128;
// Token `ahead` tokens after `first`, or the last one before `end`; and
// whether the `n` tokens from it on all lie before `end`. In unsigned
// arithmetic: the copies of mla_decode_dims.hip run up to three 64-token steps
// past the end (first + ahead < 2^32).
constexpr int32_t token_or_last(int32_t first, uint32_t ahead, int32_t end) {
  const uint32_t t = (uint32_t)first + ahead;
  return t < (uint32_t)end ? (int32_t)t : end - 1;
}
constexpr bool tokens_before(int32_t first, uint32_t ahead, uint32_t n, int32_t end) {
  return (uint32_t)first + ahead + n <= (uint32_t)end;
}
constexpr int64_t kDimsMaxGrid = 1 << 22;  // workgroups along x (512 threads each)

// Workspace of a generic call: the float32 partial rows, then their lse
// values (both 256-byte aligned); 0 for invalid or too large arguments.
inline size_t generic_workspace_bytes(int32_t batch, int32_t heads, int32_t dv, int32_t splits) {
  if (batch < 0 || heads <= 0 || dv <= 0 || splits <= 0) return 0;
  int64_t rows = (int64_t)batch * heads;  // below 2^62
  if (rows > 0 && splits > kMaxWorkspaceBytes / rows) return 0;
  rows *= splits;
  if (rows > 0 && ((int64_t)dv + 1) * 4 > kMaxWorkspaceBytes / rows) return 0;
  auto al = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  const int64_t total = al(rows * dv * 4) + al(rows * 4) + 256;
  return total > kMaxWorkspaceBytes ? 0 : (size_t)total;
}

// Workspace of a balanced generic call: num_workers + batch slots.
inline size_t generic_balanced_workspace_bytes(int32_t batch, int32_t heads, int32_t dv, int32_t workers) {
  if (batch < 0 || workers <= 0 || batch > INT32_MAX - workers) return 0;
  return generic_workspace_bytes(batch + workers, heads, dv, 1);
}

struct GenericCall {
  int32_t batch, heads, dv, dr, dtype, splits;
  bool paged;
  int32_t page_size, bt_cols;
  int64_t num_blocks;
};

inline int check_generic(const GenericCall& c, const void* workspace, size_t ws_bytes) {
  if (c.batch < 0 || c.heads <= 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "batch must be >= 0 and num_heads > 0");
  if (c.dtype != TMLA_BF16 && c.dtype != TMLA_FP16 && c.dtype != TMLA_FP32)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "dtype must be TMLA_BF16, TMLA_FP16 or TMLA_FP32");
  if (!pow2_between(c.dv, 16, 1024) || !pow2_between(c.dr, 16, 256))
    return fail(TMLA_ERR_UNSUPPORTED,
                "head_dim_v must be a power of two in [16, 1024] and rope_dim a power of two in [16, 256]");
  if (c.splits < 1 || c.splits > kGenMaxSplits) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_splits must be in [1, 65535]");
  if (c.batch > kGenMaxBatchHeads || c.heads > kGenMaxBatchHeads)
    return fail(TMLA_ERR_UNSUPPORTED, "batch and num_heads must be at most 65535");
  if (c.paged && (c.page_size < 1 || c.bt_cols < 1 || c.num_blocks < 1))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "a paged cache needs page_size, bt_cols and num_blocks >= 1");
  if (!c.paged && (c.page_size != 1 || c.num_blocks < 0))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "a dense cache needs page_size 1 and num_blocks (its capacity) >= 0");
  const size_t need = generic_workspace_bytes(c.batch, c.heads, c.dv, c.splits);
  if (need == 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "the call's workspace would exceed 2^62 bytes");
  if (workspace == nullptr || ws_bytes < need)
    return fail(TMLA_ERR_WORKSPACE_TOO_SMALL, "workspace is missing or smaller than tmla_generic_workspace_bytes()");
  return TMLA_OK;
}

// ---------------------------------------------------------------------------
// Decode over shared prefixes (mla_decode_shared.hip)
// ---------------------------------------------------------------------------
// Positions charged for the start of an item (its rows' Q^T, the first tiles'
// way, the partials' stores), in tiles. Measured with 1 / 2 / 4 / 8: 64 x 16
// rows over 32K 104 / 94 / 94 / 93 us, fp8 with 16 x 256 rows over 8K 137 / 119 /
// 115 / 118, 6 x 192 rows over 27K 104 / 89 / 86 / 85.
constexpr int kSharedSegTiles = 4;
constexpr int kSharedMaxGroups = 4096;  // what the plan kernel's LDS holds
constexpr int kSharedMaxWorkers = 65535;
constexpr int32_t kSharedItemBytes = 64, kSharedMergeBytes = 48;
// Calls of at most so many sequences (and groups) and items are planned in LDS
constexpr int kSharedSmallBatch = 256, kSharedSmallItems = 512;

struct SharedCall {
  int32_t batch, q_len, heads, groups, workers, dv, dr, dtype, page_size, bt_cols;
  int64_t num_blocks, kv_stride_1;
};

// Work items of a call: the groups' prefixes in blocks of 128 rows (a group's
// last one may be shorter; no more groups that hold a sequence than
// sequences), and each sequence's own tokens in blocks of 128 of its rows.
inline int64_t shared_prefix_items(int64_t batch, int64_t rows, int64_t groups) {
  return batch * rows / 128 + (groups < batch ? groups : batch);
}
inline int64_t shared_own_items(int64_t batch, int64_t rows) { return batch * ((rows + 127) / 128); }

// Whether the workers make the plan themselves, in LDS.
inline bool shared_small(int64_t batch, int64_t rows, int64_t groups) {
  return batch <= kSharedSmallBatch && groups <= kSharedSmallBatch &&
         shared_prefix_items(batch, rows, groups) + shared_own_items(batch, rows) <= kSharedSmallItems;
}

// Workspace: the plan kernel's output, then the partials' lse values and the
// partials (512 fractions of 16 bits a row). Every piece of an item has the
// item's rows; there are at most workers + items pieces, those of a
// sequence's own tokens of at most min(rows, 128) rows.
struct SharedWs {
  size_t items, merges, worker_first, worker_list, mid_lse, mid_o;
  size_t total;  // 0: invalid or too large
};
inline SharedWs shared_ws(int32_t batch, int32_t rows, int32_t groups, int32_t workers) {
  SharedWs w{0, 0, 0, 0, 0, 0, 0};
  if (batch < 0 || rows <= 0 || groups <= 0 || workers <= 0) return w;
  if ((int64_t)batch * rows > INT32_MAX / 2) return w;
  const int64_t np = shared_prefix_items(batch, rows, groups), ns = shared_own_items(batch, rows);
  const int64_t mid = (workers + np) * 128 + ns * (rows < 128 ? rows : 128);
  if (mid > INT32_MAX) return w;  // row numbers are 32 bits
  auto al = [](int64_t x) { return (x + 255) & ~(int64_t)255; };
  w.items = 256;
  w.worker_first = w.items + (size_t)al((np + ns) * kSharedItemBytes);
  w.worker_list = w.worker_first + (size_t)al((int64_t)workers * kSharedItemBytes);
  w.merges = w.worker_list +
             (shared_small(batch, rows, groups) ? (size_t)al((int64_t)workers * kSharedSmallItems * kSharedItemBytes) : 0);
  w.mid_lse = w.merges + (size_t)al(ns * kSharedMergeBytes);
  w.mid_o = w.mid_lse + (size_t)al(mid * 8);  // (log-sum-exp and factor of a row)
  w.total = w.mid_o + (size_t)(mid * 1024);
  return w;
}

// Tokens the block table can name; lengths are cut to it (and kept below
// 2^31 with the sub-tiles that are looked ahead to).
inline int32_t shared_capacity(const SharedCall& c) {
  const int64_t cap = (int64_t)c.bt_cols * c.page_size;
  return (int32_t)(cap < INT32_MAX - 256 ? cap : INT32_MAX - 256);
}

inline int check_shared(const SharedCall& c, const void* workspace, size_t ws_bytes) {
  if (c.batch < 0 || c.heads <= 0 || c.q_len < 1)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "batch must be >= 0, num_heads and q_len > 0");
  if (c.dtype != TMLA_BF16 && c.dtype != TMLA_FP16) return fail(TMLA_ERR_INVALID_ARGUMENT, "dtype must be TMLA_BF16 or TMLA_FP16");
  if (c.dv != 512 || c.dr != 64) return fail(TMLA_ERR_UNSUPPORTED, "head_dim_v must be 512 and rope_dim 64");
  if (c.groups < 1) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_groups must be >= 1");
  if (c.groups > kSharedMaxGroups) return fail(TMLA_ERR_UNSUPPORTED, "num_groups must be at most 4096");
  if (c.workers < 1 || c.workers > kSharedMaxWorkers)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "num_workers must be in [1, 65535]");
  if (c.batch == 0) return TMLA_OK;
  if (c.page_size <= 0 || c.num_blocks <= 0 || c.bt_cols <= 0)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "page_size, num_blocks and bt_cols must be > 0");
  if (c.kv_stride_1 <= 0 || c.kv_stride_1 > (1 << 25))
    return fail(TMLA_ERR_UNSUPPORTED, "kv token stride must be in (0, 2^25] elements");
  const int64_t rows = (int64_t)c.q_len * c.heads;
  if (rows > 65535 * 4) return fail(TMLA_ERR_UNSUPPORTED, "q_len * num_heads must be at most 262140");
  const size_t need = shared_ws(c.batch, (int32_t)rows, c.groups, c.workers).total;
  // the line's positions are 32 bits
  const int64_t items = shared_prefix_items(c.batch, rows, c.groups) + shared_own_items(c.batch, rows);
  const int64_t tiles = (int64_t)shared_capacity(c) / kTileTokens + 1 + kSharedSegTiles;
  // (a launch has fewer than 2^32 threads along an axis)
  if (need == 0 || c.batch >= 1 << 24 || items * tiles > INT32_MAX - 2 * kSharedMaxWorkers)
    return fail(TMLA_ERR_UNSUPPORTED, "batch, heads and block-table width are too large together");
  if (workspace == nullptr || ws_bytes < need)
    return fail(TMLA_ERR_WORKSPACE_TOO_SMALL, "workspace is missing or smaller than tmla_shared_workspace_bytes()");
  return TMLA_OK;
}

// ---------------------------------------------------------------------------
// Page operations (cache_pages.hip)
// ---------------------------------------------------------------------------
constexpr int kPagesMaxChunks = 4096;
// Tables and pools that one workgroup does in LDS
constexpr int kPagesSmallRows = 1024, kPagesSmallPages = 12288, kPagesSmallEntries = 1 << 13;
constexpr int32_t kPagesMaxRows = 1 << 20;  // rows of a table

// Pages per chunk of the counts: at most 4,096 chunks of at least 1,024 pages,
// one turn of a workgroup of 256 threads with four pages each.
inline int32_t pages_chunk(int32_t pages) {
  const int64_t per = ((int64_t)pages + kPagesMaxChunks - 1) / kPagesMaxChunks;
  return (int32_t)(per < 1024 ? 1024 : (per + 1023) / 1024 * 1024);
}

// Largest unit of 16, 4, 2 or 1 bytes that address, strides and row bytes allow.
inline int32_t pages_unit(uintptr_t base, int64_t s0, int64_t s1, int64_t row_bytes) {
  const uint64_t x = (uint64_t)base | (uint64_t)s0 | (uint64_t)s1 | (uint64_t)row_bytes;
  return x % 16 == 0 ? 16 : x % 4 == 0 ? 4 : x % 2 == 0 ? 2 : 1;
}

inline int check_pool(int64_t pages, int32_t page_size, int32_t row_elems, int32_t elem_bytes, int64_t s0, int64_t s1) {
  if (pages < 1 || pages > INT32_MAX - 8192) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_pages must be in [1, 2^31 - 8193]");
  if (page_size < 1 || row_elems < 1) return fail(TMLA_ERR_INVALID_ARGUMENT, "page_size and row_elems must be > 0");
  if (elem_bytes != 1 && elem_bytes != 2 && elem_bytes != 4)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "elem_bytes must be 1, 2 or 4");
  const int64_t row = row_elems, page = (int64_t)page_size * row;  // elements
  if (page * elem_bytes > INT32_MAX) return fail(TMLA_ERR_UNSUPPORTED, "a page must be smaller than 2^31 bytes");
  // rows of a page and pages of the pool apart, or writes would meet: pages
  // one after another, or their rows dealt out in turn
  const int64_t r1 = page_size > 1 ? s1 : row, p0 = pages > 1 ? s0 : row;
  if (r1 < row || p0 < row || r1 > kMaxWorkspaceBytes / page_size || p0 > kMaxWorkspaceBytes / pages ||
      (pages > 1 && page_size > 1 && p0 < (page_size - 1) * r1 + row && r1 < (pages - 1) * p0 + row))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "pages and their rows must not overlap");
  return TMLA_OK;
}

inline int check_tables(int32_t batch, int32_t width, int64_t pages, int32_t page_size) {
  if (batch < 0 || width < 1) return fail(TMLA_ERR_INVALID_ARGUMENT, "batch must be >= 0 and the table's width > 0");
  if ((int64_t)batch * width > INT32_MAX) return fail(TMLA_ERR_UNSUPPORTED, "a table must have fewer than 2^31 entries");
  if (batch > kPagesMaxRows) return fail(TMLA_ERR_UNSUPPORTED, "batch must be at most 2^20");
  if (pages < 1 || pages > INT32_MAX - 8192) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_pages must be in [1, 2^31 - 8193]");
  if (page_size < 1) return fail(TMLA_ERR_INVALID_ARGUMENT, "page_size must be > 0");
  return TMLA_OK;
}

// Workspace: a flag, the chunks' counts, three values a row of the table,
// three lists of pages and the pairs of a copy.
struct PagesWs {
  size_t flag, chunks, rows, ids, ids2, ids3, pairs, total;  // total 0: invalid arguments
};
inline PagesWs pages_ws(int64_t pages, int32_t batch, int32_t pairs) {
  PagesWs w{0, 0, 0, 0, 0, 0, 0, 0};
  if (pages < 1 || pages > INT32_MAX || batch < 0 || pairs < 0) return w;
  auto al = [](int64_t x) { return (size_t)((x + 255) & ~(int64_t)255); };
  w.chunks = 256;
  w.rows = w.chunks + al(kPagesMaxChunks * 4);
  w.ids = w.rows + al((int64_t)batch * 12);
  w.ids2 = w.ids + al(pages * 4);
  // (also the pairs that a fork lists)
  w.ids3 = w.ids2 + al(pages * 4 > (int64_t)batch * 8 ? pages * 4 : (int64_t)batch * 8);
  w.pairs = w.ids3 + al(pages * 4);
  w.total = w.pairs + al((int64_t)pairs * 8);
  return w;
}
inline int check_pages_ws(int64_t pages, int32_t batch, int32_t pairs, const void* workspace, size_t bytes) {
  const size_t need = pages_ws(pages, batch, pairs).total;
  if (need == 0) return fail(TMLA_ERR_INVALID_ARGUMENT, "num_pages, batch and pairs must not be negative");
  if (workspace == nullptr || bytes < need)
    return fail(TMLA_ERR_WORKSPACE_TOO_SMALL, "workspace is missing or smaller than tmla_pages_workspace_bytes()");
  if ((uintptr_t)workspace & 15) return fail(TMLA_ERR_INVALID_ARGUMENT, "workspace must be 16-byte aligned");
  return TMLA_OK;
}

}  // namespace tmla
