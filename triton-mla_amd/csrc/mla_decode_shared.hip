// Decode over shared prefixes (tmla_mla_decode_shared): the sequences of a
// group begin with the same pages, and those are attended to once for the
// whole group. No counterpart in the reference, whose kernels read every
// sequence's cache on their own (src/triton_mla/kernel.py:83-123).
//
// Softmax attention over a row's tokens splits at any point: with
//   lse_i = log sum_{t in part i} e^{s_t},  o_i = sum_{t in part i} e^{s_t - lse_i} v_t
// over disjoint parts i, the row's result is sum_i e^{lse_i - lse} o_i with
// lse = log sum_i e^{lse_i}. So the rows of all sequences of a group (row =
// one query token's head of one sequence) form one tall matrix against the
// group's prefix, 128 rows to a workgroup, and each sequence's rows meet only
// its own tokens behind it. Three launches:
//   1. mla_shared_plan_kernel: lengths and groups -> work items and their
//      places on the line that the workers share;
//   2. mla_partial_own_kernel<..., SharedArgs> (mla_decode.hip): the items' partials;
//   3. mla_shared_combine_kernel: the log-sum-exp merge of each row's partials.
// Reading a prefix once per 128 rows turns the cache's bytes into matrix
// work: 64 sequences of 16 heads over 32K tokens need 73 GFLOP against 38 MB
// of prefix instead of 2.4 GB.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "cdna.h"
#include "decode_common.h"
#include "host_plan.h"
#include "merge.h"

namespace tmla {

int hip_fail(hipError_t e, const char* where);

namespace {

struct PlanArgs {
  const int32_t* seqlens;
  const int32_t* prefix_lens;   // [groups], or null: prefix_len for each
  const int32_t* group_starts;  // [groups + 1], or null: one group of the whole batch
  int32_t prefix_len, groups, batch, rows_per_seq, q_len, capacity, workers;
  SharedHeader* header;
  SharedItem* items;
  SharedItem* worker_first;  // [workers]
  SharedMerge* merges;       // [batch, blocks of 128 rows]
};

// Inclusive maximum over the lanes of a wave (as wave_scan: by DPP moves); x >= 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_imax(int x) {
  return max(x, __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xF, false));
}
__device__ __forceinline__ int wave_scan_max(int x) {
  x = dpp_imax<0x111, 0xF>(x);
  x = dpp_imax<0x112, 0xF>(x);
  x = dpp_imax<0x114, 0xF>(x);
  x = dpp_imax<0x118, 0xF>(x);
  x = dpp_imax<0x142, 0xA>(x);
  return dpp_imax<0x143, 0xC>(x);
}

// Scans over the T threads of a workgroup in turns of one barrier each: a scan
// writes the sums that its predecessor did not, which every thread has read
// by the time of the scan after next.
template <int T>
struct Scanner {
  int (*sums)[T / 64];
  int turn = 0;
  // values in front of this thread (of x >= 0: sum or maximum); total of all
  template <bool MAX>
  __device__ __forceinline__ int before(int x, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int incl = MAX ? wave_scan_max(x) : wave_scan(x);
    int* s = sums[turn];
    turn ^= 1;
    if (lane == 63) s[wave] = incl;
    __syncthreads();
    int head = 0;
    total = 0;
    for (int w = 0; w < T / 64; ++w) {
      const int v = s[w];
      if (w < wave) head = MAX ? max(head, v) : head + v;
      total = MAX ? max(total, v) : total + v;
    }
    return MAX ? max(head, incl) : head + incl - x;  // (MAX: with this thread)
  }
};

// Last index i of the ascending a[0..n] with a[i] <= x (a[0] <= x).
template <class F>
__device__ __forceinline__ int last_at_most(F&& a, int n, int x) {
  int lo = 0, hi = n + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a(mid) <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One workgroup makes the plan: what it costs is its chain of loads and
// barriers, so the lengths and bounds are loaded at once and everything else
// stays in LDS (SMALL), four waves. 64 sequences of one group: PLAN_US us. Calls
// beyond kSharedSmall... keep lengths and items in memory, with 16 waves.
template <bool SMALL>
__global__ __launch_bounds__(SMALL ? 256 : 1024) void mla_shared_plan_kernel(PlanArgs p) {
  constexpr int T = SMALL ? 256 : 1024;
  constexpr int GROUPS = SMALL ? kSharedSmallBatch : kSharedMaxGroups;
  __shared__ int s_start[GROUPS + 1];  // first sequence of each group, ascending
  __shared__ int s_tiles[GROUPS];      // prefix tokens, then prefix tiles of each group
  __shared__ int s_first[GROUPS];      // the group's first sequence that holds a token
  __shared__ int s_base[GROUPS + 1];   // its first prefix item
  __shared__ int s_sums[2][T / 64];
  __shared__ int s_len[SMALL ? kSharedSmallBatch : 1];
  __shared__ int s_pos[SMALL ? kSharedSmallItems : 1], s_mid[SMALL ? kSharedSmallItems : 1];
  const int tid = threadIdx.x, G = p.groups, R = p.rows_per_seq;
  Scanner<T> scan{s_sums};
  int total;
  // Groups: bounds that are out of order or out of the batch leave groups
  // shorter or empty, never overlapping.
  auto bound = [&](int g) {
    return min(max(p.group_starts ? p.group_starts[g] : (g == 0 ? 0 : p.batch), 0), p.batch);
  };
  auto prefix = [&](int g) { return max(p.prefix_lens ? p.prefix_lens[g] : p.prefix_len, 0); };
  auto load_length = [&](int b) { return min(p.seqlens[b], p.capacity); };
  auto length = [&](int b) {
    if constexpr (SMALL) return s_len[b];
    else return load_length(b);
  };
  const int first_prefix = tid < G ? prefix(tid) : 0;
  if constexpr (SMALL) {
    if (tid < p.batch) s_len[tid] = load_length(tid);
    s_first[tid] = INT32_MAX;
  }
  int carry = 0;
  for (int g0 = 0; g0 <= G; g0 += T) {
    const int g = g0 + tid;
    const int v = max(scan.template before<true>(g <= G ? bound(g) : 0, total), carry);
    if (g <= G) s_start[g] = v;
    carry = max(carry, total);
  }
  for (int g = tid; g < G; g += T) {
    s_tiles[g] = g == tid ? first_prefix : prefix(g);
    if constexpr (!SMALL) s_first[g] = INT32_MAX;
  }
  __syncthreads();
  // No row of a group may see fewer tokens than its prefix (but for sequences
  // that hold nothing, whose rows no prefix partial counts for).
  auto group_of = [&](int b) {
    const int g = last_at_most([&](int i) { return s_start[i]; }, G, b);
    return g < G && b >= s_start[0] ? g : -1;
  };
  for (int b = tid; b < p.batch; b += T) {
    const int n = length(b), g = group_of(b);
    if (g >= 0 && n > 0) {
      atomicMin(&s_tiles[g], max(n - (p.q_len - 1), 0));
      atomicMin(&s_first[g], b);
    }
  }
  __syncthreads();
  int n_prefix = 0;
  for (int g0 = 0; g0 < G; g0 += T) {
    const int g = g0 + tid;
    int blocks = 0;
    if (g < G) {
      // whole tiles (what is left of the prefix each sequence reads itself),
      // of groups that have somebody to share with
      const int n = s_start[g + 1] - s_start[g];
      const int tiles = n < 2 || s_first[g] == INT32_MAX ? 0 : s_tiles[g] / kTileTokens;
      s_tiles[g] = tiles;
      if (tiles > 0) blocks = (n * R + kSharedRows - 1) / kSharedRows;
    }
    const int at = scan.template before<false>(blocks, total) + n_prefix;
    if (g < G) s_base[g] = at;
    n_prefix += total;
  }
  if (tid == 0) s_base[G] = n_prefix;
  __syncthreads();
  // items and their positions on the line
  const int per_seq = (R + kSharedRows - 1) / kSharedRows;
  const int n_items = n_prefix + p.batch * per_seq;
  struct Place {
    int row0, rows, seq, tile0, tiles, len;
  };
  auto place = [&](int i) {
    Place x;
    if (i < n_prefix) {
      const int g = last_at_most([&](int j) { return s_base[j]; }, G - 1, i);
      const int lo = (i - s_base[g]) * kSharedRows;
      x.row0 = s_start[g] * R + lo;
      x.rows = min(kSharedRows, (s_start[g + 1] - s_start[g]) * R - lo);
      x.seq = s_first[g];
      x.tile0 = 0;
      x.tiles = s_tiles[g];
      x.len = x.tiles * kTileTokens;
    } else {
      x.seq = (i - n_prefix) / per_seq;
      const int lo = (i - n_prefix - x.seq * per_seq) * kSharedRows;
      const int g = group_of(x.seq);
      x.row0 = x.seq * R + lo;
      x.rows = min(kSharedRows, R - lo);
      x.len = length(x.seq);
      x.tile0 = g >= 0 ? s_tiles[g] : 0;
      x.tiles = max(tiles_of(x.len) - x.tile0, 0);
    }
    return x;
  };
  int line = 0;
  for (int i0 = 0; i0 < n_items; i0 += T) {
    const int i = i0 + tid;
    int span = 0;
    if (i < n_items) {
      const int tiles = place(i).tiles;
      span = tiles > 0 ? tiles + kSegCostTiles : 0;
    }
    const int pos = scan.template before<false>(span, total) + line + kSegCostTiles;
    if (i < n_items) {
      if constexpr (SMALL) s_pos[i] = pos;
      else p.items[i].pos = pos;
    }
    line += total;
  }
  const int chunk = max((line + p.workers - 1) / p.workers, 1);
  if (tid == 0) *p.header = SharedHeader{n_items, chunk, line};
  auto pos_of = [&](int i) {
    if constexpr (SMALL) return s_pos[i];
    else return p.items[i].pos;
  };
  auto pieces_of = [&](int pos, int tiles) { return tiles > 0 ? (pos + tiles - 1) / chunk - pos / chunk + 1 : 0; };
  int rows_line = 0;
  for (int i0 = 0; i0 < n_items; i0 += T) {
    const int i = i0 + tid;
    Place x{};
    int pos = 0, pieces = 0;
    if (i < n_items) {  // (pos: this thread's own)
      x = place(i);
      pos = pos_of(i);
      pieces = pieces_of(pos, x.tiles);
    }
    const int mid = scan.template before<false>(pieces * x.rows, total) + rows_line;
    if (i < n_items) {
      SharedItem* it = p.items + i;
      it->row0 = x.row0;
      it->rows = x.rows;
      it->seq = x.seq;
      it->tile0 = x.tile0;
      it->tiles = x.tiles;
      it->len = x.len;
      it->causal = i >= n_prefix;
      it->pos = pos;
      it->first_worker = pos / chunk;
      it->pieces = pieces;
      it->mid_row = mid;
      it->index = i;
      if constexpr (SMALL) s_mid[i] = mid;
    }
    rows_line += total;
  }
  if constexpr (!SMALL) __threadfence();  // the items, for the other waves
  __syncthreads();
  auto mid_of = [&](int i) {
    if constexpr (SMALL) return s_mid[i];
    else return p.items[i].mid_row;
  };
  // the item that each worker's range begins in: the last whose positions
  // (with those before its first tile) begin at or before it
  for (int w = tid; w < p.workers; w += T) {
    const int lo = w * chunk;
    if (lo >= line) break;
    const int i = last_at_most([&](int j) { return pos_of(j) - kSegCostTiles; }, n_items - 1, lo);
    const Place x = place(i);
    SharedItem* it = p.worker_first + w;
    const int pos = pos_of(i);
    it->row0 = x.row0;
    it->rows = x.rows;
    it->seq = x.seq;
    it->tile0 = x.tile0;
    it->tiles = x.tiles;
    it->len = x.len;
    it->causal = i >= n_prefix;
    it->pos = pos;
    it->first_worker = pos / chunk;
    it->mid_row = mid_of(i);
    it->index = i;
  }
  // where each block of rows finds its partials
  for (int i = n_prefix + tid; i < n_items; i += T) {
    const Place x = place(i);
    const int g = group_of(x.seq);
    SharedMerge m{};
    m.own_row = mid_of(i);
    m.own_rows = x.rows;
    m.own_pieces = pieces_of(pos_of(i), x.tiles);
    m.split = kSharedRows;
    if (g >= 0 && s_tiles[g] > 0 && x.len > 0) {
      const int row = x.row0 - s_start[g] * R, at = row % kSharedRows;
      for (int k = 0; k < 2; ++k) {
        const int j = s_base[g] + row / kSharedRows + k;
        if (k == 1) {
          m.split = kSharedRows - at;
          if (m.split >= x.rows) break;
        }
        const Place y = place(j);
        m.rows[k] = y.rows;
        m.pieces[k] = pieces_of(pos_of(j), y.tiles);
        m.row[k] = mid_of(j) + (k == 0 ? at : -m.split);
      }
    }
    p.merges[i - n_prefix] = m;
  }
}

struct SharedCombineArgs {
  const SharedMerge* merges;
  const short* mid_o;
  const float* mid_lse;
  int32_t rows_per_seq;
  char* out;
  int64_t out_sb, out_sh;
  float* lse;
};

// One row of the output per wave: its partials of the group's prefix, then
// those of the sequence's own tokens, merged in that order. What bounds it is
// the chain record -> partials, two memory round trips, so the rows of the
// first partials are requested beside their lse values.
template <int DT>
__global__ __launch_bounds__(256) void mla_shared_combine_kernel(SharedCombineArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x, R = a.rows_per_seq;
  const int head = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + wave);
  if (head >= R) return;
  const SharedMerge m = a.merges[(int64_t)b * ((R + kSharedRows - 1) / kSharedRows) + head / kSharedRows];
  const int h = head % kSharedRows, k = h >= m.split;
  const int np = m.pieces[k], count = np + m.own_pieces;
  const int p0 = m.row[k] + h, ps = m.rows[k], s0 = m.own_row + h, ss = m.own_rows;
  auto row_of = [&](int j) { return (int64_t)(j < np ? p0 + j * ps : s0 + (j - np) * ss); };
  const MergeView mv{a.mid_o, a.mid_lse, R, a.out, a.out_sb, a.out_sh, a.lse};
  if (count == 0) {
    merge_zero(mv, b, head, lane);
    return;
  }
  const PlainLoads ld{a.mid_o, a.mid_lse};
  constexpr int NR = 16;  // rows in flight
  float top = 0.0f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, wsum = 0.0f;
  for (int j0 = 0; j0 < count; j0 += NR) {
    i16x8 v[NR];
    const float lv = ld.lse(row_of(min(j0 + lane % NR, count - 1)));
#pragma unroll
    for (int j = 0; j < NR; ++j) v[j] = ld.rowv(row_of(min(j0 + j, count - 1)), lane);
    if (j0 == 0) {
      float x = lv;  // (lanes past the last partial repeat it)
      for (int j = NR + lane; j < count; j += 64) x = fmaxf(x, ld.lse(row_of(j)));
      top = group_max<64>(x);
      if (top == -INFINITY) top = 0.0f;
    }
    const float w = j0 + lane % NR < count ? fast_exp2(lv - top) : 0.0f;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const float wj = lane_value(w, j);
      wsum += wj;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += wj * Elt<DT>::to_float(v[j][e]);
    }
  }
  merge_store<DT>(mv, b, head, acc, wsum, top, lane);
}

}  // namespace
}  // namespace tmla

using namespace tmla;

extern "C" {

size_t tmla_shared_workspace_bytes(int32_t batch, int32_t num_heads, int32_t num_groups, int32_t num_workers) {
  return shared_ws(batch, num_heads, num_groups, num_workers).total;
}

int tmla_mla_decode_shared(const void* q, int64_t q_stride_b, int64_t q_stride_h, const void* kv, int64_t kv_stride_0,
                           int64_t kv_stride_1, int64_t num_blocks, int32_t page_size, const float* kv_scale,
                           int64_t scale_stride_0, const int32_t* block_table,
                           int64_t bt_stride_b, int32_t bt_cols, const int32_t* cache_seqlens,
                           const int32_t* prefix_lens, int32_t prefix_len, const int32_t* group_starts,
                           int32_t num_groups, int32_t batch, int32_t q_len, int32_t num_heads, int32_t head_dim_v,
                           int32_t rope_dim, int32_t dtype, float softmax_scale, int32_t num_workers, void* out,
                           int64_t out_stride_b, int64_t out_stride_h, float* lse, void* workspace,
                           size_t workspace_bytes, void* stream) {
  const SharedCall c{batch, q_len, num_heads, num_groups, num_workers, head_dim_v, rope_dim, dtype,
                     page_size, bt_cols, num_blocks, kv_stride_1};
  const int rc = check_shared(c, workspace, workspace_bytes);
  if (rc != TMLA_OK) return rc;
  if (batch == 0) return TMLA_OK;
  if (!q || !kv || !block_table || !cache_seqlens || !out) return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  if (!group_starts && num_groups != 1)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "group_starts may be NULL for one group only");
  if (((uintptr_t)q | (uintptr_t)kv | (uintptr_t)out | (uintptr_t)workspace) & 15)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "q, kv, out and workspace must be 16-byte aligned");
  if ((q_stride_b | q_stride_h | kv_stride_0 | kv_stride_1 | out_stride_b | out_stride_h) & 7)
    return fail(TMLA_ERR_INVALID_ARGUMENT, "strides must be multiples of 8 elements");

  const bool fp8 = kv_scale != nullptr;
  if (fp8) {
    if (((uintptr_t)kv_scale & 3) || ((kv_stride_0 | kv_stride_1) & 15))
      return fail(TMLA_ERR_INVALID_ARGUMENT, "kv_scale must be 4-byte aligned, fp8 cache strides multiples of 16");
    if (page_size % 32 || (page_size & (page_size - 1)))
      return fail(TMLA_ERR_UNSUPPORTED, "an fp8 cache needs pages of a power of two of at least 32 tokens");
  }
  const int32_t rows = q_len * num_heads;
  const SharedWs w = shared_ws(batch, rows, num_groups, num_workers);
  char* ws = static_cast<char*>(workspace);
  PlanArgs p{};
  p.seqlens = cache_seqlens;
  p.prefix_lens = prefix_lens;
  p.group_starts = group_starts;
  p.prefix_len = prefix_len;
  p.groups = num_groups;
  p.batch = batch;
  p.rows_per_seq = rows;
  p.q_len = q_len;
  p.capacity = shared_capacity(c);
  p.workers = num_workers;
  p.header = reinterpret_cast<SharedHeader*>(ws);
  p.items = reinterpret_cast<SharedItem*>(ws + w.items);
  p.worker_first = reinterpret_cast<SharedItem*>(ws + w.worker_first);
  p.merges = reinterpret_cast<SharedMerge*>(ws + w.merges);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool small = batch <= kSharedSmallBatch && num_groups <= kSharedSmallBatch &&
                     shared_prefix_items(batch, rows, num_groups) + shared_own_items(batch, rows) <= kSharedSmallItems;
  if (small)
    hipLaunchKernelGGL(mla_shared_plan_kernel<true>, dim3(1), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL(mla_shared_plan_kernel<false>, dim3(1), dim3(1024), 0, s, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return hip_fail(e, "mla_shared_plan_kernel launch");

  SharedArgs a{};
  a.q = static_cast<const char*>(q);
  a.q_sb = q_stride_b;
  a.q_sh = q_stride_h;
  a.kv = static_cast<const char*>(kv);
  a.kv_s0 = kv_stride_0 * (fp8 ? 1 : 2);
  a.kv_s1 = kv_stride_1 * (fp8 ? 1 : 2);
  a.num_blocks = num_blocks;
  a.max_page = (int32_t)(num_blocks - 1 < INT32_MAX ? num_blocks - 1 : INT32_MAX);
  a.page_size = page_size;
  a.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1;
  a.bt = block_table;
  a.bt_sb = bt_stride_b;
  a.bt_cols = bt_cols;
  a.seqlens = cache_seqlens;
  a.batch = batch;
  a.num_heads = rows;
  a.q_len = q_len;
  a.heads_per_token = num_heads;
  a.qk_scale_log2 = softmax_scale * kLog2e;
  if (a.qk_scale_log2 == 0.0f) a.qk_scale_log2 = 1.17549435e-38f;  // see decode_launch
  a.num_workers = num_workers;
  a.xcds = 1;
  a.mid_o = reinterpret_cast<short*>(ws + w.mid_o);
  a.mid_lse = reinterpret_cast<float*>(ws + w.mid_lse);
  a.header = p.header;
  a.items = p.items;
  a.worker_first = p.worker_first;
  const bool uni = page_size % 32 == 0 && a.page_shift >= 0;
  if (fp8) {
    a.kv_scale = kv_scale;
    a.sc_s0 = scale_stride_0;
  }
  e = launch_partial_shared(a, num_workers, dtype, uni, fp8, s);
  if (e != hipSuccess) return hip_fail(e, "stage 1 launch");

  const SharedCombineArgs ca{p.merges, a.mid_o, a.mid_lse, rows, static_cast<char*>(out), out_stride_b, out_stride_h,
                             lse};
  const dim3 grid(batch, (rows + 3) / 4);
  if (dtype == TMLA_BF16)
    hipLaunchKernelGGL(mla_shared_combine_kernel<TMLA_BF16>, grid, dim3(256), 0, s, ca);
  else
    hipLaunchKernelGGL(mla_shared_combine_kernel<TMLA_FP16>, grid, dim3(256), 0, s, ca);
  e = hipGetLastError();
  if (e != hipSuccess) return hip_fail(e, "mla_shared_combine_kernel launch");
  return TMLA_OK;
}

}  // extern "C"
