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

constexpr int kPlanThreads = 1024;

struct PlanArgs {
  const int32_t* seqlens;
  const int32_t* prefix_lens;   // [groups], or null: prefix_len for each
  const int32_t* group_starts;  // [groups + 1], or null: one group of the whole batch
  int32_t prefix_len, groups, batch, rows_per_seq, q_len, capacity, workers;
  SharedHeader* header;
  SharedItem* items;
  int32_t* worker_item;
  int2* seq_info;  // [batch]: the prefix item of the sequence's first row (-1: none), its place there
};

// Inclusive scan over the 1024 threads of a workgroup (sum, or maximum).
template <bool MAX>
__device__ __forceinline__ int block_scan(int x, int* wave_sums) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if constexpr (MAX) {
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d);
      if (lane >= d) x = max(x, y);
    }
  } else {
    x = wave_scan(x);
  }
  __syncthreads();
  if (lane == 63) wave_sums[wave] = x;
  __syncthreads();
  int before = MAX ? INT32_MIN : 0;
  for (int w = 0; w < wave; ++w) before = MAX ? max(before, wave_sums[w]) : before + wave_sums[w];
  return MAX ? max(x, before) : x + before;
}

// Last index i of the ascending a[0..n] with a[i] <= x (a[0] <= x).
__device__ __forceinline__ int last_at_most(const int* a, int n, int x) {
  int lo = 0, hi = n + 1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One workgroup: every sum below runs over the batch, its groups or the items
// (some hundreds), and what it costs is their chain of loads and barriers.
__global__ __launch_bounds__(kPlanThreads) void mla_shared_plan_kernel(PlanArgs p) {
  __shared__ int s_start[kSharedMaxGroups + 1];  // first sequence of each group, ascending
  __shared__ int s_tiles[kSharedMaxGroups];      // prefix tokens, then prefix tiles of each group
  __shared__ int s_first[kSharedMaxGroups];      // the group's first sequence that holds a token
  __shared__ int s_base[kSharedMaxGroups + 1];   // its first prefix item
  __shared__ int s_sums[kPlanThreads / 64];
  __shared__ int s_carry;
  const int tid = threadIdx.x, G = p.groups, R = p.rows_per_seq;
  // Groups: bounds that are out of order or out of the batch leave groups
  // shorter or empty, never overlapping.
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int g0 = 0; g0 <= G; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int v = 0;
    if (g <= G) v = p.group_starts ? p.group_starts[g] : (g == 0 ? 0 : p.batch);
    v = max(block_scan<true>(min(max(v, 0), p.batch), s_sums), s_carry);
    if (g <= G) s_start[g] = v;
    __syncthreads();
    if (tid == kPlanThreads - 1) s_carry = v;
    __syncthreads();
  }
  for (int g = tid; g < G; g += kPlanThreads) {
    int n = p.prefix_lens ? p.prefix_lens[g] : p.prefix_len;
    if (s_start[g + 1] - s_start[g] < 2) n = 0;  // nobody to share with
    s_tiles[g] = max(n, 0);
    s_first[g] = INT32_MAX;
  }
  __syncthreads();
  // No row of a group may see fewer tokens than its prefix (but for sequences
  // that hold nothing, whose rows no prefix partial counts for).
  auto length = [&](int b) { return min(p.seqlens[b], p.capacity); };
  auto group_of = [&](int b) {
    const int g = last_at_most(s_start, G, b);
    return g < G && b >= s_start[0] ? g : -1;
  };
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    const int n = length(b), g = group_of(b);
    if (g >= 0 && n > 0) {
      atomicMin(&s_tiles[g], max(n - (p.q_len - 1), 0));
      atomicMin(&s_first[g], b);
    }
  }
  __syncthreads();
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int g0 = 0; g0 < G; g0 += kPlanThreads) {
    const int g = g0 + tid;
    int blocks = 0;
    if (g < G) {
      // whole tiles: what is left of the prefix each sequence reads itself
      const int tiles = s_first[g] == INT32_MAX ? 0 : s_tiles[g] / kTileTokens;
      s_tiles[g] = tiles;
      if (tiles > 0) blocks = ((s_start[g + 1] - s_start[g]) * R + kSharedRows - 1) / kSharedRows;
    }
    const int incl = block_scan<false>(blocks, s_sums) + s_carry;
    if (g < G) s_base[g] = incl - blocks;
    __syncthreads();
    if (tid == kPlanThreads - 1) s_carry = incl;
    __syncthreads();
  }
  const int n_prefix = s_carry;
  if (tid == 0) s_base[G] = n_prefix;
  __syncthreads();
  for (int b = tid; b < p.batch; b += kPlanThreads) {
    const int g = group_of(b);
    int2 info = make_int2(-1, 0);
    if (g >= 0 && s_tiles[g] > 0 && length(b) > 0) {
      const int row = (b - s_start[g]) * R;
      info = make_int2(s_base[g] + row / kSharedRows, row % kSharedRows);
    }
    p.seq_info[b] = info;
  }
  // items and their positions
  const int per_seq = (R + kSharedRows - 1) / kSharedRows;
  const int n_items = n_prefix + p.batch * per_seq;
  if (tid == 0) s_carry = 0;
  __syncthreads();
  for (int i0 = 0; i0 < n_items; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int row0 = 0, rows = 0, seq = 0, tile0 = 0, tiles = 0, len = 0;
    if (i < n_prefix) {
      const int g = last_at_most(s_base, G - 1, i);
      const int lo = (i - s_base[g]) * kSharedRows;
      row0 = s_start[g] * R + lo;
      rows = min(kSharedRows, (s_start[g + 1] - s_start[g]) * R - lo);
      seq = s_first[g];
      tiles = s_tiles[g];
      len = tiles * kTileTokens;
    } else if (i < n_items) {
      seq = (i - n_prefix) / per_seq;
      const int lo = (i - n_prefix - seq * per_seq) * kSharedRows;
      const int g = group_of(seq);
      row0 = seq * R + lo;
      rows = min(kSharedRows, R - lo);
      len = length(seq);
      tile0 = g >= 0 ? s_tiles[g] : 0;
      tiles = max(tiles_of(len) - tile0, 0);
    }
    const int span = tiles > 0 ? tiles + kSegCostTiles : 0;
    const int incl = block_scan<false>(span, s_sums) + s_carry;
    if (i < n_items) {
      SharedItem* it = p.items + i;
      it->row0 = row0;
      it->rows = rows;
      it->seq = seq;
      it->tile0 = tile0;
      it->tiles = tiles;
      it->len = len;
      it->causal = i >= n_prefix;
      it->pos = incl - span + kSegCostTiles;
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) s_carry = incl;
    __syncthreads();
  }
  const int total = s_carry;
  const int chunk = max((total + p.workers - 1) / p.workers, 1);
  __syncthreads();
  if (tid == 0) {
    s_carry = 0;
    *p.header = SharedHeader{n_items, n_prefix, chunk, total};
  }
  __syncthreads();
  for (int i0 = 0; i0 < n_items; i0 += kPlanThreads) {
    const int i = i0 + tid;
    int rows = 0, pieces = 0, first = 0;
    if (i < n_items) {
      const int pos = p.items[i].pos, tiles = p.items[i].tiles;
      if (tiles > 0) {
        first = pos / chunk;
        pieces = (pos + tiles - 1) / chunk - first + 1;
        rows = pieces * p.items[i].rows;
        // the workers whose range begins in this item's positions
        for (int w = (pos - kSegCostTiles + chunk - 1) / chunk; w < first + pieces; ++w) p.worker_item[w] = i;
      }
    }
    const int incl = block_scan<false>(rows, s_sums) + s_carry;
    if (i < n_items) {
      p.items[i].first_worker = first;
      p.items[i].pieces = pieces;
      p.items[i].mid_row = incl - rows;
    }
    __syncthreads();
    if (tid == kPlanThreads - 1) s_carry = incl;
    __syncthreads();
  }
}

struct SharedCombineArgs {
  const SharedHeader* header;
  const SharedItem* items;
  const int2* seq_info;
  const short* mid_o;
  const float* mid_lse;
  int32_t batch, rows_per_seq;
  char* out;
  int64_t out_sb, out_sh;
  float* lse;
};

// One row of the output per wave: its partials of the group's prefix, then
// those of the sequence's own tokens, merged in that order. What bounds it is
// the chain info -> items -> partials, each a memory round trip.
template <int DT>
__global__ __launch_bounds__(256) void mla_shared_combine_kernel(SharedCombineArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int b = blockIdx.x, R = a.rows_per_seq;
  const int head = __builtin_amdgcn_readfirstlane(blockIdx.y * 4 + wave);
  if (head >= R) return;
  const int2 info = a.seq_info[b];
  const int n_prefix = a.header->prefix_items;
  const int per_seq = (R + kSharedRows - 1) / kSharedRows;
  const SharedItem* si = a.items + n_prefix + b * per_seq + head / kSharedRows;
  const bool shared = info.x >= 0;
  const int prow = info.y + head;
  const SharedItem* pi = shared ? a.items + info.x + prow / kSharedRows : si;
  const int ps = pi->pieces, prs = pi->rows, pm = pi->mid_row;
  const int ss = si->pieces, srs = si->rows, sm = si->mid_row;
  const int np = shared ? ps : 0;
  const int count = np + ss;
  const int p0 = pm + prow % kSharedRows, s0 = sm + head % kSharedRows;
  auto row_of = [&](int j) { return (int64_t)(j < np ? p0 + j * prs : s0 + (j - np) * srs); };
  const MergeView mv{a.mid_o, a.mid_lse, R, a.out, a.out_sb, a.out_sh, a.lse};
  if (count == 0) {
    merge_zero(mv, b, head, lane);
    return;
  }
  const PlainLoads ld{a.mid_o, a.mid_lse};
  constexpr int NR = 16;  // rows in flight
  float m = -INFINITY;
  for (int j = lane; j < count; j += 64) m = fmaxf(m, ld.lse(row_of(j)));
  m = group_max<64>(m);
  if (m == -INFINITY) m = 0.0f;
  float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, wsum = 0.0f;
  for (int j0 = 0; j0 < count; j0 += NR) {
    i16x8 v[NR];
    const int jl = min(j0 + lane % NR, count - 1);
    const float lv = ld.lse(row_of(jl));
#pragma unroll
    for (int j = 0; j < NR; ++j) v[j] = ld.rowv(row_of(min(j0 + j, count - 1)), lane);
    const float w = j0 + lane % NR < count ? fast_exp2(lv - m) : 0.0f;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      const float wj = lane_value(w, j);
      wsum += wj;
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += wj * Elt<DT>::to_float(v[j][e]);
    }
  }
  merge_store<DT>(mv, b, head, acc, wsum, m, lane);
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
  p.worker_item = reinterpret_cast<int32_t*>(ws + w.worker_item);
  p.seq_info = reinterpret_cast<int2*>(ws + w.seq_info);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(mla_shared_plan_kernel, dim3(1), dim3(kPlanThreads), 0, s, p);
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
  a.worker_item = p.worker_item;
  const bool uni = page_size % 32 == 0 && a.page_shift >= 0;
  if (fp8) {
    a.kv_scale = kv_scale;
    a.sc_s0 = scale_stride_0;
  }
  e = launch_partial_shared(a, num_workers, dtype, uni, fp8, s);
  if (e != hipSuccess) return hip_fail(e, "stage 1 launch");

  const SharedCombineArgs ca{p.header, p.items, p.seq_info, a.mid_o, a.mid_lse, batch, rows,
                             static_cast<char*>(out), out_stride_b, out_stride_h, lse};
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
