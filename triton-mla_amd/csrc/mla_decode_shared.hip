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
// its own tokens behind it. Two launches:
//   1. mla_partial_own_kernel<..., SharedFusedArgs> (mla_decode.hip; fp8 caches
//      mla_partial_kernel): every worker plans the call (shared_plan.h: lengths
//      and groups -> work items and their places on the line that the workers
//      share) and makes the partials of its part of the line;
//   2. mla_shared_combine_kernel: the log-sum-exp merge of each row's partials.
// Above 256 sequences or groups or 512 items mla_shared_plan_kernel makes the
// plan once, in a launch of its own before them (SharedArgs).
// Reading a prefix once per 128 rows turns the cache's bytes into matrix
// work: 64 sequences of 16 heads over 32K tokens need 73 GFLOP against 38 MB
// of prefix instead of 2.4 GB.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "cdna.h"
#include "decode_common.h"
#include "host_plan.h"
#include "merge.h"
#include "shared_plan.h"

namespace tmla {

int hip_fail(hipError_t e, const char* where);

namespace {

// The plan of calls too large for the workers to make it themselves.
__global__ __launch_bounds__(1024) void mla_shared_plan_kernel(SharedArgs p) {
  constexpr int T = 1024;
  using Plan = SharedPlan<T, false>;
  __shared__ Plan::Lds lds;
  Plan plan(p, lds);
  plan.make();
  const int tid = threadIdx.x;
  if (tid == 0) *p.header = SharedHeader{plan.n_items, plan.chunk, plan.line};
  for (int w = tid; w < p.num_workers && w * plan.chunk < plan.line; w += T) {
    const int i = plan.first_item(w);
    plan.write(p.worker_first + w, i, plan.place(i), plan.pos_of(i), plan.mid_of(i));
  }
  for (int i = plan.n_prefix + tid; i < plan.n_items; i += T) plan.write_merge(i);
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
  const PlainLoads ld{a.mid_o, nullptr};
  // (log-sum-exp, factor) of a row's partials
  auto lse_of = [&](int j) { return reinterpret_cast<const float2*>(a.mid_lse)[row_of(j)]; };
  constexpr int NR = 16;  // rows in flight
  float top = 0.0f, acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, wsum = 0.0f;
  for (int j0 = 0; j0 < count; j0 += NR) {
    i16x8 v[NR];
    const float2 lv = lse_of(min(j0 + lane % NR, count - 1));
#pragma unroll
    for (int j = 0; j < NR; ++j) v[j] = ld.rowv(row_of(min(j0 + j, count - 1)), lane);
    if (j0 == 0) {
      float x = lv.x;  // (lanes past the last partial repeat it)
      for (int j = NR + lane; j < count; j += 64) x = fmaxf(x, lse_of(j).x);
      top = group_max<64>(x);
      if (top == -INFINITY) top = 0.0f;
    }
    const float w = j0 + lane % NR < count ? fast_exp2(lv.x - top) : 0.0f;
    const float ws = w * lv.y;
#pragma unroll
    for (int j = 0; j < NR; ++j) {
      wsum += lane_value(w, j);
      const float wj = lane_value(ws, j);
#pragma unroll
      for (int e = 0; e < 8; ++e) acc[e] += wj * (float)v[j][e];
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
  hipStream_t s = static_cast<hipStream_t>(stream);
  SharedFusedArgs a{};
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
  a.prefix_lens = prefix_lens;
  a.group_starts = group_starts;
  a.prefix_len = prefix_len;
  a.groups = num_groups;
  a.capacity = shared_capacity(c);
  a.merges = reinterpret_cast<SharedMerge*>(ws + w.merges);
  a.header = reinterpret_cast<SharedHeader*>(ws);
  a.items = reinterpret_cast<SharedItem*>(ws + w.items);
  a.worker_first = reinterpret_cast<SharedItem*>(ws + w.worker_first);
  a.worker_list = reinterpret_cast<SharedItem*>(ws + w.worker_list);
  const bool uni = page_size % 32 == 0 && a.page_shift >= 0;
  if (fp8) {
    a.kv_scale = kv_scale;
    a.sc_s0 = scale_stride_0;
  }
  const bool fused = shared_small(batch, rows, num_groups);
  hipError_t e;
  if (!fused) {
    hipLaunchKernelGGL(mla_shared_plan_kernel, dim3(1), dim3(1024), 0, s, a);
    e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, "mla_shared_plan_kernel launch");
  }
  e = launch_partial_shared(a, dtype, uni, fp8, fused, s);
  if (e != hipSuccess) return hip_fail(e, "stage 1 launch");

  const SharedCombineArgs ca{a.merges, a.mid_o, a.mid_lse, rows, static_cast<char*>(out), out_stride_b, out_stride_h,
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
