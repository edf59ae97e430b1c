// The plan of a decode over shared prefixes: lengths, prefixes and groups ->
// work items, their places on the line that the workers share, and where each
// row finds its partials. Made by one workgroup for everybody
// (mla_decode_shared.hip), or, for calls of at most kSharedSmall... sequences
// and items, by every worker's workgroup for itself (mla_decode.hip): the same
// 3 us of loads and barriers on every compute unit instead of a launch of 5.4 us
// before them.
#pragma once

#include <hip/hip_runtime.h>

#include <stdint.h>

#include "decode_common.h"

namespace tmla {

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

struct PlanPlace {
  int row0, rows, seq, tile0, tiles, len;
};

// T threads; SMALL: lengths and items' places in LDS, else in memory (p.items).
template <int T, bool SMALL>
struct SharedPlan {
  static constexpr int GROUPS = SMALL ? kSharedSmallBatch : kSharedMaxGroups;
  struct Lds {
    int start[GROUPS + 1];  // first sequence of each group, ascending
    int tiles[GROUPS];      // prefix tokens, then prefix tiles of each group
    int first[GROUPS];      // the group's first sequence that holds a token
    int base[GROUPS + 1];   // its first prefix item
    int sums[2][T / 64];
    int len[SMALL ? kSharedSmallBatch : 1];
    int pos[SMALL ? kSharedSmallItems : 1], mid[SMALL ? kSharedSmallItems : 1];
  };
  const SharedArgs& p;
  Lds& s;
  int tid, G, R, per_seq;
  int n_prefix, n_items, line, chunk;

  __device__ __forceinline__ SharedPlan(const SharedArgs& args, Lds& lds) : p(args), s(lds) {
    tid = threadIdx.x;
    G = p.groups;
    R = p.num_heads;
    per_seq = (R + kSharedRows - 1) / kSharedRows;
  }
  __device__ __forceinline__ int load_length(int b) const { return min(p.seqlens[b], p.capacity); }
  __device__ __forceinline__ int length(int b) const {
    if constexpr (SMALL) return s.len[b];
    else return load_length(b);
  }
  __device__ __forceinline__ int group_of(int b) const {
    const int g = last_at_most([&](int i) { return s.start[i]; }, G, b);
    return g < G && b >= s.start[0] ? g : -1;
  }
  // Item i, but for its place on the line.
  __device__ __forceinline__ PlanPlace place(int i) const {
    PlanPlace x;
    if (i < n_prefix) {
      const int g = last_at_most([&](int j) { return s.base[j]; }, G - 1, i);
      const int lo = (i - s.base[g]) * kSharedRows;
      x.row0 = s.start[g] * R + lo;
      x.rows = min(kSharedRows, (s.start[g + 1] - s.start[g]) * R - lo);
      x.seq = s.first[g];
      x.tile0 = 0;
      x.tiles = s.tiles[g];
      x.len = x.tiles * kTileTokens;
    } else {
      x.seq = (i - n_prefix) / per_seq;
      const int lo = (i - n_prefix - x.seq * per_seq) * kSharedRows;
      const int g = group_of(x.seq);
      x.row0 = x.seq * R + lo;
      x.rows = min(kSharedRows, R - lo);
      x.len = length(x.seq);
      x.tile0 = g >= 0 ? s.tiles[g] : 0;
      x.tiles = max(tiles_of(x.len) - x.tile0, 0);
    }
    return x;
  }
  __device__ __forceinline__ int pos_of(int i) const {
    if constexpr (SMALL) return s.pos[i];
    else return p.items[i].pos;
  }
  __device__ __forceinline__ int mid_of(int i) const {
    if constexpr (SMALL) return s.mid[i];
    else return p.items[i].mid_row;
  }
  __device__ __forceinline__ int pieces_of(int pos, int tiles) const {
    return tiles > 0 ? (pos + tiles - 1) / chunk - pos / chunk + 1 : 0;
  }
  __device__ __forceinline__ void write(SharedItem* it, int i, const PlanPlace& x, int pos, int mid) const {
    it->row0 = x.row0;
    it->rows = x.rows;
    it->seq = x.seq;
    it->tile0 = x.tile0;
    it->tiles = x.tiles;
    it->len = x.len;
    it->causal = i >= n_prefix;
    it->pos = pos;
    it->first_worker = pos / chunk;
    it->mid_row = mid;
    it->index = i;
  }
  // The item that worker w's range begins in: the last whose positions (with
  // those before its first tile) begin at or before it.
  __device__ __forceinline__ int first_item(int w) const {
    return last_at_most([&](int j) { return pos_of(j) - kSharedSegTiles; }, n_items - 1, w * chunk);
  }
  // Where the rows of own item i (i >= n_prefix) find their partials.
  __device__ __forceinline__ void write_merge(int i) const {
    const PlanPlace x = place(i);
    const int g = group_of(x.seq);
    SharedMerge m{};
    m.own_row = mid_of(i);
    m.own_rows = x.rows;
    m.own_pieces = pieces_of(pos_of(i), x.tiles);
    m.split = kSharedRows;
    if (g >= 0 && s.tiles[g] > 0 && x.len > 0) {
      const int row = x.row0 - s.start[g] * R, at = row % kSharedRows;
      for (int k = 0; k < 2; ++k) {
        const int j = s.base[g] + row / kSharedRows + k;
        if (k == 1) {
          m.split = kSharedRows - at;
          if (m.split >= x.rows) break;
        }
        const PlanPlace y = place(j);
        m.rows[k] = y.rows;
        m.pieces[k] = pieces_of(pos_of(j), y.tiles);
        m.row[k] = mid_of(j) + (k == 0 ? at : -m.split);
      }
    }
    p.merges[i - n_prefix] = m;
  }
  __device__ __forceinline__ void make() {
    Scanner<T> scan{s.sums};
    int total;
    // Groups: bounds that are out of order or out of the batch leave groups
    // shorter or empty, never overlapping.
    auto bound = [&](int g) {
      return min(max(p.group_starts ? p.group_starts[g] : (g == 0 ? 0 : p.batch), 0), p.batch);
    };
    auto prefix = [&](int g) { return max(p.prefix_lens ? p.prefix_lens[g] : p.prefix_len, 0); };
    const int first_prefix = tid < G ? prefix(tid) : 0;
    if constexpr (SMALL) {
      if (tid < p.batch) s.len[tid] = load_length(tid);
      s.first[tid] = INT32_MAX;
    }
    int carry = 0;
    for (int g0 = 0; g0 <= G; g0 += T) {
      const int g = g0 + tid;
      const int v = max(scan.template before<true>(g <= G ? bound(g) : 0, total), carry);
      if (g <= G) s.start[g] = v;
      carry = max(carry, total);
    }
    for (int g = tid; g < G; g += T) {
      s.tiles[g] = g == tid ? first_prefix : prefix(g);
      if constexpr (!SMALL) s.first[g] = INT32_MAX;
    }
    __syncthreads();
    // No row of a group may see fewer tokens than its prefix (but for sequences
    // that hold nothing, whose rows no prefix partial counts for).
    for (int b = tid; b < p.batch; b += T) {
      const int n = length(b), g = group_of(b);
      if (g >= 0 && n > 0) {
        atomicMin(&s.tiles[g], max(n - (p.q_len - 1), 0));
        atomicMin(&s.first[g], b);
      }
    }
    __syncthreads();
    n_prefix = 0;
    for (int g0 = 0; g0 < G; g0 += T) {
      const int g = g0 + tid;
      int blocks = 0;
      if (g < G) {
        // whole tiles (what is left of the prefix each sequence reads itself),
        // of groups that have somebody to share with
        const int n = s.start[g + 1] - s.start[g];
        const int tiles = n < 2 || s.first[g] == INT32_MAX ? 0 : s.tiles[g] / kTileTokens;
        s.tiles[g] = tiles;
        if (tiles > 0) blocks = (n * R + kSharedRows - 1) / kSharedRows;
      }
      const int at = scan.template before<false>(blocks, total) + n_prefix;
      if (g < G) s.base[g] = at;
      n_prefix += total;
    }
    if (tid == 0) s.base[G] = n_prefix;
    __syncthreads();
    // items and their positions on the line
    n_items = n_prefix + p.batch * per_seq;
    line = 0;
    for (int i0 = 0; i0 < n_items; i0 += T) {
      const int i = i0 + tid;
      int span = 0;
      if (i < n_items) {
        const int tiles = place(i).tiles;
        span = tiles > 0 ? tiles + kSharedSegTiles : 0;
      }
      const int pos = scan.template before<false>(span, total) + line + kSharedSegTiles;
      if (i < n_items) {
        if constexpr (SMALL) s.pos[i] = pos;
        else p.items[i].pos = pos;
      }
      line += total;
    }
    chunk = max((line + p.num_workers - 1) / p.num_workers, 1);
    int rows_line = 0;
    for (int i0 = 0; i0 < n_items; i0 += T) {
      const int i = i0 + tid;
      PlanPlace x{};
      int pos = 0, pieces = 0;
      if (i < n_items) {  // (pos: this thread's own)
        x = place(i);
        pos = pos_of(i);
        pieces = pieces_of(pos, x.tiles);
      }
      const int mid = scan.template before<false>(pieces * x.rows, total) + rows_line;
      if (i < n_items) {
        if constexpr (!SMALL) write(p.items + i, i, x, pos, mid);
        if constexpr (SMALL) s.mid[i] = mid;
      }
      rows_line += total;
    }
    if constexpr (!SMALL) __threadfence();  // the items, for the other waves
    __syncthreads();
  }
};

// A worker's way along the items of a call whose workers plan for themselves:
// its items, the first kSharedList of them in LDS, the others (where many
// sequences have little of their own behind long prefixes) in memory that only
// this worker uses.
struct SharedOwnWalk {
  int at, count;  // next item of the worker's list, and their number
  int lo, hi;     // the worker's positions
};
using SharedSmallPlan = SharedPlan<256, true>;

// Called by all 256 threads; `space` is free again when it returns. Also writes
// this worker's share of the merge records.
__device__ __forceinline__ bool shared_begin(const SharedFusedArgs& a, int worker, SharedOwnWalk& w, void* space,
                                             SharedItem* list) {
  SharedSmallPlan plan(a, *static_cast<SharedSmallPlan::Lds*>(space));
  plan.make();
  const int tid = threadIdx.x;
  w.lo = __builtin_amdgcn_readfirstlane(worker * plan.chunk);
  w.hi = __builtin_amdgcn_readfirstlane(min(w.lo + plan.chunk, plan.line));
  w.at = 0;
  w.count = 0;
  if (w.lo < w.hi) {
    const int first = plan.first_item(worker);
    // (the first item beyond the range, by its positions)
    const int end = last_at_most([&](int j) { return plan.pos_of(j) - kSharedSegTiles; }, plan.n_items - 1, w.hi - 1) + 1;
    w.count = __builtin_amdgcn_readfirstlane(end - first);
    SharedItem* more = a.worker_list + (int64_t)worker * kSharedSmallItems;
    for (int k = tid; k < w.count; k += 256)
      plan.write(k < kSharedList ? list + k : more + k, first + k, plan.place(first + k), plan.pos_of(first + k),
                 plan.mid_of(first + k));
  }
  for (int i = plan.n_prefix + worker + a.num_workers * tid; i < plan.n_items; i += a.num_workers * 256)
    plan.write_merge(i);
  __syncthreads();
  return w.lo < w.hi;
}
__device__ __forceinline__ bool shared_next(const SharedFusedArgs& a, int worker, SharedOwnWalk& w, SharedItem& item,
                                            int& b, int& n_b, int& t_start, int& t_end, const SharedItem* list) {
  const SharedItem* more = a.worker_list + (int64_t)worker * kSharedSmallItems;
  while (w.at < w.count) {
    const int k = w.at++;
    if (k < kSharedList ? shared_take(list + k, w.lo, w.hi, item, b, n_b, t_start, t_end)
                        : shared_take(more + k, w.lo, w.hi, item, b, n_b, t_start, t_end))
      return true;
  }
  return false;
}

}  // namespace tmla
