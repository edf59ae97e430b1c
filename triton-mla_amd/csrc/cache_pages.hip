// Page operations of a latent cache (tmla_pages_*): copying pages, forking and
// ending sequences, reserving pages for the tokens to come, and compacting the
// pool. No counterpart in the reference, which reads a block table that its
// caller made (src/triton_mla/model.py:86-94 only writes rows through one).
//
// State: a block table [batch, width] of page ids (an id outside [0, pages)
// holds nothing; -1 is written for that), the sequences' lengths, and a count
// per page of the entries that hold it. A page is free when its count is not
// positive. All choices are by order (the lowest free page first, rows and
// columns in order), so equal inputs give equal results; nothing is read back
// to the host. Tables, lengths and counts are written to new arrays (a fork
// reads the old rows while it writes the new ones); the cache is written in
// place.
//
// Ranks. In a large pool the k-th free page is found without a pass of one
// workgroup over it: the first launch counts the free pages of each chunk
// while it copies the counts, and a later launch's workgroup of chunk c sums
// the counts before c and ranks its own pages. A small table and pool are done
// by one workgroup in LDS instead (pages_small_kernel). What bounds the
// operations is launches and memory round trips where little is copied, and
// the copies' bytes (each page read and written once) where much is.
#include <hip/hip_runtime.h>

#include <stdint.h>

#include "decode_common.h"
#include "host_plan.h"
#include "triton_mla.h"

namespace tmla {

int hip_fail(hipError_t e, const char* where);

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr int kCopyUnits = 4;       // units per thread and part of a page
constexpr int kFusedPairs = 256;    // copy: pairs that one launch checks and copies
constexpr int kMarkThreads = 1024;
constexpr int kCopyGrid = 8192;     // workgroups of a copy, at most
constexpr int kMaxGrid = (1 << 24) - 1;  // workgroups of a launch of kThreads: fewer than 2^32 threads

// Pages in units of `unit` bytes (16, 4, 2 or 1: what strides and alignment
// allow); strides in bytes.
struct Pool {
  char* kv;
  int64_t s0, s1;
  int32_t pages, rows, row_units, unit;
  int32_t parts;  // kThreads * kCopyUnits units each
  char* scale;    // float32, or null
  int64_t sc0, sc1;
  int32_t sc_cols;
};

// Loads that leave nothing in the caches, and ordinary stores: 4,096 pages of
// 73,728 bytes (604 MB read and written) in 100 us, 6.0 TB/s; 122 us with
// ordinary loads, 125 with both non-temporal, 102 to 151 with the stores alone.
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <class U>
__device__ __forceinline__ void copy_part_t(const Pool& p, int src, int dst, int part) {
  const char* s = p.kv + (int64_t)src * p.s0;
  char* d = p.kv + (int64_t)dst * p.s0;
  const int units = p.rows * p.row_units;
  const bool flat = p.s1 == (int64_t)p.row_units * (int64_t)sizeof(U);
  int64_t off[kCopyUnits];
  U v[kCopyUnits];
#pragma unroll
  for (int i = 0; i < kCopyUnits; ++i) {
    const int u = min((part * kCopyUnits + i) * kThreads + (int)threadIdx.x, units - 1);
    if (flat) {
      off[i] = (int64_t)u * sizeof(U);
    } else {
      const int r = u / p.row_units;
      off[i] = r * p.s1 + (int64_t)(u - r * p.row_units) * sizeof(U);
    }
    v[i] = __builtin_nontemporal_load(reinterpret_cast<const U*>(s + off[i]));
  }
#pragma unroll
  for (int i = 0; i < kCopyUnits; ++i)
    if ((part * kCopyUnits + i) * kThreads + (int)threadIdx.x < units) *reinterpret_cast<U*>(d + off[i]) = v[i];
}

// One part of page src to page dst, and with part 0 its scales. The pages
// differ.
__device__ __forceinline__ void copy_part(const Pool& p, int src, int dst, int part) {
  if (p.unit == 16) copy_part_t<u32x4>(p, src, dst, part);
  else if (p.unit == 4) copy_part_t<uint32_t>(p, src, dst, part);
  else if (p.unit == 2) copy_part_t<uint16_t>(p, src, dst, part);
  else copy_part_t<uint8_t>(p, src, dst, part);
  if (part == 0 && p.scale)
    for (int j = threadIdx.x; j < p.sc_cols; j += kThreads)
      *reinterpret_cast<float*>(p.scale + (int64_t)dst * p.sc0 + j * p.sc1) =
          *reinterpret_cast<const float*>(p.scale + (int64_t)src * p.sc0 + j * p.sc1);
}

// Four consecutive values of an array of n, on any boundary (0 past its end).
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x4a __attribute__((ext_vector_type(4), aligned(4)));
__device__ __forceinline__ i32x4a load4(const int32_t* a, int i, int n) {
  if (i + 4 <= n) return *reinterpret_cast<const i32x4a*>(a + i);
  i32x4a v = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) v[k] = a[i + k];
  return v;
}
__device__ __forceinline__ void store4(int32_t* a, int i, int n, i32x4a v) {
  if (i + 4 <= n) {
    *reinterpret_cast<i32x4a*>(a + i) = v;
    return;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (i + k < n) a[i + k] = v[k];
}

__device__ __forceinline__ bool held(int e, int pages) { return e >= 0 && e < pages; }

// Sums over a workgroup of kThreads: of every thread, and of the threads before.
__device__ __forceinline__ int block_total(int x, int* sums) {
  x = wave_total(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  int t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t += sums[w];
  return t;
}
__device__ __forceinline__ int64_t block_total64(int64_t x, int64_t* sums) {
  for (int d = 32; d >= 1; d >>= 1) x += __shfl_xor(x, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = x;
  __syncthreads();
  int64_t t = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) t += sums[w];
  return t;
}
__device__ __forceinline__ int block_before(int x, int* sums, int& total) {
  const int incl = wave_scan(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) sums[threadIdx.x >> 6] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    if (w < (int)(threadIdx.x >> 6)) before += sums[w];
    total += sums[w];
  }
  return before + incl - x;
}

// ---------------------------------------------------------------------------
// copy
// ---------------------------------------------------------------------------
// Pair i copies page src[i] to page dst[i]. Refused: an id outside the pool, a
// destination that a later pair has too, and a source that another pair
// writes (what it holds would depend on the order). A page copied onto itself
// is not written.

// Up to kFusedPairs pairs: every workgroup checks the pair it copies against
// all of them; the first one counts the refused pairs.
__global__ __launch_bounds__(kThreads) void pages_copy_few_kernel(Pool p, const int32_t* src, const int32_t* dst, int n,
                                                                  int32_t* refused) {
  __shared__ int s_src[kFusedPairs];
  __shared__ __attribute__((aligned(16))) int s_dst[kFusedPairs];
  __shared__ int s_sums[kWaves], s_last;
  const int tid = threadIdx.x;
  bool valid = false;  // of pair tid; others can have no page in common with a valid pair
  {
    int a = -1, b = -1;
    if (tid < n) {
      a = src[tid];
      b = dst[tid];
      valid = held(a, p.pages) && held(b, p.pages);
    }
    s_src[tid] = valid ? a : -1;
    s_dst[tid] = valid ? b : -1;
  }
  if (tid == 0) s_last = -1;
  __syncthreads();
  if (blockIdx.x == 0) {
    bool bad = tid < n && !valid;
    if (valid) {
      const int a = s_src[tid], b = s_dst[tid];
      int writer = -1;  // last pair that writes the source
      for (int j = 0; j < n; j += 4) {
        const i32x4 d = *reinterpret_cast<const i32x4*>(s_dst + j);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          bad |= j + k > tid && d[k] == b;
          writer = d[k] == a ? j + k : writer;
        }
      }
      bad |= writer >= 0 && s_src[writer] != s_dst[writer];
    }
    const int t = block_total(bad, s_sums);
    if (tid == 0) *refused = t;
    return;
  }
  const int i = (blockIdx.x - 1) / p.parts, part = blockIdx.x - 1 - i * p.parts;
  const int a = s_src[i], b = s_dst[i];
  if (a < 0 || a == b) return;
  if (valid && s_dst[tid] == a) atomicMax(&s_last, tid);
  if (__syncthreads_or(valid && tid > i && s_dst[tid] == b)) return;
  if (s_last >= 0 && s_src[s_last] != s_dst[s_last]) return;
  copy_part(p, a, b, part);
}

// More pairs: one workgroup checks them and lists what is to be copied. It
// sets the destinations' bits in LDS (of pools of up to kMarkBits pages): where
// no bit is met twice, no source has one, every id is in the pool and no page
// goes to itself, all pairs copy. Otherwise it marks each destination with the last pair that
// writes it; mark[page] counts only if that pair's destination is the page, as
// the other pages' marks are never initialised. (Atomics of the workgroup's
// scope: a fence for the whole device would write the L2 back.) 4,096 pairs:
// 5 us, 28 when every call marked the pool's memory.
constexpr int kMarkBits = 1 << 20;

__global__ __launch_bounds__(kMarkThreads) void pages_mark_kernel(const int32_t* src, const int32_t* dst, int n,
                                                                  int pages, int32_t* mark, int2* list,
                                                                  int32_t* refused) {
  __shared__ unsigned s_bits[kMarkBits / 32];
  __shared__ int s_refused;
  constexpr int T = kMarkThreads, PER = 4;
  const int tid = threadIdx.x;
  auto valid = [&](int a, int b) { return held(a, pages) && held(b, pages); };
  if (pages <= kMarkBits) {
    int a[PER], b[PER];  // the first pairs of this thread
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = tid + k * T;
      a[k] = i < n ? src[i] : -1;
      b[k] = i < n ? dst[i] : -1;
    }
    for (int w = tid; w < (pages + 31) / 32; w += T) s_bits[w] = 0;
    __syncthreads();
    bool bad = false;
    auto set = [&](int x, int y) {
      if (!valid(x, y) || x == y) bad = true;
      else bad |= (atomicOr(&s_bits[y / 32], 1u << (y % 32)) >> (y % 32)) & 1;
    };
    auto test = [&](int x) { bad |= held(x, pages) && (s_bits[x / 32] >> (x % 32) & 1); };
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (tid + k * T < n) set(a[k], b[k]);
    for (int i = tid + PER * T; i < n; i += T) set(src[i], dst[i]);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) test(a[k]);
    for (int i = tid + PER * T; i < n; i += T) test(src[i]);
    if (!__syncthreads_or(bad)) {
#pragma unroll
      for (int k = 0; k < PER; ++k)
        if (tid + k * T < n) list[tid + k * T] = make_int2(a[k], b[k]);
      for (int i = tid + PER * T; i < n; i += T) list[i] = make_int2(src[i], dst[i]);
      if (tid == 0) *refused = 0;
      return;
    }
  }
  if (tid == 0) s_refused = 0;
  auto store = [&](int page, int v) {
    __hip_atomic_store(&mark[page], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  auto load = [&](int page) {
    return __hip_atomic_load(&mark[page], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  };
  // this wave's memory operations are done before the others go on
  auto barrier = [&]() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };
  for (int i = tid; i < n; i += T)
    if (valid(src[i], dst[i])) store(dst[i], -1);
  barrier();
  for (int i = tid; i < n; i += T)
    if (valid(src[i], dst[i]))
      __hip_atomic_fetch_max(&mark[dst[i]], i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
  barrier();
  int bad = 0;
  for (int i = tid; i < n; i += T) {
    const int a = src[i], b = dst[i];
    bool ok = valid(a, b);
    if (ok) {
      ok = load(b) == i;
      const int m = load(a);
      if (a != b && m >= 0 && m < n) {
        const int ma = src[m], mb = dst[m];
        if (valid(ma, mb) && mb == a && ma != a) ok = false;
      }
    }
    bad += !ok;
    list[i] = ok && a != b ? make_int2(a, b) : make_int2(-1, -1);
  }
  if (bad) atomicAdd(&s_refused, bad);
  __syncthreads();
  if (tid == 0) *refused = s_refused;
}

// count: the pairs listed, if the host does not know.
__global__ __launch_bounds__(kThreads) void pages_copy_kernel(Pool p, const int2* list, int n, const int32_t* count) {
  const int64_t total = (int64_t)(count ? min(n, *count) : n) * p.parts;
  for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
    const int i = (int)(w / p.parts), part = (int)(w - (int64_t)i * p.parts);
    const int2 pair = list[i];
    if (pair.x >= 0) copy_part(p, pair.x, pair.y, part);
  }
}

// ---------------------------------------------------------------------------
// tables
// ---------------------------------------------------------------------------
struct Tables {
  const int32_t* table;
  int64_t table_s;
  int32_t* new_table;  // [batch, width], packed
  int32_t batch, width;
  const int32_t* seqlens;
  int32_t* new_seqlens;
  const int32_t* refs;
  int32_t* new_refs;
  int32_t pages, page_size;
  int32_t chunk, chunks;  // pages per chunk of the counts, chunks
  int32_t* chunk_count;   // [chunks] free pages (compact: pages in use)
  // fork: parents[batch], or (free) ended[batch] flags
  const int32_t* parents;
  const uint8_t* ended;
  int32_t* need;    // [batch] pages that the row is to be given
  int32_t* source;  // [batch] fork: page to copy into it; -2: row is its parent's first child, -1: other
  int32_t* has_child;  // [batch]
  // reserve
  const int32_t* new_tokens;
  int32_t new_tokens_all;
  int32_t* beyond;  // [batch] pages that the table has no column for
  int32_t* ids;     // [pages] the free pages taken, in order
  int32_t* missing;
};

// The counts' part of a first launch: workgroup c copies the counts of chunk c
// and counts its free (or used) pages.
template <bool USED>
__device__ __forceinline__ void count_chunk(const Tables& t, int c, int* sums) {
  const int lo = c * t.chunk, hi = min(lo + t.chunk, t.pages);
  int n = 0;
  for (int i = lo + 4 * threadIdx.x; i < hi; i += 4 * kThreads) {
    const i32x4a r = load4(t.refs, i, hi);
    if (t.new_refs) store4(t.new_refs, i, hi, r);
#pragma unroll
    for (int k = 0; k < 4; ++k) n += i + k < hi && (USED ? r[k] > 0 : r[k] <= 0);
  }
  n = block_total(n, sums);
  if (threadIdx.x == 0) t.chunk_count[c] = n;
}

// Sum of a[0..n) by a workgroup, and of a[0..before).
__device__ __forceinline__ void sums_of(const int32_t* a, int n, int before, int* sums, int& all, int& head) {
  int x = 0, y = 0;
  for (int i = threadIdx.x; i < n; i += kThreads) {
    const int v = a[i];
    x += v;
    if (i < before) y += v;
  }
  all = block_total(x, sums);
  head = block_total(y, sums);
}

// fork, first launch: workgroups [0, chunks) copy the counts, the others
// write one new row each, but for the pages it will be given.
__global__ __launch_bounds__(kThreads) void pages_fork_kernel(Tables t) {
  __shared__ int sums[kWaves];
  if ((int)blockIdx.x < t.chunks) {
    count_chunk<false>(t, blockIdx.x, sums);
    return;
  }
  const int i = blockIdx.x - t.chunks, tid = threadIdx.x;
  int p = t.parents[i];
  const bool valid = p >= 0 && p < t.batch;
  // the parent's first child keeps its last page and what it has reserved
  bool earlier = false, child = false;
  for (int j = tid; j < t.batch; j += kThreads) {
    const int pj = t.parents[j];
    earlier |= j < i && pj == p;
    child |= pj == i;
  }
  const int flags = __syncthreads_or(earlier) ? 1 : 0;
  const int is_parent = __syncthreads_or(child) ? 1 : 0;
  const bool keeper = valid && !flags;
  const int n = valid ? t.seqlens[p] : 0;
  const int full = min(max(n, 0) / t.page_size, t.width);
  const int32_t* row = t.table + (int64_t)(valid ? p : 0) * t.table_s;
  for (int j = tid; j < t.width; j += kThreads) {
    const int e = row[j];
    t.new_table[(int64_t)i * t.width + j] = valid && (keeper || j < full) && held(e, t.pages) ? e : -1;
  }
  if (tid == 0) {
    int src = -1;
    if (valid && !keeper && n > 0 && n % t.page_size && full < t.width && held(row[full], t.pages)) src = row[full];
    t.need[i] = src >= 0;
    t.source[i] = keeper ? -2 : src;
    t.has_child[i] = is_parent;
    t.new_seqlens[i] = n;
  }
}

// fork and free, second launch: the counts of rows that nobody continues and of
// rows that share another's pages. A page's count passes zero as often up as
// down, whatever the order, so the chunk's free pages come out right too.
// (The chunks' sums meet in LDS first: 3,000 atomics on three addresses took
// 20 us of a kernel of 24.)
__global__ __launch_bounds__(kThreads) void pages_fork_refs_kernel(Tables t) {
  __shared__ int s_free[kPagesMaxChunks];
  const int i = blockIdx.x, tid = threadIdx.x;
  const bool release = !t.has_child[i], share = t.source[i] != -2;
  if (!release && !share) return;
  if (t.chunk_count)
    for (int c = tid; c < t.chunks; c += kThreads) s_free[c] = 0;
  __syncthreads();
  auto add = [&](int e, int d) {
    const int old = atomicAdd(&t.new_refs[e], d);
    const int was = old <= 0, is = old + d <= 0;
    if (t.chunk_count && was != is) atomicAdd(&s_free[e / t.chunk], is - was);
  };
  if (release) {
    const int32_t* row = t.table + (int64_t)i * t.table_s;
    for (int j = tid; j < t.width; j += kThreads)
      if (held(row[j], t.pages)) add(row[j], -1);
  }
  if (share) {
    const int32_t* row = t.new_table + (int64_t)i * t.width;
    for (int j = tid; j < t.width; j += kThreads)
      if (row[j] >= 0) add(row[j], 1);
  }
  if (!t.chunk_count) return;
  __syncthreads();
  for (int c = tid; c < t.chunks; c += kThreads)
    if (s_free[c]) atomicAdd(&t.chunk_count[c], s_free[c]);
}

// How many pages are lacking: free ones for all rows' needs, columns for them.
// Also the needs of all rows and of those before `row`, the free pages before
// chunk `c`.
__device__ __forceinline__ int64_t lacking(const Tables& t, int row, int c, int& want, int& first, int& before) {
  __shared__ int sums[kWaves];
  __shared__ int64_t sums64[kWaves];
  int free;
  sums_of(t.need, t.batch, row, sums, want, first);
  sums_of(t.chunk_count, t.chunks, c, sums, free, before);
  int64_t missing = max(want - free, 0);
  if (t.beyond) {
    int64_t x = 0;
    for (int i = threadIdx.x; i < t.batch; i += kThreads) x += t.beyond[i];
    missing += block_total64(x, sums64);
  }
  return missing;
}

// The pages taken (fork and reserve): workgroup c ranks the free pages of chunk
// c and gives those among the `want` lowest a count of 1 (fork: lists them).
// Nothing is taken when there are too few.
__device__ __forceinline__ void take_chunk(const Tables& t) {
  __shared__ int sums[kWaves];
  int want, unused, before;
  const int64_t missing = lacking(t, 0, blockIdx.x, want, unused, before);
  if (blockIdx.x == 0 && threadIdx.x == 0) *t.missing = (int32_t)min(missing, (int64_t)INT32_MAX);
  if (missing > 0 || before >= want) return;
  const int lo = blockIdx.x * t.chunk, hi = min(lo + t.chunk, t.pages);
  for (int i0 = lo; i0 < hi && before < want; i0 += 4 * kThreads) {
    const int i = i0 + 4 * threadIdx.x;
    const i32x4a r = load4(t.new_refs, i, hi);
    int f = 0, n;
#pragma unroll
    for (int k = 0; k < 4; ++k) f += i + k < hi && r[k] <= 0;
    int rank = before + block_before(f, sums, n);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < hi && r[k] <= 0) {
        if (rank < want) {
          if (t.ids) t.ids[rank] = i + k;
          t.new_refs[i + k] = 1;
        }
        ++rank;
      }
    before += n;
  }
}
__global__ __launch_bounds__(kThreads) void pages_take_kernel(Tables t) { take_chunk(t); }

// fork, last launch: workgroups (row, part) copy the row's last page and
// enter it; when pages were missing, everything is put back as it was.
__global__ __launch_bounds__(kThreads) void pages_fork_copy_kernel(Tables t, Pool p) {
  __shared__ int sums[kWaves];
  const int i = blockIdx.x / p.parts, part = blockIdx.x - i * p.parts, tid = threadIdx.x;
  const int missing = *t.missing, src = t.source[i], at = t.new_seqlens[i] / t.page_size;
  int before = 0;  // pages given to the rows before
  for (int j = tid; j < i; j += kThreads) before += t.need[j];
  if (missing > 0) {
    if (part == 0) {
      for (int j = tid; j < t.width; j += kThreads)
        t.new_table[(int64_t)i * t.width + j] = t.table[(int64_t)i * t.table_s + j];
      if (tid == 0) t.new_seqlens[i] = t.seqlens[i];
    }
    for (int64_t j = (int64_t)blockIdx.x * kThreads + tid; j < t.pages; j += (int64_t)gridDim.x * kThreads)
      t.new_refs[j] = t.refs[j];
    return;
  }
  if (src < 0) return;
  const int dst = t.ids[block_total(before, sums)];
  copy_part(p, src, dst, part);
  if (part == 0 && tid == 0) t.new_table[(int64_t)i * t.width + at] = dst;
}

// free, first launch
__global__ __launch_bounds__(kThreads) void pages_free_kernel(Tables t) {
  __shared__ int sums[kWaves];
  if ((int)blockIdx.x < t.chunks) {
    count_chunk<false>(t, blockIdx.x, sums);
    return;
  }
  const int i = blockIdx.x - t.chunks;
  const bool end = t.ended[i] != 0;
  for (int j = threadIdx.x; j < t.width; j += kThreads)
    t.new_table[(int64_t)i * t.width + j] = end ? -1 : t.table[(int64_t)i * t.table_s + j];
  if (threadIdx.x == 0) {
    t.new_seqlens[i] = end ? 0 : t.seqlens[i];
    t.has_child[i] = !end;
    t.source[i] = -2;
  }
}

// reserve, first launch: workgroups [0, chunks) copy the counts, the others a
// row each and count the entries it lacks.
__device__ __forceinline__ int pages_needed(const Tables& t, int i) {
  const int64_t n = (int64_t)max(t.seqlens[i], 0) + max(t.new_tokens ? t.new_tokens[i] : t.new_tokens_all, 0);
  const int64_t pages = (n + t.page_size - 1) / t.page_size;
  return (int)(pages < INT32_MAX ? pages : INT32_MAX);
}

__global__ __launch_bounds__(kThreads) void pages_reserve_kernel(Tables t) {
  __shared__ int sums[kWaves];
  if ((int)blockIdx.x < t.chunks) {
    count_chunk<false>(t, blockIdx.x, sums);
    return;
  }
  const int i = blockIdx.x - t.chunks;
  const int want = pages_needed(t, i);
  int lack = 0;
  for (int j = threadIdx.x; j < t.width; j += kThreads) {
    const int e = t.table[(int64_t)i * t.table_s + j];
    t.new_table[(int64_t)i * t.width + j] = e;
    lack += j < want && !held(e, t.pages);
  }
  lack = block_total(lack, sums);
  if (threadIdx.x == 0) {
    t.need[i] = lack;
    t.beyond[i] = max(want - t.width, 0);
  }
}

// reserve, second launch: workgroups [0, chunks) take the pages, the others find
// those of one row each: the free pages of ranks [first, first + need), from the
// chunk that holds the first of them on (in the old counts: the new ones change
// meanwhile). Pages for 1,024 sequences from a pool of 524,288: 16.9 us, 19.9 with a
// launch between the two that lists the pages.
constexpr int kFillIds = 1024;  // pages found before they are entered

__global__ __launch_bounds__(kThreads) void pages_reserve_fill_kernel(Tables t) {
  __shared__ int sums[kWaves], s_ids[kFillIds], s_chunk, s_before;
  if ((int)blockIdx.x < t.chunks) {
    take_chunk(t);
    return;
  }
  const int row_i = blockIdx.x - t.chunks, tid = threadIdx.x;
  const int mine = t.need[row_i];
  if (mine == 0) return;
  int all, first, unused;
  if (lacking(t, row_i, 0, all, first, unused) > 0) return;
  // the chunk of the page of rank `first`, and the free pages before it
  for (int c0 = 0, head = 0; c0 < t.chunks && head <= first; c0 += kThreads) {
    const int c = c0 + tid, f = c < t.chunks ? t.chunk_count[c] : 0;
    int n;
    const int before = head + block_before(f, sums, n);
    if (before <= first && first < before + f) {
      s_chunk = c;
      s_before = before;
    }
    head += n;
  }
  __syncthreads();
  int page0 = s_chunk * t.chunk, rank = s_before;  // free pages before page0
  const int want = min(pages_needed(t, row_i), t.width);
  int32_t* row = t.new_table + (int64_t)row_i * t.width;
  int j0 = 0;
  for (int k0 = first; k0 < first + mine; k0 += kFillIds) {
    const int end = min(k0 + kFillIds, first + mine);  // ranks [k0, end) are found, then entered
    while (true) {
      const int i = page0 + 4 * tid;
      i32x4a r = {1, 1, 1, 1};
      if (i < t.pages) r = load4(t.refs, i, t.pages);
      int f = 0, n;
#pragma unroll
      for (int k = 0; k < 4; ++k) f += i + k < t.pages && r[k] <= 0;
      int at = rank + block_before(f, sums, n);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (i + k < t.pages && r[k] <= 0) {
          if (at >= k0 && at < end) s_ids[at - k0] = i + k;
          ++at;
        }
      // (the pages of a turn that a later window needs are looked at again)
      if (rank + n >= end || page0 >= t.pages - 4 * kThreads) break;
      rank += n;
      page0 += 4 * kThreads;
    }
    __syncthreads();
    // the row's entries that hold nothing, but for those filled before
    int at = k0;
    while (at < end) {
      const int j = j0 + tid;
      const bool lack = j < want && !held(row[j], t.pages);
      int n;
      const int r = at + block_before(lack, sums, n);
      if (lack && r < end) row[j] = s_ids[r - k0];
      at += n;
      if (at < end || j0 >= want) j0 += kThreads;
      if (j0 >= want) break;
    }
    __syncthreads();
  }
}

// ---------------------------------------------------------------------------
// Fork, free or reserve by one workgroup, the counts and the rows' values in
// LDS: tables of at most kPagesSmallEntries entries and pools of at most
// kPagesSmallPages pages. One launch (and the copies') instead of three or
// four: a call that reserves for 64 sequences 13.9 us instead of 19.9, a fork
// into 16 sequences 19.1 instead of 25.
// ---------------------------------------------------------------------------
enum class Op { kFork, kFree, kReserve };
constexpr int kSmallThreads = 1024;

template <Op OP>
__global__ __launch_bounds__(kSmallThreads) void pages_small_kernel(Tables t, int2* list, int32_t* listed) {
  constexpr int T = kSmallThreads;
  __shared__ int s_refs[kPagesSmallPages];
  __shared__ int s_len[kPagesSmallRows];     // length of the row's parent (reserve: entries it should hold)
  __shared__ int s_parent[kPagesSmallRows];  // -1: the row ends empty
  __shared__ int s_first[kPagesSmallRows];   // lowest child of the row
  __shared__ int s_need[kPagesSmallRows], s_rank[kPagesSmallRows];
  __shared__ int s_src[kPagesSmallRows];
  __shared__ int s_ids[kPagesSmallPages];
  __shared__ int s_sums[T / 64];
  __shared__ long long s_beyond;
  const int tid = threadIdx.x, B = t.batch, W = t.width, entries = B * W;
  auto before_of = [&](int x, int& total) {  // scan over the workgroup
    const int incl = wave_scan(x);
    __syncthreads();
    if ((tid & 63) == 63) s_sums[tid >> 6] = incl;
    __syncthreads();
    int head = 0;
    total = 0;
    for (int w = 0; w < T / 64; ++w) {
      const int v = s_sums[w];
      if (w < (tid >> 6)) head += v;
      total += v;
    }
    return head + incl - x;
  };
  if (tid == 0) s_beyond = 0;
  for (int i = 4 * tid; i < t.pages; i += 4 * T) {
    const i32x4a r = load4(t.refs, i, t.pages);
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < t.pages) s_refs[i + k] = r[k];
  }
  for (int i = tid; i < B; i += T) {
    s_first[i] = INT32_MAX;
    s_need[i] = 0;
    s_src[i] = -1;
    if constexpr (OP == Op::kFork) {
      const int p = t.parents[i];
      s_parent[i] = p >= 0 && p < B ? p : -1;
    } else if constexpr (OP == Op::kFree) {
      s_parent[i] = t.ended[i] ? -1 : i;
    } else {
      const int want = pages_needed(t, i);
      s_len[i] = min(want, W);
      if (want > W) atomicAdd(reinterpret_cast<unsigned long long*>(&s_beyond), (unsigned long long)(want - W));
    }
  }
  __syncthreads();
  if constexpr (OP != Op::kReserve) {
    for (int i = tid; i < B; i += T) {
      const int p = s_parent[i], n = p >= 0 ? t.seqlens[p] : 0;
      s_len[i] = n;
      t.new_seqlens[i] = n;
      if (p >= 0) atomicMin(&s_first[p], i);
    }
    __syncthreads();
  }
  // the rows, but for the pages they will be given
  for (int x = tid; x < entries; x += T) {
    const int i = x / W, j = x - i * W;
    if constexpr (OP == Op::kReserve) {
      const int e = t.table[(int64_t)i * t.table_s + j];
      t.new_table[x] = e;
      if (j < s_len[i] && !held(e, t.pages)) atomicAdd(&s_need[i], 1);
    } else {
      const int p = s_parent[i];
      int e = -1;
      if (p >= 0) {
        const int old = t.table[(int64_t)p * t.table_s + j];
        const bool keeper = s_first[p] == i;
        if constexpr (OP == Op::kFree) {
          e = old;
        } else if (held(old, t.pages)) {
          const int n = s_len[i], full = n > 0 ? n / t.page_size : 0;
          if (keeper || j < full) {
            e = old;
            if (!keeper) atomicAdd(&s_refs[e], 1);
          } else if (j == full && n > 0 && n % t.page_size) {
            s_src[i] = old;
            s_need[i] = 1;
          }
        }
      }
      t.new_table[x] = e;
      if (s_first[i] == INT32_MAX) {  // nobody continues row i
        const int own = t.table[(int64_t)i * t.table_s + j];
        if (held(own, t.pages)) atomicSub(&s_refs[own], 1);
      }
    }
  }
  __syncthreads();
  int want = 0, missing = 0;
  if constexpr (OP != Op::kFree) {
    for (int i0 = 0; i0 < B; i0 += T) {
      const int i = i0 + tid;
      int n;
      const int at = before_of(i < B ? s_need[i] : 0, n) + want;
      if (i < B) s_rank[i] = at;
      want += n;
    }
    // the lowest `want` free pages
    int found = 0;
    for (int i0 = 0; i0 < t.pages && found < want; i0 += 4 * T) {
      const int i = i0 + 4 * tid;
      int f = 0, n;
#pragma unroll
      for (int k = 0; k < 4; ++k) f += i + k < t.pages && s_refs[min(i + k, t.pages - 1)] <= 0;
      int rank = before_of(f, n) + found;
      if (f)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (i + k < t.pages && s_refs[i + k] <= 0) {
            if (rank < want) s_ids[rank] = i + k;
            ++rank;
          }
      found += n;
    }
    const int64_t lack = max(want - found, 0) + s_beyond;
    missing = (int)min(lack, (int64_t)INT32_MAX);
    if (tid == 0) *t.missing = missing;
    __syncthreads();
  }
  if (missing > 0) {  // everything as it was
    for (int x = tid; x < entries; x += T) t.new_table[x] = t.table[(int64_t)(x / W) * t.table_s + x % W];
    for (int i = tid; i < t.pages; i += T) t.new_refs[i] = t.refs[i];
    if constexpr (OP == Op::kFork) {
      for (int i = tid; i < B; i += T) t.new_seqlens[i] = t.seqlens[i];
      if (tid == 0) *listed = 0;
    }
    return;
  }
  if constexpr (OP != Op::kFree) {
    for (int k = tid; k < want; k += T) s_refs[s_ids[k]] = 1;
    if constexpr (OP == Op::kFork) {
      for (int i = tid; i < B; i += T)
        if (s_need[i]) {
          const int page = s_ids[s_rank[i]];
          t.new_table[(int64_t)i * W + s_len[i] / t.page_size] = page;
          list[s_rank[i]] = make_int2(s_src[i], page);
        }
      if (tid == 0) *listed = want;
    } else {
      // a wave per row, its lacking entries in order
      const int lane = tid & 63;
      for (int i = tid >> 6; i < B; i += T / 64) {
        if (s_need[i] == 0) continue;
        int rank = s_rank[i];
        for (int j0 = 0; j0 < s_len[i]; j0 += 64) {
          const int j = j0 + lane;
          const bool lack = j < s_len[i] && !held(t.table[(int64_t)i * t.table_s + j], t.pages);
          const uint64_t m = __ballot(lack);
          if (lack) t.new_table[(int64_t)i * W + j] = s_ids[rank + __popcll(m & ((1ull << lane) - 1))];
          rank += __popcll(m);
        }
      }
    }
    __syncthreads();
  }
  for (int i = 4 * tid; i < t.pages; i += 4 * T) {
    i32x4a r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = s_refs[min(i + k, t.pages - 1)];
    store4(t.new_refs, i, t.pages, r);
  }
}

// ---------------------------------------------------------------------------
// compact: with L pages in use, the k-th used page behind the first L goes to
// the k-th free one among them.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void pages_used_kernel(Tables t) {
  __shared__ int sums[kWaves];
  count_chunk<true>(t, blockIdx.x, sums);
}

// second launch: workgroup c lists the pages of chunk c that move (from) and
// those that are moved to (to), and notes a moving page's rank.
__global__ __launch_bounds__(kThreads) void pages_rank_kernel(Tables t, int32_t* from, int32_t* to, int32_t* rank_of,
                                                              int32_t* live) {
  __shared__ int sums[kWaves];
  int used, before;
  sums_of(t.chunk_count, t.chunks, blockIdx.x, sums, used, before);
  const int L = used;
  // used pages among the first L
  const int cl = L / t.chunk;
  int stay, unused;
  sums_of(t.chunk_count, min(cl, t.chunks), 0, sums, stay, unused);
  int part = 0;
  for (int i = cl * t.chunk + threadIdx.x; i < L; i += kThreads) part += t.refs[i] > 0;
  stay += block_total(part, sums);
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    live[0] = L;
    t.missing[0] = L - stay;  // pages that move
  }
  const int lo = blockIdx.x * t.chunk, hi = min(lo + t.chunk, t.pages);
  for (int i0 = lo; i0 < hi; i0 += 4 * kThreads) {
    const int i = i0 + 4 * threadIdx.x;
    const i32x4a r = load4(t.refs, i, hi);
    int u = 0, n;
#pragma unroll
    for (int k = 0; k < 4; ++k) u += i + k < hi && r[k] > 0;
    int b = before + block_before(u, sums, n);  // used pages before page i + k
    i32x4a counts = r, ranks;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool used = r[k] > 0;
      ranks[k] = -1;
      if (i + k < hi) {
        if (i + k < L) {
          if (!used) to[i + k - b] = i + k;
        } else if (used) {
          from[b - stay] = i + k;
          ranks[k] = b - stay;
          counts[k] = 0;
        }
      }
      b += used;
    }
    store4(rank_of, i, hi, ranks);
    // (the counts of the free pages among the first L come with their pages)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (i + k < hi && !(i + k < L && r[k] <= 0)) t.new_refs[i + k] = counts[k];
    before += n;
  }
}

// last launch: workgroups [0, rows) a row of the table each, the others the
// pages and their counts.
__global__ __launch_bounds__(kThreads) void pages_compact_kernel(Tables t, Pool p, const int32_t* from,
                                                                 const int32_t* to, const int32_t* rank_of,
                                                                 const int32_t* live) {
  if ((int)blockIdx.x < t.batch) {
    const int i = blockIdx.x, L = *live;
    for (int j = threadIdx.x; j < t.width; j += kThreads) {
      int e = t.table[(int64_t)i * t.table_s + j];
      if (held(e, t.pages) && e >= L) {
        const int r = rank_of[e];
        if (r >= 0) e = to[r];
      }
      t.new_table[(int64_t)i * t.width + j] = e;
    }
    return;
  }
  const int64_t total = (int64_t)*t.missing * p.parts;
  for (int64_t w = blockIdx.x - t.batch; w < total; w += gridDim.x - t.batch) {
    const int i = (int)(w / p.parts), part = (int)(w - (int64_t)i * p.parts);
    const int a = from[i], b = to[i];
    copy_part(p, a, b, part);
    if (part == 0 && threadIdx.x == 0) t.new_refs[b] = t.refs[a];
  }
}

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
int make_pool(Pool& p, void* kv, int64_t s0, int64_t s1, int64_t pages, int32_t page_size, int32_t row_elems,
              int32_t elem_bytes, float* scale, int64_t sc0, int64_t sc1, int32_t sc_cols) {
  if (!kv) return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  const int rc = check_pool(pages, page_size, row_elems, elem_bytes, s0, s1);
  if (rc != TMLA_OK) return rc;
  if (scale && (sc_cols < 1 || ((uintptr_t)scale & 3)))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "kv_scale must be 4-byte aligned with at least one column");
  p.kv = static_cast<char*>(kv);
  p.s0 = s0 * elem_bytes;
  p.s1 = s1 * elem_bytes;
  p.pages = (int32_t)pages;
  p.rows = page_size;
  p.unit = pages_unit((uintptr_t)kv, p.s0, page_size > 1 ? p.s1 : 0, (int64_t)row_elems * elem_bytes);
  p.row_units = (int32_t)((int64_t)row_elems * elem_bytes / p.unit);
  if (page_size == 1) p.s1 = (int64_t)p.row_units * p.unit;
  const int64_t units = (int64_t)page_size * p.row_units, per = kThreads * kCopyUnits;
  p.parts = (int32_t)((units + per - 1) / per);
  p.scale = reinterpret_cast<char*>(scale);
  p.sc0 = sc0 * 4;
  p.sc1 = sc1 * 4;
  p.sc_cols = sc_cols;
  return TMLA_OK;
}

void set_chunks(Tables& t) {
  t.chunk = pages_chunk(t.pages);
  t.chunks = (t.pages + t.chunk - 1) / t.chunk;
}

bool is_small(const Tables& t) {
  return t.batch > 0 && t.batch <= kPagesSmallRows && t.pages <= kPagesSmallPages &&
         (int64_t)t.batch * t.width <= kPagesSmallEntries;
}

}  // namespace
}  // namespace tmla

using namespace tmla;

#define TMLA_LAUNCHED(name)                              \
  do {                                                   \
    const hipError_t e_ = hipGetLastError();             \
    if (e_ != hipSuccess) return hip_fail(e_, name " launch"); \
  } while (0)

extern "C" {

size_t tmla_pages_workspace_bytes(int64_t num_pages, int32_t batch, int32_t pairs) {
  return pages_ws(num_pages, batch, pairs).total;
}

int tmla_pages_copy(void* kv, int64_t kv_stride_0, int64_t kv_stride_1, int64_t num_pages, int32_t page_size,
                    int32_t row_elems, int32_t elem_bytes, float* kv_scale, int64_t scale_stride_0,
                    int64_t scale_stride_1, int32_t scale_cols, const int32_t* src, const int32_t* dst, int32_t pairs,
                    int32_t* refused, void* workspace, size_t workspace_bytes, void* stream) {
  Pool p{};
  int rc = make_pool(p, kv, kv_stride_0, kv_stride_1, num_pages, page_size, row_elems, elem_bytes, kv_scale,
                     scale_stride_0, scale_stride_1, scale_cols);
  if (rc == TMLA_OK) rc = check_pages_ws(num_pages, 0, pairs, workspace, workspace_bytes);
  if (rc != TMLA_OK) return rc;
  if (!refused || (pairs > 0 && (!src || !dst))) return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (pairs <= kFusedPairs) {
    if ((int64_t)pairs * p.parts + 1 > kMaxGrid) return fail(TMLA_ERR_UNSUPPORTED, "pages of too many bytes");
    hipLaunchKernelGGL(pages_copy_few_kernel, dim3(pairs * p.parts + 1), dim3(kThreads), 0, s, p, src, dst, pairs,
                       refused);
    TMLA_LAUNCHED("pages_copy_few_kernel");
    return TMLA_OK;
  }
  const PagesWs w = pages_ws(num_pages, 0, pairs);
  char* ws = static_cast<char*>(workspace);
  int32_t* mark = reinterpret_cast<int32_t*>(ws + w.ids);
  int2* list = reinterpret_cast<int2*>(ws + w.pairs);
  hipLaunchKernelGGL(pages_mark_kernel, dim3(1), dim3(kMarkThreads), 0, s, src, dst, pairs, p.pages, mark, list,
                     refused);
  TMLA_LAUNCHED("pages_mark_kernel");
  const int64_t total = (int64_t)pairs * p.parts;
  hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)(total < kCopyGrid ? total : kCopyGrid)), dim3(kThreads), 0, s,
                     p, list, pairs, (const int32_t*)nullptr);
  TMLA_LAUNCHED("pages_copy_kernel");
  return TMLA_OK;
}

int tmla_pages_fork(void* kv, int64_t kv_stride_0, int64_t kv_stride_1, int64_t num_pages, int32_t page_size,
                    int32_t row_elems, int32_t elem_bytes, float* kv_scale, int64_t scale_stride_0,
                    int64_t scale_stride_1, int32_t scale_cols, const int32_t* table, int64_t table_stride,
                    int32_t batch, int32_t width, const int32_t* seqlens, const int32_t* refs, const int32_t* parents,
                    int32_t* new_table, int32_t* new_seqlens, int32_t* new_refs, int32_t* missing, void* workspace,
                    size_t workspace_bytes, void* stream) {
  Pool p{};
  int rc = make_pool(p, kv, kv_stride_0, kv_stride_1, num_pages, page_size, row_elems, elem_bytes, kv_scale,
                     scale_stride_0, scale_stride_1, scale_cols);
  if (rc == TMLA_OK) rc = check_tables(batch, width, num_pages, page_size);
  if (rc == TMLA_OK) rc = check_pages_ws(num_pages, batch, 0, workspace, workspace_bytes);
  if (rc != TMLA_OK) return rc;
  if (!refs || !new_refs || !missing || (batch > 0 && (!table || !seqlens || !parents || !new_table || !new_seqlens)))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  if ((int64_t)batch * p.parts > kMaxGrid) return fail(TMLA_ERR_UNSUPPORTED, "pages of too many bytes for the batch");
  const PagesWs w = pages_ws(num_pages, batch, 0);
  char* ws = static_cast<char*>(workspace);
  Tables t{};
  t.table = table;
  t.table_s = table_stride;
  t.new_table = new_table;
  t.batch = batch;
  t.width = width;
  t.seqlens = seqlens;
  t.new_seqlens = new_seqlens;
  t.refs = refs;
  t.new_refs = new_refs;
  t.pages = (int32_t)num_pages;
  t.page_size = page_size;
  set_chunks(t);
  t.chunk_count = reinterpret_cast<int32_t*>(ws + w.chunks);
  t.parents = parents;
  t.need = reinterpret_cast<int32_t*>(ws + w.rows);
  t.source = t.need + batch;
  t.has_child = t.source + batch;
  t.ids = reinterpret_cast<int32_t*>(ws + w.ids);
  t.missing = missing;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (is_small(t)) {
    int2* list = reinterpret_cast<int2*>(ws + w.ids2);
    int32_t* listed = reinterpret_cast<int32_t*>(ws + w.flag);
    hipLaunchKernelGGL(pages_small_kernel<Op::kFork>, dim3(1), dim3(kSmallThreads), 0, s, t, list, listed);
    TMLA_LAUNCHED("pages_small_kernel");
    const int64_t most = (int64_t)batch * p.parts;
    hipLaunchKernelGGL(pages_copy_kernel, dim3((unsigned)(most < kCopyGrid ? most : kCopyGrid)), dim3(kThreads), 0, s, p,
                       list, batch, listed);
    TMLA_LAUNCHED("pages_copy_kernel");
    return TMLA_OK;
  }
  hipLaunchKernelGGL(pages_fork_kernel, dim3(t.chunks + batch), dim3(kThreads), 0, s, t);
  TMLA_LAUNCHED("pages_fork_kernel");
  if (batch > 0) {
    hipLaunchKernelGGL(pages_fork_refs_kernel, dim3(batch), dim3(kThreads), 0, s, t);
    TMLA_LAUNCHED("pages_fork_refs_kernel");
  }
  hipLaunchKernelGGL(pages_take_kernel, dim3(t.chunks), dim3(kThreads), 0, s, t);
  TMLA_LAUNCHED("pages_take_kernel");
  if (batch > 0) {
    hipLaunchKernelGGL(pages_fork_copy_kernel, dim3(batch * p.parts), dim3(kThreads), 0, s, t, p);
    TMLA_LAUNCHED("pages_fork_copy_kernel");
  }
  return TMLA_OK;
}

int tmla_pages_free(const int32_t* table, int64_t table_stride, int32_t batch, int32_t width, const int32_t* seqlens,
                    const int32_t* refs, int64_t num_pages, const uint8_t* ended, int32_t* new_table,
                    int32_t* new_seqlens, int32_t* new_refs, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tables(batch, width, num_pages, 1);
  if (rc == TMLA_OK) rc = check_pages_ws(num_pages, batch, 0, workspace, workspace_bytes);
  if (rc != TMLA_OK) return rc;
  if (!refs || !new_refs || (batch > 0 && (!table || !seqlens || !ended || !new_table || !new_seqlens)))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  const PagesWs w = pages_ws(num_pages, batch, 0);
  char* ws = static_cast<char*>(workspace);
  Tables t{};
  t.table = table;
  t.table_s = table_stride;
  t.new_table = new_table;
  t.batch = batch;
  t.width = width;
  t.seqlens = seqlens;
  t.new_seqlens = new_seqlens;
  t.refs = refs;
  t.new_refs = new_refs;
  t.pages = (int32_t)num_pages;
  t.page_size = 1;
  set_chunks(t);
  t.chunk_count = reinterpret_cast<int32_t*>(ws + w.chunks);
  t.ended = ended;
  t.need = reinterpret_cast<int32_t*>(ws + w.rows);
  t.source = t.need + batch;
  t.has_child = t.source + batch;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (is_small(t)) {
    hipLaunchKernelGGL(pages_small_kernel<Op::kFree>, dim3(1), dim3(kSmallThreads), 0, s, t, (int2*)nullptr,
                       (int32_t*)nullptr);
    TMLA_LAUNCHED("pages_small_kernel");
    return TMLA_OK;
  }
  hipLaunchKernelGGL(pages_free_kernel, dim3(t.chunks + batch), dim3(kThreads), 0, s, t);
  TMLA_LAUNCHED("pages_free_kernel");
  if (batch > 0) {
    t.chunk_count = nullptr;  // nobody asks for free pages
    hipLaunchKernelGGL(pages_fork_refs_kernel, dim3(batch), dim3(kThreads), 0, s, t);
    TMLA_LAUNCHED("pages_fork_refs_kernel");
  }
  return TMLA_OK;
}

int tmla_pages_reserve(const int32_t* table, int64_t table_stride, int32_t batch, int32_t width,
                       const int32_t* seqlens, const int32_t* refs, int64_t num_pages, int32_t page_size,
                       const int32_t* new_tokens, int32_t new_tokens_all, int32_t* new_table, int32_t* new_refs,
                       int32_t* missing, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tables(batch, width, num_pages, page_size);
  if (rc == TMLA_OK) rc = check_pages_ws(num_pages, batch, 0, workspace, workspace_bytes);
  if (rc != TMLA_OK) return rc;
  if (!refs || !new_refs || !missing || (batch > 0 && (!table || !seqlens || !new_table)))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  const PagesWs w = pages_ws(num_pages, batch, 0);
  char* ws = static_cast<char*>(workspace);
  Tables t{};
  t.table = table;
  t.table_s = table_stride;
  t.new_table = new_table;
  t.batch = batch;
  t.width = width;
  t.seqlens = seqlens;
  t.refs = refs;
  t.new_refs = new_refs;
  t.pages = (int32_t)num_pages;
  t.page_size = page_size;
  set_chunks(t);
  t.chunk_count = reinterpret_cast<int32_t*>(ws + w.chunks);
  t.need = reinterpret_cast<int32_t*>(ws + w.rows);
  t.beyond = t.need + batch;
  t.new_tokens = new_tokens;
  t.new_tokens_all = new_tokens_all;
  t.missing = missing;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (is_small(t)) {
    hipLaunchKernelGGL(pages_small_kernel<Op::kReserve>, dim3(1), dim3(kSmallThreads), 0, s, t, (int2*)nullptr,
                       (int32_t*)nullptr);
    TMLA_LAUNCHED("pages_small_kernel");
    return TMLA_OK;
  }
  hipLaunchKernelGGL(pages_reserve_kernel, dim3(t.chunks + batch), dim3(kThreads), 0, s, t);
  TMLA_LAUNCHED("pages_reserve_kernel");
  hipLaunchKernelGGL(pages_reserve_fill_kernel, dim3(t.chunks + batch), dim3(kThreads), 0, s, t);
  TMLA_LAUNCHED("pages_reserve_fill_kernel");
  return TMLA_OK;
}

int tmla_pages_compact(void* kv, int64_t kv_stride_0, int64_t kv_stride_1, int64_t num_pages, int32_t page_size,
                       int32_t row_elems, int32_t elem_bytes, float* kv_scale, int64_t scale_stride_0,
                       int64_t scale_stride_1, int32_t scale_cols, const int32_t* table, int64_t table_stride,
                       int32_t batch, int32_t width, const int32_t* refs, int32_t* new_table, int32_t* new_refs,
                       int32_t* live, void* workspace, size_t workspace_bytes, void* stream) {
  Pool p{};
  int rc = make_pool(p, kv, kv_stride_0, kv_stride_1, num_pages, page_size, row_elems, elem_bytes, kv_scale,
                     scale_stride_0, scale_stride_1, scale_cols);
  if (rc == TMLA_OK) rc = check_tables(batch, width, num_pages, page_size);
  if (rc == TMLA_OK) rc = check_pages_ws(num_pages, batch, 0, workspace, workspace_bytes);
  if (rc != TMLA_OK) return rc;
  if (!refs || !new_refs || !live || (batch > 0 && (!table || !new_table)))
    return fail(TMLA_ERR_INVALID_ARGUMENT, "null pointer argument");
  const PagesWs w = pages_ws(num_pages, batch, 0);
  char* ws = static_cast<char*>(workspace);
  Tables t{};
  t.table = table;
  t.table_s = table_stride;
  t.new_table = new_table;
  t.batch = batch;
  t.width = width;
  t.refs = refs;
  t.pages = (int32_t)num_pages;
  t.page_size = page_size;
  set_chunks(t);
  t.chunk_count = reinterpret_cast<int32_t*>(ws + w.chunks);
  t.missing = reinterpret_cast<int32_t*>(ws + w.flag);
  int32_t* from = reinterpret_cast<int32_t*>(ws + w.ids);
  int32_t* to = reinterpret_cast<int32_t*>(ws + w.ids2);
  int32_t* rank_of = reinterpret_cast<int32_t*>(ws + w.ids3);
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(pages_used_kernel, dim3(t.chunks), dim3(kThreads), 0, s, t);
  TMLA_LAUNCHED("pages_used_kernel");
  t.new_refs = new_refs;
  hipLaunchKernelGGL(pages_rank_kernel, dim3(t.chunks), dim3(kThreads), 0, s, t, from, to, rank_of, live);
  TMLA_LAUNCHED("pages_rank_kernel");
  const int64_t most = (num_pages / 2 + 1) * p.parts;
  hipLaunchKernelGGL(pages_compact_kernel, dim3((unsigned)(batch + (most < kCopyGrid ? most : kCopyGrid))),
                     dim3(kThreads), 0, s, t, p, from, to, rank_of, live);
  TMLA_LAUNCHED("pages_compact_kernel");
  return TMLA_OK;
}

}  // extern "C"
