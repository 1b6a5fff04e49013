// Page tables of the paged KV cache, built on the GPU from the requests' lengths (no reference
// counterpart: the reference grows one dense cache per layer with mx.concatenate,
// dspark_mlx/arch/qwen3.py:294-295).
//
//   dsm_paged_extend  sequence i grows from len_i by new_i tokens: have_i = ceil(len_i / P) pages
//                     become want_i = ceil((len_i + new_i) / P); the new ones come from the top of a
//                     stack of free pages, in order of sequences (off_i = sum_{j<i} want_j - have_j):
//                     table[i][have_i + k] = free[n_free - 1 - off_i - k]. Row r of the step
//                     (cu_i <= r < cu_i + new_i, cu_i = sum_{j<i} new_j) is token
//                     p = len_i + r - cu_i in slot table[i][p / P] * P + p % P.
//   dsm_paged_trim    sequence i shrinks to keep_i tokens; its surplus pages go back on the stack in
//                     the mirrored order, so a trim to the lengths before an extend restores the stack.
//
// Bound by latency: a decode step moves a few KB, a prefill step 12 bytes per row. A decode step is one
// CTA's. A prefill step goes to a cluster: every CTA scans all sequences itself (their lengths come
// from L2), then the CTAs share out the pages by flat index, each finding its sequence by
// bisection in shared memory, so that one long sequence among short ones costs no more than an
// even batch. The cluster barrier between the reads of lengths / n_free and their updates is
// what lets the update be in place: a captured step replays on the buffers it leaves behind. The rows of
// such a step are written by a second kernel on the whole GPU: 130,000 rows of 253 sequences took
// a cluster of 8 alone 21 us, of 47 with a bisection per row; extend and trim together now take 15.8 us (a decode
// step of 64 sequences 8.7 us, two launches), 0.4 us of it the look at the pages before they are handed out.
#include <cooperative_groups.h>

#include "kv8.cuh"

namespace cg = cooperative_groups;

namespace dsm {
namespace {

constexpr int kPagedThreads = 512;
constexpr int kPagedWarps = kPagedThreads / 32;
constexpr int kPagedCluster = 8;

// Exclusive scan over the CTA of one pair per thread; returns the pair's prefix, and the totals in
// `ta`, `tb`. Row counts are summed in 64 bits: the sum of unchecked lengths may pass 32.
__device__ __forceinline__ void cta_scan(int64_t& a, int& b, int64_t& ta, int& tb, int64_t (&sa)[kPagedWarps],
                                         int (&sb)[kPagedWarps]) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t a0 = a;
  const int b0 = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t x = __shfl_up_sync(0xffffffffu, a, o);
    const int y = __shfl_up_sync(0xffffffffu, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  if (lane == 31) {
    sa[warp] = a;
    sb[warp] = b;
  }
  __syncthreads();
  int64_t pa = 0;
  int pb = 0;
  ta = 0;
  tb = 0;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) {
    if (w == warp) {
      pa = ta;
      pb = tb;
    }
    ta += sa[w];
    tb += sb[w];
  }
  a = pa + a - a0;
  b = pb + b - b0;
  __syncthreads();  // sa / sb are written again by the next scan
}

// the last i in [0, n) with a[i] <= x (a ascending, a[0] <= x)
__device__ __forceinline__ int last_not_above(const int* a, int n, int x) {
  int lo = 0, hi = n;  // a[lo] <= x, and hi == n or a[hi] > x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct ExtendArgs {
  int32_t* lengths;
  const int32_t* new_len;
  int batch, page;
  int32_t* table;
  int64_t table_stride;
  int max_pages;
  const int32_t* free_pages;
  int32_t* n_free;
  int n_pages;
  int32_t* cu_rows;
  int64_t* slot_map;
  int32_t* positions;
  int64_t max_rows;
  uint32_t per_page;  // kv8_per_page
  bool rows_after;    // paged_rows_kernel follows
};
__device__ __forceinline__ int page_of(const ExtendArgs& p, int pos) {
  return p.per_page ? int(__umulhi(unsigned(pos) / kKv8Group, p.per_page)) : pos / kKv8Group;
}

// shared memory: cu [batch + 1], off [batch], len [batch] (len < 0: the sequence gets nothing)
__global__ void __launch_bounds__(kPagedThreads) paged_extend_kernel(const ExtendArgs p) {
  extern __shared__ int sm[];
  __shared__ int64_t sa[kPagedWarps];
  __shared__ int sb[kPagedWarps];
  __shared__ int used_sm, bad_sm;
  cg::cluster_group cluster = cg::this_cluster();
  int* cu = sm;
  int* off = cu + p.batch + 1;
  int* len = off + p.batch;
  const int tid = threadIdx.x;
  const int rank = int(cluster.block_rank()), ctas = int(cluster.num_blocks());
  const int free0 = min(max(*p.n_free, 0), p.n_pages);
  // The stack ends at a page outside the pool: should one be among those that are handed out, the sequences are gone
  // through once more with the pages above it.
  int avail = free0;
  bool failed = false;
  int64_t rows_before = 0;
  for (bool again = true; again;) {
    if (tid == 0) {
      used_sm = 0;
      bad_sm = 0x7fffffff;
    }
    __syncthreads();
    rows_before = 0;
    int pages_before = 0;
    failed = false;
    for (int base = 0; base < p.batch; base += kPagedThreads) {
      const int i = base + tid;
      int n0 = -1, n1 = 0, have = 0, need = 0;
      if (i < p.batch) {
        n0 = p.lengths[i];
        n1 = p.new_len[i];
        const int64_t end = int64_t(n0) + n1;
        if (n0 < 0 || n1 < 0 || end > int64_t(p.max_pages) * p.page || end > 0x7fffffff) {
          failed |= n1 != 0;
          n0 = -1;
          n1 = max(n1, 0);
        } else {
          have = int((int64_t(n0) + p.page - 1) / p.page);
          need = int((end + p.page - 1) / p.page) - have;
        }
      }
      int64_t r0 = n1;
      int p0 = need;
      int64_t rt;
      int pt;
      cta_scan(r0, p0, rt, pt, sa, sb);
      r0 += rows_before;
      p0 += pages_before;
      if (i < p.batch) {
        // once a sequence finds too few pages or rows, so does every later one that needs any: the
        // pages that are handed out stay one run from the top of the stack
        const bool fits = n0 >= 0 && r0 + n1 <= p.max_rows && (need == 0 || int64_t(p0) + need <= avail);
        failed |= !fits && n1 > 0;
        cu[i] = int(min(r0, int64_t(0x7fffffff)));
        off[i] = min(p0, avail);
        len[i] = fits ? n0 : -1;
        if (fits && need) atomicMax(&used_sm, p0 + need);
      }
      rows_before += rt;
      pages_before = int(min(int64_t(pages_before) + pt, int64_t(0x3fffffff)));
    }
    __syncthreads();
    const int taken = used_sm;
    for (int k = tid; k < taken; k += kPagedThreads) {
      const int pg = p.free_pages[free0 - 1 - k];
      if (pg < 0 || pg >= p.n_pages) atomicMin(&bad_sm, k);
    }
    __syncthreads();
    again = bad_sm < taken;
    if (again) {
      avail = bad_sm;
      if (rank == 0 && tid == 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
      __syncthreads();  // bad_sm has been read
    }
  }
  if (tid == 0) cu[p.batch] = int(min(rows_before, int64_t(0x7fffffff)));
  if (failed && rank == 0) raise_device_error(DSM_DEV_ERR_PAGES_SHORT);
  cluster.sync();  // every CTA has read lengths and n_free
  const int used = used_sm, total = cu[p.batch];
  if (rank == 0) {
    for (int i = tid; i <= p.batch; i += kPagedThreads) {
      p.cu_rows[i] = cu[i];
      if (i < p.batch && len[i] >= 0) p.lengths[i] = len[i] + (cu[i + 1] - cu[i]);
    }
    if (tid == 0) *p.n_free = free0 - used;
  }
  const int me = rank * kPagedThreads + tid, all = ctas * kPagedThreads;
  for (int k = me; k < used; k += all) {
    const int i = last_not_above(off, p.batch, k);
    const int j = (len[i] + p.page - 1) / p.page + (k - off[i]);
    p.table[int64_t(i) * p.table_stride + j] = p.free_pages[free0 - 1 - k];
  }
  // a row's slot: all rows, or each sequence's first (the others follow in paged_rows_kernel)
  const int64_t rows = p.rows_after ? p.batch : p.max_rows;
  for (int64_t x = me; x < rows; x += all) {
    const int64_t r = p.rows_after ? cu[x] : x;
    if (p.rows_after && (cu[x + 1] == r || r >= p.max_rows)) continue;
    int64_t slot = -1;
    int pos = 0;
    if (r < total) {
      const int i = p.rows_after ? int(x) : last_not_above(cu, p.batch, int(r));
      if (len[i] >= 0) {
        pos = len[i] + int(r) - cu[i];
        const int j = page_of(p, pos), have = (len[i] + p.page - 1) / p.page;
        const int pg = j < have ? p.table[int64_t(i) * p.table_stride + j] : p.free_pages[free0 - 1 - off[i] - (j - have)];
        slot = int64_t(pg) * p.page + (pos - j * p.page);
      }
    }
    p.slot_map[r] = slot;
    p.positions[r] = pos;
  }
}

// The rows of a long step, from what paged_extend_kernel has left: a sequence's rows, its new length, its table, and
// in its first row's slot whether it got what it asked for (that slot is written once more, as it is). A
// warp takes 128 neighbouring rows, finds their sequence by a 32-way search, and a lane keeps its
// sequence from row to row.
constexpr int kRowThreads = 256, kRowsPerLane = 4;

__global__ void __launch_bounds__(kRowThreads) paged_rows_kernel(const ExtendArgs p) {
  const int lane = threadIdx.x & 31;
  const int64_t first = (int64_t(blockIdx.x) * (kRowThreads / 32) + (threadIdx.x >> 5)) * (32 * kRowsPerLane);
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while paged_extend_kernel runs
  if (first >= p.max_rows) return;
  const int64_t total = p.cu_rows[p.batch];
  int i = 0;
  if (first < total) {
    for (int n = p.batch; n > 1;) {  // the last sequence that starts at or before `first` is among n from i on
      const int step = (n + 31) / 32;
      const unsigned m = __ballot_sync(0xffffffffu, lane * step < n && p.cu_rows[i + min(lane * step, n - 1)] <= first);
      const int k = 31 - __clz(m);
      i += k * step;
      n = min(step, n - k * step);
    }
  }
  int c0 = 0, c1 = 0, n0 = -1;  // the lane's sequence: its rows, its cached rows (-1: it got nothing)
  int64_t slot[kRowsPerLane];
  int pos[kRowsPerLane], at[kRowsPerLane];
  const int32_t* from[kRowsPerLane];
#pragma unroll
  for (int u = 0; u < kRowsPerLane; ++u) {
    const int64_t r = first + u * 32 + lane;
    pos[u] = 0;
    from[u] = nullptr;
    if (r >= total || r >= p.max_rows) continue;
    if (c1 <= int(r)) {
      i += last_not_above(p.cu_rows + i, p.batch - i, int(r));
      c0 = p.cu_rows[i];
      c1 = p.cu_rows[i + 1];
      n0 = p.slot_map[c0] < 0 ? -1 : p.lengths[i] - (c1 - c0);
    }
    if (n0 < 0) continue;
    pos[u] = n0 + int(r) - c0;
    const int j = page_of(p, pos[u]);
    at[u] = pos[u] - j * p.page;
    from[u] = p.table + int64_t(i) * p.table_stride + j;
  }
#pragma unroll
  for (int u = 0; u < kRowsPerLane; ++u) slot[u] = from[u] ? int64_t(*from[u]) * p.page + at[u] : -1;
#pragma unroll
  for (int u = 0; u < kRowsPerLane; ++u) {
    const int64_t r = first + u * 32 + lane;
    if (r >= p.max_rows) continue;
    p.slot_map[r] = slot[u];
    p.positions[r] = pos[u];
  }
}

struct TrimArgs {
  int32_t* lengths;
  const int32_t* keep_len;
  int batch, page;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  int32_t* free_pages;
  int32_t* n_free;
  int n_pages;
};

// one CTA; shared memory: off [batch], left [batch]
__global__ void __launch_bounds__(kPagedThreads) paged_trim_kernel(const TrimArgs p) {
  extern __shared__ int sm[];
  __shared__ int64_t sa[kPagedWarps];
  __shared__ int sb[kPagedWarps];
  int* off = sm;
  int* left = off + p.batch;
  const int tid = threadIdx.x;
  const int free0 = min(max(*p.n_free, 0), p.n_pages);
  const int64_t most = int64_t(p.max_pages) * p.page;
  int64_t total = 0;
  for (int base = 0; base < p.batch; base += kPagedThreads) {
    const int i = base + tid;
    int have = 0, keep = 0;
    if (i < p.batch) {
      const int n = int(min(int64_t(max(p.lengths[i], 0)), most));
      const int k = min(max(p.keep_len[i], 0), n);
      have = int((int64_t(n) + p.page - 1) / p.page);
      keep = int((int64_t(k) + p.page - 1) / p.page);
    }
    int64_t o = have - keep;
    int unused = 0;
    int64_t t;
    int ut;
    cta_scan(o, unused, t, ut, sa, sb);
    if (i < p.batch) {
      off[i] = int(min(total + o, int64_t(0x7fffffff)));
      left[i] = keep;
    }
    total += t;
  }
  __syncthreads();  // lengths and n_free have been read, off and left are complete
  if (free0 + total > p.n_pages) {  // more pages than the pool holds come back: leave everything as it is
    if (tid == 0) raise_device_error(DSM_DEV_ERR_PAGES_SHORT);
    return;
  }
  const int back = int(total);
  // an entry that is no page must not reach the stack: all are looked at before anything moves, eight per thread at a
  // time, the first of them last, which stay
  constexpr int kKept = 8, kRound = kKept * kPagedThreads;
  int kept[kKept], bad = 0;
  auto load = [&](int base) {
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      const int k = base + j * kPagedThreads + tid;
      kept[j] = 0;
      if (k >= back) continue;
      const int i = last_not_above(off, p.batch, k);
      kept[j] = p.table[int64_t(i) * p.table_stride + left[i] + (k - off[i])];
    }
  };
  for (int base = (back - 1) / kRound * kRound; base >= 0; base -= kRound) {
    load(base);
#pragma unroll
    for (int j = 0; j < kKept; ++j) bad |= kept[j] < 0 || kept[j] >= p.n_pages;
  }
  if (__syncthreads_or(bad)) {
    if (tid == 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
    return;
  }
  for (int i = tid; i < p.batch; i += kPagedThreads) {
    const int n = int(min(int64_t(max(p.lengths[i], 0)), most));
    p.lengths[i] = min(max(p.keep_len[i], 0), n);
  }
  if (tid == 0) *p.n_free = free0 + back;
  for (int base = 0; base < back; base += kRound) {
    if (base > 0) load(base);
#pragma unroll
    for (int j = 0; j < kKept; ++j) {
      const int k = base + j * kPagedThreads + tid;
      if (k < back) p.free_pages[free0 + back - 1 - k] = kept[j];
    }
  }
}

// words of shared memory
constexpr size_t extend_words(int batch) { return size_t(3 * batch + 1); }
constexpr size_t trim_words(int batch) { return size_t(2 * batch); }

template <typename A>
int launch_cluster(void (*kernel)(const A), const A& args, int ctas, size_t smem, size_t smem_most, void* stream,
                   const char* what) {
  // what the largest batch takes, whatever this one does: the kernel's limit is every host thread's
  if (smem > 48 * 1024 &&
      cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem_most)) != cudaSuccess)
    return check_launch(what);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ctas));
  cfg.blockDim = dim3(kPagedThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = unsigned(ctas);
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args);
  if (e != cudaSuccess) return fail(DSM_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace
}  // namespace dsm

using namespace dsm;

extern "C" int dsm_paged_extend(int32_t* lengths, const int32_t* new_len, int batch, int page_size,
                                int32_t* block_table, int64_t table_stride, int max_pages,
                                const int32_t* free_pages, int32_t* n_free, int n_pages, int32_t* cu_rows,
                                int64_t* slot_map, int32_t* positions, int64_t max_rows, void* stream) {
  DSM_REQUIRE(batch >= 0 && batch <= kKv8MaxBatch, "dsm_paged_extend: batch must be 0..8192");
  DSM_REQUIRE(page_size > 0 && page_size % kKv8Group == 0 && page_size <= kKv8MaxPage,
              "dsm_paged_extend: page_size must be a multiple of 64, at most 1024");
  DSM_REQUIRE(max_pages > 0 && max_pages <= kKv8MaxPages && table_stride >= max_pages,
              "dsm_paged_extend: bad block table shape");
  DSM_REQUIRE(n_pages > 0 && max_rows >= 0 && max_rows <= 0x7fffffff, "dsm_paged_extend: bad sizes");
  DSM_REQUIRE(cu_rows && (max_rows == 0 || (slot_map && positions)) && free_pages && n_free &&
                  (batch == 0 || (lengths && new_len && block_table)),
              "dsm_paged_extend: NULL pointer");
  const uint32_t per_page = kv8_per_page(page_size);
  // one CTA covers a decode step's rows; a prefill's are written by the whole GPU, its tables by a cluster
  const bool many = max_rows > 4 * kPagedThreads;
  const ExtendArgs a = {lengths,  new_len, batch,   page_size, block_table, table_stride, max_pages, free_pages,
                        n_free,   n_pages, cu_rows, slot_map,  positions,   max_rows, per_page,    many};
  const int st = launch_cluster(paged_extend_kernel, a, many ? kPagedCluster : 1, extend_words(batch) * 4,
                                extend_words(kKv8MaxBatch) * 4, stream, "dsm_paged_extend");
  if (st != DSM_OK || !many) return st;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(unsigned(ceil_div(max_rows, int64_t(kRowThreads * kRowsPerLane))));
  cfg.blockDim = dim3(kRowThreads);
  cfg.stream = as_stream(stream);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, paged_rows_kernel, a);
  if (e != cudaSuccess) return fail(DSM_ERR_CUDA, std::string("dsm_paged_extend rows: ") + cudaGetErrorString(e));
  return check_launch("dsm_paged_extend rows");
}

extern "C" int dsm_paged_trim(int32_t* lengths, const int32_t* keep_len, int batch, int page_size,
                              const int32_t* block_table, int64_t table_stride, int max_pages, int32_t* free_pages,
                              int32_t* n_free, int n_pages, void* stream) {
  DSM_REQUIRE(batch >= 0 && batch <= kKv8MaxBatch, "dsm_paged_trim: batch must be 0..8192");
  DSM_REQUIRE(page_size > 0 && page_size % kKv8Group == 0 && page_size <= kKv8MaxPage,
              "dsm_paged_trim: page_size must be a multiple of 64, at most 1024");
  DSM_REQUIRE(max_pages > 0 && max_pages <= kKv8MaxPages && table_stride >= max_pages && n_pages > 0,
              "dsm_paged_trim: bad block table shape");
  if (batch == 0) return DSM_OK;
  DSM_REQUIRE(lengths && keep_len && block_table && free_pages && n_free, "dsm_paged_trim: NULL pointer");
  const TrimArgs a = {lengths, keep_len, batch, page_size, block_table, table_stride, max_pages, free_pages, n_free, n_pages};
  return launch_cluster(paged_trim_kernel, a, 1, trim_words(batch) * 4, trim_words(kKv8MaxBatch) * 4, stream,
                        "dsm_paged_trim");
}
