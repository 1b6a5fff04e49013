// What the kernels of the attention over the paged 8-bit cache share: their arguments, and how the
// work is cut into ranges of equal cost.
#pragma once

#include "kv8.cuh"

namespace dsm {

constexpr int kTile = kKv8Group;  // keys per tile
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e38f;

struct AttnArgs {
  const void* q;
  int64_t q_batch, q_row, q_head;  // strides in elements
  const uint8_t *k_codes, *v_codes;
  const float *k_scale, *v_scale;
  int page, n_pages;
  const int32_t* table;
  int64_t table_stride;
  int max_pages;
  const int32_t* lengths;
  const void *blk_k, *blk_v;  // NULL: the cached rows alone
  int64_t bk_batch, bk_head, bk_row, bv_batch, bv_head, bv_row;
  int batch, block, n_heads, n_kv;
  float scale;
  void* out;
};

// A unit is one sequence's KV head (and block of query rows); its tiles of 64 keys follow one another, and
// all units' tiles form one line that is cut into ranges of equal cost, one per CTA, whatever the
// lengths are; a unit costs `cost` tiles beside its own. A cut near a unit's edge moves to the edge.
struct KvSplit {
  int row_blocks;  // CTAs' row blocks per KV head
  int rows;        // query rows of a KV head: group * block
  int cta_rows;    // query rows of a unit
  int cost;
  int snap;        // a cut within this many tiles of a unit's edge moves there
  int least;       // cost that a range should have at least
  int ctas;
  float* part;     // [2 * ctas][cta_rows][head_dim] partial sums: a range's first unit, its last
  float4* ml;      // [2 * ctas][cta_rows] their reference, weight and value exponent
  int4* places;    // [ctas] where each range starts: sequence, unit, tile, the sequence's tiles
  int* cuts;       // [ctas + 1] the line's tile there
};
// tiles and their units' costs stay in 32 bits
inline bool split_fits(const AttnArgs& a, const KvSplit& sp) {
  return (int64_t(a.max_pages) * (a.page / kTile) + sp.cost) * a.batch * a.n_kv * sp.row_blocks <= 0x7fffffff;
}
inline size_t split_ws_bytes(int ctas, int cta_rows, int hd) {
  return size_t(2 * ctas) * cta_rows * (size_t(hd) + 4) * 4 + size_t(ctas) * 16 + size_t(ctas + 1) * 4;
}
inline void split_ws(KvSplit& sp, void* ws, int hd) {
  sp.part = static_cast<float*>(ws);
  sp.ml = reinterpret_cast<float4*>(sp.part + size_t(2 * sp.ctas) * sp.cta_rows * hd);
  sp.places = reinterpret_cast<int4*>(sp.ml + size_t(2 * sp.ctas) * sp.cta_rows);
  sp.cuts = reinterpret_cast<int*>(sp.places + sp.ctas);
}

// tiles before each sequence, for one KV head and row block (P [batch + 1]); a sequence without a
// cached row counts as one tile: its block's own rows still have to be attended
__device__ __forceinline__ int seq_len(const AttnArgs& p, int b) {
  return int(min(int64_t(max(__ldg(p.lengths + b), 0)), int64_t(p.max_pages) * p.page));
}

template <int kThreads>
__device__ __forceinline__ void scan_tiles(const AttnArgs& p, int* P, int* warp_sums) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  int before = 0;
  for (int base = 0; base < p.batch; base += kThreads) {
    const int b = base + tid;
    const int mine = b < p.batch ? max(1, (seq_len(p, b) + kTile - 1) / kTile) : 0;
    int x = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (base > 0) __syncthreads();  // warp_sums have been read
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int pre = before;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) pre += warp_sums[w];
      before += warp_sums[w];
    }
    if (b < p.batch) P[b] = pre + x - mine;
  }
  if (tid == 0) P[p.batch] = before;
  __syncthreads();
}

// where tile x of the line lies: sequence b, unit u of it (KV head * row_blocks + row block), tile t of T
struct Place {
  int b, u, t, T;
};
// with `cost` > 0, x counts that many more tiles in front of each unit (t < 0 there)
__device__ __forceinline__ Place place_of(const int* P, int batch, int hr, int x, int cost) {
  int lo = 0, hi = batch;  // the last sequence that starts at or before x
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if ((P[mid] + mid * cost) * hr <= x)
      lo = mid;
    else
      hi = mid;
  }
  Place r;
  r.b = lo;
  r.T = P[lo + 1] - P[lo];
  const unsigned rem = x - (P[lo] + lo * cost) * hr, each = r.T + cost;
  r.u = rem / each;
  r.t = int(rem - r.u * each) - cost;
  return r;
}
// the first tile of CTA i's range; short lines go to fewer CTAs
__device__ __forceinline__ int cut(const int* P, int batch, int hr, int i, const KvSplit& sp) {
  const unsigned total = (P[batch] + batch * sp.cost) * hr;
  const unsigned ctas = min(unsigned(sp.ctas), (total + sp.least - 1) / sp.least);
  if (i <= 0) return 0;
  if (i >= int(ctas)) return P[batch] * hr;
  const unsigned q = total / ctas, rest = total - q * ctas;
  const Place a = place_of(P, batch, hr, q * i + rest * i / ctas, sp.cost);
  const int d = min(sp.snap, a.T / 2);
  const int t = a.t <= d ? 0 : a.T - a.t <= d ? a.T : a.t;
  return P[a.b] * hr + a.u * a.T + t;
}

// this CTA's range: n tiles of the line from tile first, which is at `at`; noted down for the join. ends[6] in
// shared memory; all threads call it, a warp for either end.
__device__ __forceinline__ int my_range(const AttnArgs& p, const int* P, const KvSplit& sp, int* ends, int& first,
                                        Place& at) {
  const int hr = p.n_kv * sp.row_blocks, i = blockIdx.x, tid = threadIdx.x;
  if (tid == 0 || tid == 32) {
    const int x = cut(P, p.batch, hr, i + (tid >> 5), sp);
    ends[tid >> 5] = x;
    if (tid == 0) {
      const Place a = place_of(P, p.batch, hr, min(x, P[p.batch] * hr - 1), 0);
      ends[2] = a.b;
      ends[3] = a.u;
      ends[4] = a.t;
      ends[5] = a.T;
      sp.places[i] = make_int4(a.b, a.u, a.t, a.T);
      sp.cuts[i] = x;
    } else if (i == sp.ctas - 1) {
      sp.cuts[i + 1] = x;
    }
  }
  __syncthreads();
  first = ends[0];
  at.b = ends[2];
  at.u = ends[3];
  at.t = ends[4];
  at.T = ends[5];
  return ends[1] - first;
}
// the unit behind one
__device__ __forceinline__ void next_unit(const int* P, int batch, int hr, Place& a) {
  a.t = 0;
  if (++a.u == hr) {
    a.u = 0;
    if (++a.b < batch) a.T = P[a.b + 1] - P[a.b];
  }
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// the barrier gets one (counted) arrival once this thread's earlier cp.async have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= -kLowest ? a : 0.f;
}
__device__ __forceinline__ float scaled(float x, float f) {  // what is not finite becomes NaN
  return fabsf(x) <= -kLowest ? x * f : __int_as_float(0x7fffffff);
}
// V (a multiple of 4) contiguous values
template <typename T, int V>
__device__ __forceinline__ void load_vals(const T* p, bool vec, float (&x)[V]) {
  if (vec) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      if constexpr (std::is_same<T, float>::value) {
        const float4 v = *reinterpret_cast<const float4*>(p + i);
        x[i] = v.x;
        x[i + 1] = v.y;
        x[i + 2] = v.z;
        x[i + 3] = v.w;
      } else {
        const uint2 v = *reinterpret_cast<const uint2*>(p + i);
        x[i] = __uint_as_float(v.x << 16);
        x[i + 1] = __uint_as_float(v.x & 0xffff0000u);
        x[i + 2] = __uint_as_float(v.y << 16);
        x[i + 3] = __uint_as_float(v.y & 0xffff0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) x[i] = ld_f(p, i);
  }
}


inline bool vec_ok(const void* p, int64_t s0, int64_t s1, int64_t s2, size_t bytes) {
  const size_t e = bytes / 4;  // one load takes four values
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && s0 * e % bytes == 0 && s1 * e % bytes == 0 && s2 * e % bytes == 0;
}

// the tcgen05 kernel for bf16 rows and blocks of up to kUmmaMaxBlock rows (kv8_umma.cu); where it returns
// DSM_ERR_UNSUPPORTED nothing was launched, and the CUDA-core kernel takes the call
constexpr int kUmmaMaxBlock = 64;
size_t kv8_umma_ws_bytes(int rows, int hd);
int kv8_umma(const AttnArgs& a, int hd, void* ws, cudaStream_t s);
// joins what the cuts of sp left in parts
int kv8_combine(const AttnArgs& a, const KvSplit& sp, int hd, int dtype, cudaStream_t s);

}  // namespace dsm
