// dsm_gqa_attn_kv8: grouped-query attention of q [batch, block, n_heads, head_dim] over each
// sequence's rows in the paged 8-bit cache (layout in kv8.cuh) and then the block's own rows, with no
// mask: the paged form of Qwen3DSparkAttention.attend_cached (dspark_mlx/arch/qwen3.py:130-143).
//
//   kv8_attn_mma_kernel   bf16: e4m3 tensor-core products straight on the stored codes, split over
//                         the keys; kv8_attn_combine_kernel joins what was split.
//   kv8_attn_core_kernel  fp32 products on the CUDA cores, any type.
// dsm_set_attn_kernel picks between them (per host thread).
#include <algorithm>

#include "kv8.cuh"

namespace dsm {
namespace {

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

// The CUDA-core kernel: one warp per query row, 32 keys at a time with an online softmax, all in
// fp32. Lanes take a key each for the scores, then head_dim / 32 columns each for the sum. Runs
// for every type; the time goes into the fp32 products (two per code and query row).
constexpr int kCoreWarps = 4;

template <typename T, int HD>
__global__ void __launch_bounds__(kCoreWarps * 32) kv8_attn_core_kernel(const AttnArgs p) {
  constexpr int kCols = HD / 32;
  __shared__ float q_sm[kCoreWarps][HD];
  __shared__ float p_sm[kCoreWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t row = int64_t(blockIdx.x) * kCoreWarps + warp;
  if (row >= int64_t(p.batch) * p.block * p.n_heads) return;  // whole warps leave; warp syncs only
  const int h = int(row % p.n_heads);
  const int64_t bs = row / p.n_heads;
  const int s = int(bs % p.block), b = int(bs / p.block);
  const int g = h / (p.n_heads / p.n_kv);
  float* q = q_sm[warp];
  float* ps = p_sm[warp];
  const T* qg = static_cast<const T*>(p.q) + b * p.q_batch + s * p.q_row + h * p.q_head;
  for (int d = lane; d < HD; d += 32) q[d] = ld_f(qg, d) * p.scale;
  __syncwarp();
  const int64_t cap = int64_t(p.max_pages) * p.page;
  const int asked = p.lengths[b];
  const int len = int(min(int64_t(max(asked, 0)), cap));
  if (asked > cap && lane == 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
  const int32_t* table = p.table + int64_t(b) * p.table_stride;
  float m = -INFINITY, l = 0.f, acc[kCols];
#pragma unroll
  for (int i = 0; i < kCols; ++i) acc[i] = 0.f;
  for (int base = 0; base < len; base += 32) {
    const int pg = table[base / p.page];  // 32 tokens never straddle a page
    if (pg < 0 || pg >= p.n_pages) {
      if (lane == 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
      continue;
    }
    const int t0 = base % p.page, n = min(32, len - base);
    const int64_t ph = int64_t(pg) * p.n_kv + g;
    const uint8_t* kc = p.k_codes + (ph * p.page + t0 + lane) * HD;
    float x = -INFINITY;
    if (lane < n) {
      x = 0.f;
#pragma unroll 4
      for (int c = 0; c < HD / 16; ++c) {
        const uint4 w = *reinterpret_cast<const uint4*>(kc + kv8_key_chunk<HD>(c, t0 + lane) * 16);
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float f[4];
          kv8_to_f32(ws[j], f);
          const float4 qq = *reinterpret_cast<const float4*>(q + c * 16 + j * 4);
          x = fmaf(f[0], qq.x, x);
          x = fmaf(f[1], qq.y, x);
          x = fmaf(f[2], qq.z, x);
          x = fmaf(f[3], qq.w, x);
        }
      }
      x *= p.k_scale[ph];
    }
    const float m_new = fmaxf(m, kv8_warp_max(x));
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = expf(m - ref), w = expf(x - ref);
    l = l * alpha + kv8_warp_sum(w);
    m = m_new;
    ps[lane] = w * p.v_scale[ph];
    __syncwarp();
    const uint8_t* vc = p.v_codes + ph * p.page * HD + (t0 / kKv8Group) * HD * kKv8Group + t0 % kKv8Group;
#pragma unroll
    for (int i = 0; i < kCols; ++i) {
      const uint4* col = reinterpret_cast<const uint4*>(vc + (lane + 32 * i) * kKv8Group);
      const uint4 a = col[0], c = col[1];
      const uint32_t ws[8] = {a.x, a.y, a.z, a.w, c.x, c.y, c.z, c.w};
      float o = acc[i] * alpha;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float f[4];
        kv8_to_f32(ws[j], f);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (j * 4 + e < n) o = fmaf(ps[j * 4 + e], f[e], o);  // what lies behind the length is not read as a number
      }
      acc[i] = o;
    }
    __syncwarp();
  }
  if (p.blk_k) {
    const T* bk = static_cast<const T*>(p.blk_k) + b * p.bk_batch + g * p.bk_head;
    const T* bv = static_cast<const T*>(p.blk_v) + b * p.bv_batch + g * p.bv_head;
    for (int base = 0; base < p.block; base += 32) {
      const int n = min(32, p.block - base);
      float x = -INFINITY;
      if (lane < n) {
        x = 0.f;
        for (int d = 0; d < HD; ++d) x = fmaf(q[d], ld_f(bk, (base + lane) * p.bk_row + d), x);
      }
      const float m_new = fmaxf(m, kv8_warp_max(x));
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = expf(m - ref), w = expf(x - ref);
      l = l * alpha + kv8_warp_sum(w);
      m = m_new;
      ps[lane] = w;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < kCols; ++i) {
        float o = acc[i] * alpha;
        for (int j = 0; j < n; ++j) o = fmaf(ps[j], ld_f(bv, (base + j) * p.bv_row + lane + 32 * i), o);
        acc[i] = o;
      }
      __syncwarp();
    }
  }
  T* out = static_cast<T*>(p.out) + row * HD;
#pragma unroll
  for (int i = 0; i < kCols; ++i) out[lane + 32 * i] = st_f<T>(l == 0.f ? 0.f : acc[i] / l);
}

template <typename T, int HD>
int launch_core(const AttnArgs& a, cudaStream_t s) {
  const int64_t rows = int64_t(a.batch) * a.block * a.n_heads, grid = ceil_div(rows, kCoreWarps);
  DSM_REQUIRE(grid <= 0x7fffffff, "dsm_gqa_attn_kv8: too many rows");
  kv8_attn_core_kernel<T, HD><<<unsigned(grid), kCoreWarps * 32, 0, s>>>(a);
  return check_launch("gqa_attn_kv8");
}


// ------------------------------------------------------------------------------------------
// the tensor-core kernel
// ------------------------------------------------------------------------------------------
// Mathematics. The codes enter mma.m16n8k32 as they are stored. q, scaled per row by a power of two to
// at most 448, is split into two e4m3 terms (hi = e4m3(x), lo = e4m3(x - hi)): exact for bf16's 8
// significant bits wherever the residual reaches e4m3's normals, 2^-10 of a unit off elsewhere (row
// maximum 224 to 448). Both terms add into one fp32 accumulator. The weights of a 64-key tile,
// p = 2^(s - m_tile), are taken relative to the tile's own row maximum, so that a heavy key elsewhere
// does not push them out of e4m3's range, scaled to at most 2^8 and split the same way (2^-8 of each
// is lost, 2^-18 of the largest). The tile's product is then joined in fp32 with the running
// (m, l, o) of the row: o = o * 2^(m - m') + (2^(m_tile - m') * v_scale) * (p v).
//
// What bounds it: reading 2 * head_dim bytes per key and KV head. At the copy peak an SM gets 64
// keys of head_dim 128 per ~700 cycles; the e4m3 products take ~300 of them for 32 query rows (one
// m16n8k32 per ~1.15 cycles; f16 products on converted codes would take ~560 and two conversions per
// code pair), so codes are neither converted nor padded to 16 bits.
//
// Layout of the work. A unit is one sequence's KV head (and block of up to 128 query rows); its
// tiles of 64 keys follow one another, and all units' tiles form one line that is cut into equal
// ranges, one per CTA (one CTA per SM), whatever the lengths are. A cut near a unit's edge moves to
// the edge. In a CTA, tile i of its range belongs to lane i % tl (tl = warps / mg lanes side by side,
// of mg warps each; a warp holds all of the CTA's query rows, or 1 / mg of them where there are many).
// Tiles come by one bulk copy of keys and one of values into stages that belong to the lane: it refills
// the keys' half as soon as the scores are taken, the values' half after the sums, and waits for no
// other lane in the main loop.
constexpr int kTile = kKv8Group;
constexpr int kMaxDepth = 2;  // stages per lane, where they fit
// warps per CTA: a stage of head_dim 256 holds 32 KB, so four lanes fill shared memory
constexpr int mma_warps(int hd) { return hd == 256 ? 4 : 8; }
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kPScale = 8.f;  // weights enter e4m3 scaled by 2^8
constexpr float kLowest = -3.402823466e38f;

struct MmaPlan {
  int mg;          // warps that share a tile, each with its own query rows
  int row_blocks;  // CTAs' row blocks per KV head
  int rows;        // query rows of a KV head: group * block
  int depth;       // stages per lane
  int snap;        // a cut within this many tiles of a unit's edge moves there
  int least;       // tiles a range should have at least
  float* part;     // [2 * grid][cta_rows][head_dim] partial sums
  float* ml;       // [2 * grid][cta_rows][2] their maximum and weight
};

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
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    int pre = before;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) pre += warp_sums[w];
      before += warp_sums[w];
    }
    if (b < p.batch) P[b] = pre + x - mine;
    __syncthreads();
  }
  if (tid == 0) P[p.batch] = before;
  __syncthreads();
}

// where tile x of the line lies: sequence b, unit u of it (KV head * row_blocks + row block), tile t of T
struct Place {
  int b, u, t, T;
};
__device__ __forceinline__ Place place_of(const int* P, int batch, int hr, int x) {
  const int q = x / hr;  // P[b] <= q < P[b + 1]
  int lo = 0, hi = batch;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (P[mid] <= q)
      lo = mid;
    else
      hi = mid;
  }
  Place r;
  r.b = lo;
  r.T = P[lo + 1] - P[lo];
  const int rem = x - P[lo] * hr;
  r.u = rem / r.T;
  r.t = rem - r.u * r.T;
  return r;
}
// the start of CTA i's range; short lines go to fewer CTAs
__device__ __forceinline__ int cut(const int* P, int batch, int hr, int i, int ctas, int snap, int least) {
  const int total = P[batch] * hr;
  ctas = min(ctas, (total + least - 1) / least);
  if (i <= 0) return 0;
  if (i >= ctas) return total;
  const int x = int(int64_t(total) * i / ctas);
  if (x >= total) return total;
  const Place a = place_of(P, batch, hr, x);
  const int d = min(snap, a.T / 2);
  if (a.t <= d) return x - a.t;
  if (a.T - a.t <= d) return x + a.T - a.t;
  return x;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// D += A (16 x 32 e4m3, row) * B (32 x 8 e4m3, col), fp32
__device__ __forceinline__ void mma_e4m3(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
// four weights -> two e4m3 terms each, four bytes in order (x0 lowest): hi = e4m3(x), lo = e4m3(x - hi).
// The weights pass through f16, whose 11 bits are more than the two terms keep.
__device__ __forceinline__ void split_quad(float x0, float x1, float x2, float x3, uint32_t& hi, uint32_t& lo) {
  asm("{\n .reg .b32 x, y, g, h;\n .reg .b16 a, b, c, d;\n"
      " cvt.rn.f16x2.f32 x, %3, %2;\n"
      " cvt.rn.f16x2.f32 y, %5, %4;\n"
      " cvt.rn.satfinite.e4m3x2.f16x2 a, x;\n"
      " cvt.rn.satfinite.e4m3x2.f16x2 b, y;\n"
      " mov.b32 %0, {a, b};\n"
      " cvt.rn.f16x2.e4m3x2 g, a;\n"
      " cvt.rn.f16x2.e4m3x2 h, b;\n"
      " sub.rn.f16x2 x, x, g;\n"
      " sub.rn.f16x2 y, y, h;\n"
      " cvt.rn.satfinite.e4m3x2.f16x2 c, x;\n"
      " cvt.rn.satfinite.e4m3x2.f16x2 d, y;\n"
      " mov.b32 %1, {c, d};\n}"
      : "=&r"(hi), "=&r"(lo)
      : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
}
// the same for four values of a query row, whose residual may need more than f16 holds: in fp32
__device__ __forceinline__ void split_quad_f32(const float (&x)[4], uint32_t& hi, uint32_t& lo) {
  asm("{\n .reg .b32 g, h;\n .reg .f32 s, t, u, v;\n .reg .b16 a, b, c, d, e, f;\n"
      " cvt.rn.satfinite.e4m3x2.f32 a, %3, %2;\n"
      " cvt.rn.satfinite.e4m3x2.f32 b, %5, %4;\n"
      " mov.b32 %0, {a, b};\n"
      " cvt.rn.f16x2.e4m3x2 g, a;\n"
      " cvt.rn.f16x2.e4m3x2 h, b;\n"
      " mov.b32 {c, d}, g;\n mov.b32 {e, f}, h;\n"
      " cvt.f32.f16 s, c;\n cvt.f32.f16 t, d;\n cvt.f32.f16 u, e;\n cvt.f32.f16 v, f;\n"
      " sub.rn.f32 s, %2, s;\n sub.rn.f32 t, %3, t;\n sub.rn.f32 u, %4, u;\n sub.rn.f32 v, %5, v;\n"
      " cvt.rn.satfinite.e4m3x2.f32 c, t, s;\n"
      " cvt.rn.satfinite.e4m3x2.f32 d, v, u;\n"
      " mov.b32 %1, {c, d};\n}"
      : "=&r"(hi), "=&r"(lo)
      : "f"(x[0]), "f"(x[1]), "f"(x[2]), "f"(x[3]));
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
// the barrier gets one (counted) arrival once this thread's earlier cp.async have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <typename T, int V>
__device__ __forceinline__ void load_vals(const T* p, int lane, float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; ++i) x[i] = ld_f(p, lane * V + i);
}

// The last step of a query row, by one warp: the cached rows' (m, l, o) (base-2 maximum, weight and
// sum relative to it; m = -inf for none), then the block's own rows in fp32, then the division and the
// one rounding to T. Lane i holds columns [i * V, (i + 1) * V).
template <typename T, int HD>
__device__ __forceinline__ void finish_row(const AttnArgs& p, int b, int g, int r, float m, float l,
                                           float (&o)[HD / 32], int lane) {
  constexpr int V = HD / 32;
  const int group = p.n_heads / p.n_kv;
  const int h = g * group + r / p.block, s = r % p.block;
  if (p.blk_k) {
    float q[V];
    load_vals<T, V>(static_cast<const T*>(p.q) + b * p.q_batch + s * p.q_row + h * p.q_head, lane, q);
    const T* bk = static_cast<const T*>(p.blk_k) + b * p.bk_batch + g * p.bk_head;
    const T* bv = static_cast<const T*>(p.blk_v) + b * p.bv_batch + g * p.bv_head;
    const float c = p.scale * kLog2e;
    for (int base = 0; base < p.block; base += 8) {
      float x[8];
      float top = kLowest;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] = 0.f;
        if (base + j < p.block) {
          float k[V];
          load_vals<T, V>(bk + (base + j) * p.bk_row, lane, k);
#pragma unroll
          for (int i = 0; i < V; ++i) x[j] = fmaf(q[i], k[i], x[j]);
        }
      }
#pragma unroll
      for (int w = 16; w; w >>= 1) {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] += __shfl_xor_sync(0xffffffffu, x[j], w);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[j] *= c;
        if (base + j < p.block) top = fmaxf(top, x[j]);
      }
      const float mn = fmaxf(m, top);
      const float alpha = ex2(m - mn);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] *= alpha;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (base + j < p.block) {
          const float w = exp2f(x[j] - mn);
          float v[V];
          load_vals<T, V>(bv + (base + j) * p.bv_row, lane, v);
          l += w;
#pragma unroll
          for (int i = 0; i < V; ++i) o[i] = fmaf(w, v[i], o[i]);
        }
      }
      m = mn;
    }
  }
  T* out = static_cast<T*>(p.out) + ((int64_t(b) * p.block + s) * p.n_heads + h) * HD + lane * V;
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = st_f<T>(l == 0.f ? 0.f : o[i] / l);
}

// shared memory of the kernel, in bytes from its start
struct MmaSmem {
  int buf, qf, rowf, ml, top, scales, full, empty, sums, P, bytes;
};
__host__ __device__ inline MmaSmem mma_smem(int hd, int mt, int mg, int depth, int batch) {
  MmaSmem s;
  const int warps = mma_warps(hd), rows = 16 * mt * mg, tl = warps / mg, stages = depth * tl;
  s.buf = stages * 2 * kTile * hd;
  const int halves = tl / 2 * mg;  // warps that hand their sums over in the first round
  s.qf = s.buf + (halves * 16 * mt > rows ? halves * 16 * mt : rows) * hd * 4;
  s.rowf = s.qf + rows * hd * 2;
  s.ml = s.rowf + rows * 4;
  s.top = s.ml + warps * 16 * mt * 8;
  s.scales = s.top + rows * 8;
  s.full = s.scales + stages * 8;
  s.empty = s.full + stages * 16;
  s.sums = s.empty + stages * 8;
  s.P = s.sums + 64;
  s.bytes = s.P + (batch + 1) * 4;
  return s;
}

template <typename T, int HD, int MT>
__global__ void __launch_bounds__(mma_warps(HD) * 32, 1) kv8_attn_mma_kernel(const AttnArgs p, const MmaPlan pl) {
  constexpr int kWarps = mma_warps(HD);
  constexpr int kThreads = kWarps * 32;
  constexpr int NT = HD / 8;      // column tiles of the output
  constexpr int KS = HD / 32;     // k32 steps of q k
  constexpr int CH = HD / 64;     // 16-byte chunks of a key row per thread
  constexpr int V = HD / 32;
  constexpr int kKeyBytes = kTile * HD;
  constexpr int kWarpRows = 16 * MT;
  extern __shared__ __align__(128) uint8_t smem[];
  const MmaSmem L = mma_smem(HD, MT, pl.mg, pl.depth, p.batch);
  float* buf = reinterpret_cast<float*>(smem + L.buf);
  uint32_t* qf = reinterpret_cast<uint32_t*>(smem + L.qf);
  float* rowf = reinterpret_cast<float*>(smem + L.rowf);
  float2* ml = reinterpret_cast<float2*>(smem + L.ml);
  float2* top = reinterpret_cast<float2*>(smem + L.top);
  float2* scales = reinterpret_cast<float2*>(smem + L.scales);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.full);  // per stage: keys, values
  uint64_t* empty = reinterpret_cast<uint64_t*>(smem + L.empty);
  int* P = reinterpret_cast<int*>(smem + L.P);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gq = lane >> 2, cq = lane & 3;
  const int mg = pl.mg, tl = kWarps / mg, S = pl.depth * tl;
  const int my_mg = warp / tl, my_tl = warp % tl;
  const int hr = p.n_kv * pl.row_blocks;
  const int cta_rows = kWarpRows * mg;

  if (tid < S) {
    mbar_init(full + 2 * tid, 2);  // the copy's expect_tx, and the scale's cp.async
    mbar_init(full + 2 * tid + 1, 2);
    mbar_init(empty + tid, mg);
  }
  fence_mbar_init();
  scan_tiles<kThreads>(p, P, reinterpret_cast<int*>(smem + L.sums));
  const int ctas = gridDim.x;
  const int start = cut(P, p.batch, hr, blockIdx.x, ctas, pl.snap, pl.least);
  const int n_tiles = cut(P, p.batch, hr, blockIdx.x + 1, ctas, pl.snap, pl.least) - start;
  if (blockIdx.x == 0)
    for (int b = tid; b < p.batch; b += kThreads)
      if (p.lengths[b] > int64_t(p.max_pages) * p.page) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
  if (n_tiles <= 0) return;

  // ---- filling the stages: a cursor over the tiles that this lane fetches, one lane of warps my_mg == 0
  auto page_at = [&](const Place& a) -> int {  // the page of a tile, -1: nothing to fetch
    if (a.t * kTile >= seq_len(p, a.b)) return -1;
    const int pg = __ldg(p.table + int64_t(a.b) * p.table_stride + a.t * kTile / p.page);
    if (pg >= 0 && pg < p.n_pages) return pg;
    if (lane == 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
    return -1;
  };
  // half 0: keys, 1: values of tile a into stage st
  auto fetch = [&](int st, int half, const Place& a, int pg) {
    float* sc = reinterpret_cast<float*>(scales + st) + half;
    uint64_t* bar = full + 2 * st + half;
    if (pg < 0) {
      sc[0] = __int_as_float(0x7fc00000);  // marks a tile without keys
      mbar_arrive(bar);
      mbar_arrive(bar);
      return;
    }
    const int64_t ph = int64_t(pg) * p.n_kv + a.u / pl.row_blocks;
    const int64_t off = ph * p.page * HD + int64_t((a.t * kTile % p.page) / kTile) * kKeyBytes;
    cp_async4(smem_u32(sc), (half ? p.v_scale : p.k_scale) + ph);
    cp_async_arrive(bar);
    mbar_arrive_expect_tx(bar, kKeyBytes);
    bulk_g2s(smem + (2 * st + half) * kKeyBytes, (half ? p.v_codes : p.k_codes) + off, kKeyBytes, bar,
             policy_evict_first());
  };
  Place cur;  // the next tile that this lane fetches
  auto advance = [&]() {
    cur.t += tl;
    while (cur.t >= cur.T) {
      cur.t -= cur.T;
      if (++cur.u == hr) {
        cur.u = 0;
        if (++cur.b >= p.batch) return;
        cur.T = P[cur.b + 1] - P[cur.b];
      }
    }
  };
  if (my_mg == 0 && my_tl < n_tiles) {
    cur = place_of(P, p.batch, hr, start + my_tl);
    for (int i = my_tl; i < min(S, n_tiles); i += tl) {
      const int pg = page_at(cur);
      if (lane == 0) {
        fetch(i, 0, cur, pg);
        fetch(i, 1, cur, pg);
      }
      advance();
    }
  }
  bool ok = true;  // no wait has run out

  // ---- the range, unit by unit
  for (int a0 = 0; a0 < n_tiles;) {
    const Place un = place_of(P, p.batch, hr, start + a0);
    const int a1 = min(n_tiles, a0 + un.T - un.t);
    const int g = un.u / pl.row_blocks, r0 = (un.u % pl.row_blocks) * cta_rows;
    const int n_rows = min(cta_rows, pl.rows - r0);
    const int len = seq_len(p, un.b);
    const int group = p.n_heads / p.n_kv;

    // q: a warp per row, split into two e4m3 terms in the A-fragment order of the products
    __syncthreads();  // the previous unit's fragments and sums are used up
    for (int r = warp; r < cta_rows; r += kWarps) {
      constexpr int QV = HD == 64 ? 4 : V;  // values per lane, whole words of codes
      const bool mine = lane * QV < HD;
      float x[QV];
      int e = kKv8MinExp;
#pragma unroll
      for (int i = 0; i < QV; ++i) x[i] = 0.f;
      if (r < n_rows) {
        const int rr = r0 + r;
        if (mine)
          load_vals<T, QV>(static_cast<const T*>(p.q) + un.b * p.q_batch + (rr % p.block) * p.q_row +
                               (g * group + rr / p.block) * p.q_head,
                           lane, x);
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < QV; ++i) mx = fmaxf(mx, fabsf(x[i]) <= -kLowest ? fabsf(x[i]) : 0.f);
        e = kv8_scale_exp(kv8_warp_max(mx));
        // the sign of the factor goes into q: the row maximum is taken before the factor
        const float inv = p.scale < 0.f ? -kv8_exp2i(-e) : kv8_exp2i(-e);
#pragma unroll
        for (int i = 0; i < QV; ++i) x[i] = fabsf(x[i]) <= -kLowest ? x[i] * inv : __int_as_float(0x7fffffff);
      }
      if (lane == 0) rowf[r] = r < n_rows ? fabsf(p.scale) * kLog2e * kv8_exp2i(e) : 0.f;
#pragma unroll
      for (int i = 0; i < QV; i += 4) {
        uint32_t hi, lo;
        const float four[4] = {x[i], x[i + 1], x[i + 2], x[i + 3]};
        split_quad_f32(four, hi, lo);
        const int d = lane * QV + i, chunk = d >> 4, w = (d & 15) >> 2;
        int c, ks;  // the thread column and k32 step that multiply these columns
        if constexpr (HD == 64) {
          c = chunk;
          ks = w >> 1;
        } else {
          c = (chunk & 7) >> 1;
          ks = (chunk >> 3) * 4 + (chunk & 1) * 2 + (w >> 1);
        }
        const int reg = (w & 1) * 2 + ((r >> 3) & 1);
        const int at = ((((r >> 4) * KS + ks) * 2) * 32 + (r & 7) * 4 + c) * 4 + reg;
        if (mine) {
          qf[at] = hi;
          qf[at + 32 * 4] = lo;  // the lo fragment follows the hi one
        }
      }
    }
    __syncthreads();
    float cf[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      cf[mt][0] = rowf[my_mg * kWarpRows + mt * 16 + gq];
      cf[mt][1] = rowf[my_mg * kWarpRows + mt * 16 + gq + 8];
    }
    const uint4* my_q = reinterpret_cast<const uint4*>(qf) + my_mg * MT * KS * 2 * 32 + lane;

    float o[MT][NT][4], m[MT][2], l[MT][2];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[mt][n][i] = 0.f;
      m[mt][0] = m[mt][1] = -INFINITY;
      l[mt][0] = l[mt][1] = 0.f;
    }

    for (int i = a0 + (my_tl - a0 % tl + tl) % tl; i < a1; i += tl) {
      const int st = i % S;
      int next_pg = -1;
      const bool refill = my_mg == 0 && i + S < n_tiles;
      if (refill) next_pg = page_at(cur);  // its load overlaps the products below
      if (ok) ok = mbar_wait(full + 2 * st, (i / S) & 1);
      const float k_scale = scales[st].x;
      const int nv = min(kTile, len - (un.t + i - a0) * kTile);
      const bool any = ok && nv > 0 && k_scale == k_scale;
      const uint32_t kb = smem_u32(smem + st * 2 * kKeyBytes), vb = kb + kKeyBytes;
      if (any) {
        float s[MT][8][4];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[mt][j][e] = 0.f;
        // scores: column n of key tile j is key 16 * (n / 2) + 2 j + n % 2, so that a thread ends up with
        // the 16 keys whose codes of one value column lie together
        const uint32_t krow = kb + (16 * (gq >> 1) + (gq & 1)) * HD;
#pragma unroll
        for (int ch = 0; ch < CH; ++ch) {
          uint4 q[MT][2][2];
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf)
#pragma unroll
              for (int x = 0; x < 2; ++x) q[mt][hf][x] = my_q[((mt * KS + ch * 2 + hf) * 2 + x) * 32];
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            uint32_t addr = krow + 2 * j * HD;
            if constexpr (HD == 64)
              addr += cq * 16;
            else
              addr += ((ch >> 1) * 8 + ((2 * cq + (ch & 1)) ^ (((2 * j) & 7) | (gq & 1)))) * 16;
            const uint4 k = lds128(addr);
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
              mma_e4m3(s[mt][j], q[mt][0][0], k.x, k.y);
              mma_e4m3(s[mt][j], q[mt][0][1], k.x, k.y);
              mma_e4m3(s[mt][j], q[mt][1][0], k.z, k.w);
              mma_e4m3(s[mt][j], q[mt][1][1], k.z, k.w);
            }
          }
        }
        if (mg == 1 && refill) {  // the keys are used up
          __syncwarp();
          if (lane == 0) fetch(st, 0, cur, next_pg);
        }
        ok = mbar_wait(full + 2 * st + 1, (i / S) & 1);
        const float v_scale = scales[st].y;
        if (nv < kTile) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (16 * cq + 2 * j + e >= nv) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) s[mt][j][e] = s[mt][j][2 + e] = kLowest;
              }
        }
        uint4 ph[MT][2], pw[MT][2];  // the weights' two terms as A fragments of the two k32 steps
        float alpha[MT][2], beta[MT][2];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float mx = kLowest;
#pragma unroll
            for (int j = 0; j < 8; ++j) mx = fmaxf(mx, fmaxf(s[mt][j][2 * h], s[mt][j][2 * h + 1]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            const float c = cf[mt][h] * k_scale, mt_ = mx * c, off = kPScale - mt_;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                float& x = s[mt][j][2 * h + e];
                x = ex2(fmaf(x, c, off));
                if (nv < kTile && 16 * cq + 2 * j + e >= nv) x = 0.f;
                sum += x;
              }
            const float mn = fmaxf(m[mt][h], mt_);
            alpha[mt][h] = ex2(m[mt][h] - mn);
            const float bt = ex2(mt_ - mn);
            l[mt][h] = fmaf(l[mt][h], alpha[mt][h], bt * sum);
            beta[mt][h] = bt * v_scale;
            m[mt][h] = mn;
          }
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const float(&x)[8][4] = s[mt];
            const int j = 4 * k2;
            split_quad(x[j][0], x[j][1], x[j + 1][0], x[j + 1][1], ph[mt][k2].x, pw[mt][k2].x);
            split_quad(x[j][2], x[j][3], x[j + 1][2], x[j + 1][3], ph[mt][k2].y, pw[mt][k2].y);
            split_quad(x[j + 2][0], x[j + 2][1], x[j + 3][0], x[j + 3][1], ph[mt][k2].z, pw[mt][k2].z);
            split_quad(x[j + 2][2], x[j + 2][3], x[j + 3][2], x[j + 3][3], ph[mt][k2].w, pw[mt][k2].w);
          }
        }
        // values: columns 8 n + gq, this thread's 16 keys. Codes behind the length are cleared: a weight of
        // zero would not take a NaN there out
        uint32_t keep[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int k = nv - (16 * cq + 4 * w);
          keep[w] = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
        }
        const uint32_t vrow = vb + gq * kTile + cq * 16;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint4 v = lds128(vrow + n * 8 * kTile);
          if (nv < kTile) {
            v.x &= keep[0];
            v.y &= keep[1];
            v.z &= keep[2];
            v.w &= keep[3];
          }
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            float t[4] = {0.f, 0.f, 0.f, 0.f};
            mma_e4m3(t, ph[mt][0], v.x, v.y);
            mma_e4m3(t, pw[mt][0], v.x, v.y);
            mma_e4m3(t, ph[mt][1], v.z, v.w);
            mma_e4m3(t, pw[mt][1], v.z, v.w);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[mt][n][e] = fmaf(t[e], beta[mt][e >> 1], o[mt][n][e] * alpha[mt][e >> 1]);
          }
        }
      } else if (ok) {  // nothing to read; its values' half may still be on its way
        ok = mbar_wait(full + 2 * st + 1, (i / S) & 1);
      }
      __syncwarp();
      if (mg > 1) {  // the warps that share the tile are done with it
        if (lane == 0) mbar_arrive(empty + st);
        if (refill && ok) ok = mbar_wait(empty + st, (i / S) & 1);
      }
      if (refill) {
        if (ok && lane == 0) {
          if (mg > 1 || !any) fetch(st, 0, cur, next_pg);
          fetch(st, 1, cur, next_pg);
        }
        advance();
      }
    }

    // ---- the unit's sums of all lane groups into those of group 0
    const int wrow = warp * kWarpRows;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = l[mt][h];
        x += __shfl_xor_sync(0xffffffffu, x, 1);
        x += __shfl_xor_sync(0xffffffffu, x, 2);
        if (cq == 0) ml[wrow + mt * 16 + h * 8 + gq] = make_float2(m[mt][h], x);
      }
    __syncthreads();
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = mt * 16 + h * 8 + gq;
        float M = -INFINITY, W = 0.f;
        for (int t = 0; t < tl; ++t) M = fmaxf(M, ml[(my_mg * tl + t) * kWarpRows + r].x);
        const float ref = M == -INFINITY ? 0.f : M;
        for (int t = 0; t < tl; ++t) {
          const float2 x = ml[(my_mg * tl + t) * kWarpRows + r];
          W = fmaf(x.y, ex2(x.x - ref), W);
        }
        if (my_tl == 0 && cq == 0) top[my_mg * kWarpRows + r] = make_float2(M - kPScale, W);
        const float f = ex2(m[mt][h] - ref);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          o[mt][n][2 * h] *= f;
          o[mt][n][2 * h + 1] *= f;
        }
      }
    for (int half = tl / 2; half >= 1; half /= 2) {
      float4* slot = reinterpret_cast<float4*>(buf) + (my_mg * half + my_tl % half) * (kWarpRows * HD / 4) + lane;
      if (my_tl >= half && my_tl < 2 * half) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n)
            slot[(mt * NT + n) * 32] = make_float4(o[mt][n][0], o[mt][n][1], o[mt][n][2], o[mt][n][3]);
      }
      __syncthreads();
      if (my_tl < half) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float4 x = slot[(mt * NT + n) * 32];
            o[mt][n][0] += x.x;
            o[mt][n][1] += x.y;
            o[mt][n][2] += x.z;
            o[mt][n][3] += x.w;
          }
      }
      __syncthreads();
    }
    const bool whole = un.t == 0 && a1 - a0 == un.T;
    const int slot = 2 * blockIdx.x + (a0 == 0 && un.t > 0 ? 0 : 1);
    if (my_tl == 0) {  // rows as rows: to shared memory for the last step, or to the workspace
      float* dst = whole ? buf : pl.part + int64_t(slot) * cta_rows * HD;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = my_mg * kWarpRows + mt * 16 + h * 8 + gq;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            *reinterpret_cast<float2*>(dst + r * HD + 8 * n + 2 * cq) = make_float2(o[mt][n][2 * h], o[mt][n][2 * h + 1]);
        }
    }
    __syncthreads();
    if (whole) {
      for (int r = warp; r < n_rows; r += kWarps) {
        float x[V];
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = buf[r * HD + lane * V + i];
        finish_row<T, HD>(p, un.b, g, r0 + r, top[r].x, top[r].y, x, lane);
      }
    } else {
      float2* dst = reinterpret_cast<float2*>(pl.ml) + int64_t(slot) * cta_rows;
      for (int r = tid; r < cta_rows; r += kThreads) dst[r] = top[r];
    }
    a0 = a1;
  }
}

constexpr int kCombineWarps = 8;

// Joins the units that were cut: CTA (i, y) looks at the cut between ranges i and i + 1; if it is its unit's
// first, it joins the unit's rows y * 8 .. y * 8 + 7, a warp each: the partial sums of its ranges in
// order, then finish_row.
template <typename T, int HD>
__global__ void __launch_bounds__(kCombineWarps * 32) kv8_attn_combine_kernel(const AttnArgs p, const MmaPlan pl, int ctas,
                                                                        int cta_rows) {
  constexpr int V = HD / 32;
  extern __shared__ __align__(16) int P[];
  __shared__ int sums[kCombineWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hr = p.n_kv * pl.row_blocks;
  int* cuts = P + p.batch + 1;
  scan_tiles<kCombineWarps * 32>(p, P, sums);
  const int i = blockIdx.x;
  const int total = P[p.batch] * hr;
  const int x = cut(P, p.batch, hr, i + 1, ctas, pl.snap, pl.least);
  if (x >= total || x == 0) return;
  const Place un = place_of(P, p.batch, hr, x);
  const int u0 = x - un.t, u1 = u0 + un.T;
  if (un.t == 0 || cut(P, p.batch, hr, i, ctas, pl.snap, pl.least) > u0) return;
  for (int k = i + tid; k <= ctas; k += kCombineWarps * 32) cuts[k] = cut(P, p.batch, hr, k, ctas, pl.snap, pl.least);
  __syncthreads();
  int last = i + 1;  // the range that holds the unit's last tile
  while (cuts[last + 1] < u1) ++last;
  const int g = un.u / pl.row_blocks, r0 = (un.u % pl.row_blocks) * cta_rows;
  const int r = blockIdx.y * kCombineWarps + warp;
  if (r >= min(cta_rows, pl.rows - r0)) return;
  // range i's part is its last (slot 2 i + 1), the others' their first (slot 2 k); empty ranges have none
  auto slot_of = [&](int k) { return int64_t(k == i ? 2 * i + 1 : 2 * k) * cta_rows + r; };
  const float2* ml = reinterpret_cast<const float2*>(pl.ml);
  float M = -INFINITY;
  for (int k = i + lane; k <= last; k += 32)
    if (cuts[k] < cuts[k + 1]) M = fmaxf(M, ml[slot_of(k)].x);
  M = kv8_warp_max(M);
  const float ref = M == -INFINITY ? 0.f : M;
  float l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
#pragma unroll 4
  for (int k = i; k <= last; ++k) {
    if (cuts[k] == cuts[k + 1]) continue;
    const int64_t s = slot_of(k);
    const float2 w = ml[s];
    const float f = ex2(w.x - ref);
    const float* src = pl.part + s * HD + lane * V;
    l = fmaf(w.y, f, l);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] = fmaf(src[j], f, o[j]);
  }
  finish_row<T, HD>(p, un.b, g, r0 + r, M, l, o, lane);
}

constexpr int kMmaSmemMax = 232448;  // 227 KB

struct MmaShape {
  int mt, mg, row_blocks, cta_rows;
};
// Query rows of a KV head -> rows per warp and warps per tile: 16 rows where that is all, else 32 (one
// 16-row tile at head_dim 256, whose sums fill the registers), and more warps over the same tile
// up to 128 rows (64 at head_dim 256).
MmaShape mma_shape(int rows, int hd) {
  MmaShape s;
  s.mt = rows <= 16 || hd == 256 ? 1 : 2;
  const int most = hd == 256 ? 64 : 128;
  s.mg = 1;
  while (16 * s.mt * s.mg < std::min(rows, most)) s.mg *= 2;
  s.cta_rows = 16 * s.mt * s.mg;
  s.row_blocks = int(ceil_div(rows, s.cta_rows));
  return s;
}

template <typename T, int HD, int MT>
int launch_mma(const AttnArgs& a, const MmaShape& sh, MmaPlan pl, int ctas, cudaStream_t s) {
  int depth = std::max(kMaxDepth, sh.mg);
  while (depth > 1 && mma_smem(HD, MT, sh.mg, depth, a.batch).bytes > kMmaSmemMax) --depth;
  const int smem = mma_smem(HD, MT, sh.mg, depth, a.batch).bytes;
  if (smem > kMmaSmemMax) return fail(DSM_ERR_UNSUPPORTED, "dsm_gqa_attn_kv8: batch too large for shared memory");
  pl.depth = depth;
  auto k = kv8_attn_mma_kernel<T, HD, MT>;
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("gqa_attn_kv8 smem attribute");
  k<<<unsigned(ctas), mma_warps(HD) * 32, size_t(smem), s>>>(a, pl);
  const int st = check_launch("gqa_attn_kv8");
  if (st != DSM_OK || ctas == 1) return st;
  const dim3 grid(unsigned(ctas - 1), unsigned(ceil_div(std::min(sh.cta_rows, pl.rows), kCombineWarps)));
  kv8_attn_combine_kernel<T, HD><<<grid, kCombineWarps * 32, size_t(a.batch + ctas + 2) * 4, s>>>(a, pl, ctas, sh.cta_rows);
  return check_launch("gqa_attn_kv8 combine");
}

size_t mma_ws_bytes(const MmaShape& sh, int hd) {
  return size_t(2 * num_sms()) * sh.cta_rows * (size_t(hd) + 2) * 4;
}

template <typename T>
int run_mma(const AttnArgs& a, int hd, void* ws, cudaStream_t s) {
  const MmaShape sh = mma_shape(a.n_heads / a.n_kv * a.block, hd);
  const int64_t most = int64_t(a.batch) * a.max_pages * (a.page / kTile) * a.n_kv * sh.row_blocks;
  if (most > 0x7fffffff) return fail(DSM_ERR_UNSUPPORTED, "dsm_gqa_attn_kv8: block table too large");
  const int ctas = int(std::min<int64_t>(num_sms(), std::max<int64_t>(most, 1)));
  MmaPlan pl;
  pl.mg = sh.mg;
  pl.row_blocks = sh.row_blocks;
  pl.rows = a.n_heads / a.n_kv * a.block;
  pl.depth = 0;
  pl.snap = std::max(1, mma_warps(hd) / sh.mg / 2);
  pl.least = pl.snap;
  pl.part = static_cast<float*>(ws);
  pl.ml = pl.part + size_t(2 * num_sms()) * sh.cta_rows * hd;
  switch (hd) {
    case 64: return sh.mt == 1 ? launch_mma<T, 64, 1>(a, sh, pl, ctas, s) : launch_mma<T, 64, 2>(a, sh, pl, ctas, s);
    case 128: return sh.mt == 1 ? launch_mma<T, 128, 1>(a, sh, pl, ctas, s) : launch_mma<T, 128, 2>(a, sh, pl, ctas, s);
    default: return launch_mma<T, 256, 1>(a, sh, pl, ctas, s);
  }
}

}  // namespace
}  // namespace dsm

using namespace dsm;

extern "C" size_t dsm_gqa_attn_kv8_workspace_bytes(int batch, int block, int n_heads, int n_kv, int head_dim) {
  if (batch <= 0 || batch > kKv8MaxBatch || block <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0 ||
      !kv8_head_dim_ok(head_dim))
    return 0;
  return mma_ws_bytes(mma_shape(n_heads / n_kv * block, head_dim), head_dim);
}

extern "C" int dsm_gqa_attn_kv8(const dsm_kv8_attn_desc* d, const void* q, const int32_t* block_table,
                                const int32_t* lengths, const void* blk_k, const void* blk_v, void* out, void* ws,
                                size_t ws_bytes, void* stream) {
  DSM_REQUIRE(d != nullptr, "dsm_gqa_attn_kv8: desc is NULL");
  DSM_REQUIRE(d->batch >= 0 && d->batch <= kKv8MaxBatch, "dsm_gqa_attn_kv8: batch must be 0..8192");
  DSM_REQUIRE(d->block > 0 && d->n_kv > 0 && d->n_heads > 0 && d->n_heads % d->n_kv == 0,
              "dsm_gqa_attn_kv8: bad shape (n_heads must be a multiple of n_kv)");
  DSM_REQUIRE(kv8_head_dim_ok(d->head_dim), "dsm_gqa_attn_kv8: head_dim must be 64, 128 or 256");
  DSM_REQUIRE(kv8_page_ok(d->page_size), "dsm_gqa_attn_kv8: page_size must be a multiple of 64, at most 1024");
  DSM_REQUIRE(d->n_pages > 0 && d->max_pages > 0 && d->max_pages <= kKv8MaxPages && d->table_stride >= d->max_pages,
              "dsm_gqa_attn_kv8: bad block table shape");
  DSM_REQUIRE(d->dtype == DSM_DT_F32 || d->dtype == DSM_DT_BF16, "dsm_gqa_attn_kv8: dtype must be F32 or BF16");
  DSM_REQUIRE(d->q_batch_stride >= 0 && d->q_row_stride >= 0 && d->q_head_stride >= 0, "dsm_gqa_attn_kv8: bad strides");
  DSM_REQUIRE((blk_k == nullptr) == (blk_v == nullptr), "dsm_gqa_attn_kv8: blk_k and blk_v come together");
  DSM_REQUIRE(!blk_k || (d->bk_batch_stride >= 0 && d->bk_head_stride >= 0 && d->bk_row_stride >= 0 &&
                         d->bv_batch_stride >= 0 && d->bv_head_stride >= 0 && d->bv_row_stride >= 0),
              "dsm_gqa_attn_kv8: bad strides");
  if (d->batch == 0) return DSM_OK;
  DSM_REQUIRE(q && block_table && lengths && out && ws && d->k_codes && d->v_codes && d->k_scale && d->v_scale,
              "dsm_gqa_attn_kv8: NULL pointer");
  DSM_REQUIRE(kv8_aligned16(d->k_codes) && kv8_aligned16(d->v_codes), "dsm_gqa_attn_kv8: codes must be 16-byte aligned");
  DSM_REQUIRE(kv8_aligned16(ws), "dsm_gqa_attn_kv8: workspace must be 16-byte aligned");
  if (ws_bytes < dsm_gqa_attn_kv8_workspace_bytes(d->batch, d->block, d->n_heads, d->n_kv, d->head_dim))
    return fail(DSM_ERR_WORKSPACE, "dsm_gqa_attn_kv8: workspace too small");
  const AttnArgs a = {q,
                      d->q_batch_stride,
                      d->q_row_stride,
                      d->q_head_stride,
                      static_cast<const uint8_t*>(d->k_codes),
                      static_cast<const uint8_t*>(d->v_codes),
                      d->k_scale,
                      d->v_scale,
                      d->page_size,
                      d->n_pages,
                      block_table,
                      d->table_stride,
                      d->max_pages,
                      lengths,
                      blk_k,
                      blk_v,
                      d->bk_batch_stride,
                      d->bk_head_stride,
                      d->bk_row_stride,
                      d->bv_batch_stride,
                      d->bv_head_stride,
                      d->bv_row_stride,
                      d->batch,
                      d->block,
                      d->n_heads,
                      d->n_kv,
                      d->scale,
                      out};
  cudaStream_t s = as_stream(stream);
  if (d->dtype == DSM_DT_BF16 && attn_kernel() == 0) return run_mma<__nv_bfloat16>(a, d->head_dim, ws, s);
  if (d->dtype == DSM_DT_BF16) {
    switch (d->head_dim) {
      case 64: return launch_core<__nv_bfloat16, 64>(a, s);
      case 128: return launch_core<__nv_bfloat16, 128>(a, s);
      default: return launch_core<__nv_bfloat16, 256>(a, s);
    }
  }
  switch (d->head_dim) {
    case 64: return launch_core<float, 64>(a, s);
    case 128: return launch_core<float, 128>(a, s);
    default: return launch_core<float, 256>(a, s);
  }
}
