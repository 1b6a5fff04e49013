// dsm_gqa_attn_kv8: grouped-query attention of q [batch, block, n_heads, head_dim] over each
// sequence's rows in the paged 8-bit cache (layout in kv8.cuh) and then the block's own rows, with no
// mask: the paged form of Qwen3DSparkAttention.attend_cached (dspark_mlx/arch/qwen3.py:130-143).
//
//   kv8_umma_kernel       bf16 rows and blocks of up to 64 rows, on tcgen05 (kv8_umma.cu)
//   kv8_attn_mma_kernel   fp32 rows: f16 products in two terms each, split over the keys
//   kv8_attn_combine_kernel  joins what either has cut
//   kv8_attn_core_kernel  fp32 products on the CUDA cores: what the others do not take (a longer block, a
//                         batch whose prefix does not fit shared memory, a sequence's result past 2^31
//                         values), and dsm_set_attn_kernel's other choice (per host thread)
#include <algorithm>

#include "kv8_attn.cuh"

namespace dsm {
namespace {

// The CUDA-core kernel: one warp per query row, 32 keys at a time with an online softmax, all in
// fp32. Lanes take a key each for the scores, then head_dim / 32 columns each for the sum. What is not
// finite counts as NaN, as in the other kernels, whose scaled terms have no infinity. Runs for every type; the time goes into the fp32 products (two per code and query row).
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
  for (int d = lane; d < HD; d += 32) q[d] = scaled(ld_f(qg, d), p.scale);
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
        for (int d = 0; d < HD; ++d) x = fmaf(q[d], scaled(ld_f(bk, (base + lane) * p.bk_row + d), 1.f), x);
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
        for (int j = 0; j < n; ++j) o = fmaf(ps[j], scaled(ld_f(bv, (base + j) * p.bv_row + lane + 32 * i), 1.f), o);
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
// the tensor-core kernel for fp32 rows
// ------------------------------------------------------------------------------------------
// Mathematics. e4m3 codes are exact in f16, so keys and values enter mma.m16n8k16 as the codes'
// values and the page's power-of-two scales stay outside. q, scaled per row by a power of two to at
// most 448, is two f16 terms (hi + lo, 2^-22). A row's weights are p = 2^(s - m) with a reference m that
// follows its running maximum only when that has grown by more than 2^8, so that the sums are rescaled
// rarely; they enter f16, in two terms as well, as p * 2^6 * 2^(ev - rv), ev the exponent of the page's
// value scale and rv a reference that it moves when it leaves [rv - 10, rv]: the sums need no factor per
// page. The second term is held times 2^11 and summed apart, so that small weights keep their bits (in one
// sum, weights 2^-20 of the largest were 2^-12 off; apart costs 1 to 2%, 92.8 instead of 90.7 us for 32
// sequences of 4096 keys, 8 KV heads of 4 rows). Sums, weights and maxima are fp32. The tensor cores' own additions cut off what they round, too
// coarse for fp32 calls over long sums: products go into the fp32 sums a few steps at a time, by CUDA cores.
//
// What bounds it: for long sequences the products, two terms of q (and of the weights) for each code at 0.46
// mma.sync per clock and SM: 64 keys of head_dim 128 and 16 rows take 512 of them, 1,100 cycles against the ~700
// that their bytes take at the copy peak (32 sequences of 4096 keys, 8 KV heads of 4 rows: 93 us, 3 TB/s). The
// tcgen05 kernel multiplies the codes without conversion, but e4m3 terms of an fp32 row would be four. Short
// sequences are bound by what a unit costs: 8 sequences, 4 KV heads of 20 rows, take 12.3 us at one tile each, 13.2
// at four (launch, scan, staging, the lanes' join), 2 more with own rows, 7 more as soon as units are cut (a second
// unit's staging and the join: 20.3 us at eight tiles, 24.5 at 32). Hence 23 us for such sequences of up to 1000 keys.
//
// Layout of the work. A unit is one sequence's KV head (and block of up to 128 query rows); its
// tiles of 64 keys follow one another, and all units' tiles form one line that is cut into ranges of
// equal cost, one per CTA (one CTA per SM), whatever the lengths are; a unit costs kUnitCost tiles
// beside its own. A cut near a unit's edge moves to the edge. In a CTA, tile i of its range belongs to
// lane i % tl (tl = warps / mg lanes side by side, of mg warps each; a warp holds all of the CTA's query
// rows, or 1 / mg of them where there are many). Tiles come by one bulk copy of keys and one of values
// into stages that belong to the lane: it refills the keys' half as soon as the scores are taken, the
// values' half after the sums, and waits for no other lane in the main loop. The block's own rows are
// 16-key tiles of whichever CTA holds the unit's last tile, read straight from the caller's tensors.
constexpr int kMaxDepth = 2;  // stages per lane, where they fit
// a unit's q, join and output, in tiles, and the least that a range should cost. 20 ragged sequences of up to 3000, 4 KV
// heads of 20 rows of 64, 128 and 256: 20.5, 26.8 and 43.1 us; with cost 3 23.0, 29.5, 44.8; with 10 23.8, 31.3, 48.8.
// Ranges of 12 are slower still (24.5, 32.1, 58.8); of 3 as fast there, and up to 25% faster for equal short sequences.
constexpr int kUnitCost = 6;
// warps per CTA: a stage of head_dim 256 holds 32 KB, so four lanes fill shared memory
constexpr int mma_warps(int hd) { return hd == 256 ? 4 : 8; }
constexpr float kPScale = 6.f;  // weights at the reference enter f16 as 2^6,
constexpr float kPGrow = 8.f;   // and grow to 2^14 before the reference follows

struct MmaPlan {
  KvSplit sp;
  int mg;     // warps that share a tile, each with its own query rows
  int depth;  // stages per lane
  bool vec_q, vec_blk;  // q's / the block's rows can be read 4 values at a time
};

__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// (x0, x1) as two f16 terms, t[0] + t[1]
constexpr int kTerms = 2;
__device__ __forceinline__ void f16_terms(float x0, float x1, uint32_t (&t)[kTerms]) {
  t[0] = pack_f16(x0, x1);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&t[0]));
  t[1] = pack_f16(x0 - h.x, x1 - h.y);
}
// the same of weights, the second term times 2^11: it keeps 11 bits of a weight down to 2^-24, f16's smallest step,
// and its products are summed apart. What is lost is 2^-22 of a weight and 2^-36, where the largest is 2^6 or more.
constexpr float kWeightLo = 1.f / 2048.f;
__device__ __forceinline__ void weight_terms(float x0, float x1, uint32_t (&t)[kTerms]) {
  t[0] = pack_f16(x0, x1);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&t[0]));
  t[1] = pack_f16((x0 - h.x) * 2048.f, (x1 - h.y) * 2048.f);
}
__device__ __forceinline__ void mma(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1));
}
template <int A>
__device__ __forceinline__ void zero(float (&x)[A][4]) {
#pragma unroll
  for (int a = 0; a < A; ++a)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[a][e] = 0.f;
}
// 16 of the block's own rows as B fragments of f16 terms, and their exponents, in words
__host__ __device__ constexpr int mma_block_words(int hd) {
  return 2 * (hd / 16) * kTerms * 64 + hd / 8 * kTerms * 64 + 32;
}
// shared memory of the kernel, in bytes from its start
struct MmaSmem {
  int buf, qf, rowf, ml, scales, full, empty, sums, P, bytes;
};
__host__ __device__ inline MmaSmem mma_smem(int hd, int mg, int depth, int batch) {
  MmaSmem s;
  const int warps = mma_warps(hd), rows = 16 * mg, tl = warps / mg, stages = depth * tl;
  s.buf = stages * 2 * kTile * hd;
  // the lanes that hand their sums over in the first round; before that, 16 rows of the block per lane
  const int sums = tl / 2 * rows * hd * 4, block = mma_block_words(hd) * 4;
  s.qf = s.buf + (sums > block ? sums : block);
  s.rowf = s.qf + rows * hd * 2 * kTerms;
  s.ml = s.rowf + rows * 4;
  s.scales = s.ml + warps * 16 * 16;
  s.full = s.scales + stages * 8;
  s.empty = s.full + stages * 16;
  s.sums = s.empty + stages * 8;
  s.P = s.sums + 64;
  s.bytes = s.P + (batch + 1) * 4;
  return s;
}

template <int HD>
__global__ void __launch_bounds__(mma_warps(HD) * 32, 1) kv8_attn_mma_kernel(const AttnArgs p, const MmaPlan pl) {
  constexpr int kWarps = mma_warps(HD);
  constexpr int kThreads = kWarps * 32;
  constexpr int NT = HD / 8;   // column tiles of the output
  constexpr int KS = HD / 16;  // k16 steps of q k
  constexpr int CH = HD / 64;  // 16-byte chunks of a key row per thread
  constexpr int kKeyBytes = kTile * HD;
  constexpr int kWarpRows = 16;
  constexpr int TPR = kThreads / 16, VB = HD / TPR;  // staging: 16 rows at a time, threads per row, values per thread
  constexpr int kBlockWords = mma_block_words(HD);
  extern __shared__ __align__(128) uint8_t smem[];
  const MmaSmem L = mma_smem(HD, pl.mg, pl.depth, p.batch);
  float* buf = reinterpret_cast<float*>(smem + L.buf);
  uint32_t* qf = reinterpret_cast<uint32_t*>(smem + L.qf);
  float* rowf = reinterpret_cast<float*>(smem + L.rowf);
  float4* ml = reinterpret_cast<float4*>(smem + L.ml);
  float2* scales = reinterpret_cast<float2*>(smem + L.scales);
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.full);  // per stage: keys, values
  uint64_t* empty = reinterpret_cast<uint64_t*>(smem + L.empty);
  int* P = reinterpret_cast<int*>(smem + L.P);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int gq = lane >> 2, cq = lane & 3;
  const int mg = pl.mg, tl = kWarps / mg, S = pl.depth * tl;
  const int my_mg = warp / tl, my_tl = warp % tl;
  const int hr = p.n_kv * pl.sp.row_blocks;
  const int cta_rows = kWarpRows * mg;
  const int row_r = tid / TPR, row_d = tid % TPR * VB;  // this thread's row (of 16) and first column in staging

  if (tid < S) {
    mbar_init(full + 2 * tid, 2);  // the copy's expect_tx, and the scale's cp.async
    mbar_init(full + 2 * tid + 1, 2);
    mbar_init(empty + tid, mg);
  }
  fence_mbar_init();
  scan_tiles<kThreads>(p, P, reinterpret_cast<int*>(smem + L.sums));
  asm volatile("griddepcontrol.launch_dependents;");  // the join may take its place and wait
  int start;
  Place first;
  const int n_tiles = my_range(p, P, pl.sp, reinterpret_cast<int*>(smem + L.sums) + 8, start, first);
  if (blockIdx.x == 0)
    for (int b = tid; b < p.batch; b += kThreads)
      if (p.lengths[b] > int64_t(p.max_pages) * p.page) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
  if (n_tiles <= 0) return;

  // ---- filling the stages: a cursor over the tiles that this lane fetches, one thread of warps my_mg == 0
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
    const int64_t ph = int64_t(pg) * p.n_kv + a.u / pl.sp.row_blocks;
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
    cur = place_of(P, p.batch, hr, start + my_tl, 0);
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
    const Place un = place_of(P, p.batch, hr, start + a0, 0);
    const int a1 = min(n_tiles, a0 + un.T - un.t);
    const bool last = un.t + a1 - a0 == un.T, whole = last && un.t == 0;
    const int g = un.u / pl.sp.row_blocks, r0 = (un.u % pl.sp.row_blocks) * cta_rows;
    const int n_rows = min(cta_rows, pl.sp.rows - r0);
    const int len = seq_len(p, un.b);
    const int group = p.n_heads / p.n_kv;

    // the power of two of a row whose VB values lie in each of its threads
    auto row_exp = [&](const float(&x)[VB]) -> int {
      float mx = 0.f;
#pragma unroll
      for (int i = 0; i < VB; ++i) mx = fmaxf(mx, finite_abs(x[i]));
#pragma unroll
      for (int w = TPR / 2; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      return kv8_scale_exp(mx);
    };
    // thread column c multiplies chunks 2 c and 2 c + 1 of each 128 columns (chunk c of 64), four columns
    // per k16 step: its first two are k = 2 c, 2 c + 1 (reg 0), the others k + 8 (reg 1)
    auto k_place = [&](int d, int& c, int& ks, int& reg) {
      const int chunk = d >> 4, w = (d & 15) >> 2;
      c = HD == 64 ? chunk : (chunk & 7) >> 1;
      ks = HD == 64 ? w : (chunk >> 3) * 8 + (chunk & 1) * 4 + w;
      reg = (d & 3) >> 1;
    };
    // 16 rows of the block from row kb, as B fragments in the join buffer. Key r of them is column
    // 2 * (r / 4) + r % 2 of key tile (r / 2) % 2, so that a thread's four keys are 4 c .. 4 c + 3.
    auto load_block = [&](int kb, float(&x)[VB], float(&y)[VB]) {
      if (kb + row_r < p.block) {
        load_vals<float, VB>(static_cast<const float*>(p.blk_k) + un.b * p.bk_batch + g * p.bk_head +
                             (kb + row_r) * p.bk_row + row_d, pl.vec_blk, x);
        load_vals<float, VB>(static_cast<const float*>(p.blk_v) + un.b * p.bv_batch + g * p.bv_head +
                             (kb + row_r) * p.bv_row + row_d, pl.vec_blk, y);
      }
    };
    auto put_block = [&](int slot, float(&x)[VB], float(&y)[VB]) {
      uint32_t* kf = reinterpret_cast<uint32_t*>(buf) + slot * kBlockWords;
      uint32_t* vf = kf + 2 * KS * kTerms * 64;
      const int ek = row_exp(x), ev = row_exp(y);
      const float ik = kv8_exp2i(-ek), iv = kv8_exp2i(-ev);
      if (row_d == 0) {
        float* e = reinterpret_cast<float*>(vf + NT * kTerms * 64);
        e[row_r] = kv8_exp2i(ek);
        e[16 + row_r] = float(ev);
      }
      const int gk = 2 * (row_r >> 2) + (row_r & 1), jk = (row_r >> 1) & 1;
#pragma unroll
      for (int i = 0; i < VB; i += 2) {
        const int d = row_d + i;
        int c, ks, reg;
        k_place(d, c, ks, reg);
        uint32_t f[kTerms];
        f16_terms(scaled(x[i], ik), scaled(x[i + 1], ik), f);
#pragma unroll
        for (int t = 0; t < kTerms; ++t) kf[((jk * KS + ks) * kTerms + t) * 64 + (gk * 4 + c) * 2 + reg] = f[t];
        f16_terms(scaled(y[i], iv), scaled(y[i + 1], iv), f);
#pragma unroll
        for (int t = 0; t < kTerms; ++t) {
          uint16_t* v16 = reinterpret_cast<uint16_t*>(
              vf + ((d >> 3) * kTerms + t) * 64 + ((d & 7) * 4 + (row_r >> 2)) * 2 + ((row_r >> 1) & 1)) + (row_r & 1);
          v16[0] = uint16_t(f[t]);
          v16[16] = uint16_t(f[t] >> 16);  // the next column's thread, four on
        }
      }
    };

    // q and the block's own rows, TPR threads to a row: scaled per row by a power of two to at most 448, in
    // f16 terms, in the fragment order of the products
    __syncthreads();  // the previous unit's fragments and sums are used up
    {
      const float* qg = static_cast<const float*>(p.q) + un.b * p.q_batch;
      auto load_q = [&](int r, float(&x)[VB]) {
        const int rr = r0 + r;
        if (r < n_rows)
          load_vals<float, VB>(qg + (rr % p.block) * p.q_row + (g * group + rr / p.block) * p.q_head + row_d, pl.vec_q, x);
      };
      auto put_q = [&](int r, float(&x)[VB]) {
        const int e = row_exp(x);
        // the sign of the factor goes into q: the row maximum is taken before the factor
        const float inv = p.scale < 0.f ? -kv8_exp2i(-e) : kv8_exp2i(-e);
        if (row_d == 0) rowf[r] = r < n_rows ? fabsf(p.scale) * kLog2e * kv8_exp2i(e) : 0.f;
#pragma unroll
        for (int i = 0; i < VB; i += 2) {
          int c, ks, reg;
          k_place(row_d + i, c, ks, reg);
          uint32_t f[kTerms];
          f16_terms(scaled(x[i], inv), scaled(x[i + 1], inv), f);
#pragma unroll
          for (int t = 0; t < kTerms; ++t)
            qf[((((r >> 4) * KS + ks) * kTerms + t) * 32 + (r & 7) * 4 + c) * 4 + 2 * reg + ((r >> 3) & 1)] = f[t];
        }
      };
      float x[2][VB] = {}, y[2][VB] = {};
      if (last && p.blk_k) load_block(0, x[0], x[1]);
      load_q(row_r, y[0]);
      if (mg > 1) load_q(row_r + 16, y[1]);
      if (last && p.blk_k) put_block(0, x[0], x[1]);
      put_q(row_r, y[0]);
      if (mg > 1) put_q(row_r + 16, y[1]);
      for (int r = row_r + 32; r < cta_rows; r += 32) {
        float z[2][VB] = {};
        load_q(r, z[0]);
        load_q(r + 16, z[1]);
        put_q(r, z[0]);
        put_q(r + 16, z[1]);
      }
    }
    __syncthreads();
    float cf[2];
    cf[0] = rowf[my_mg * kWarpRows + gq];
    cf[1] = rowf[my_mg * kWarpRows + gq + 8];
    const uint4* my_q = reinterpret_cast<const uint4*>(qf) + my_mg * KS * kTerms * 32 + lane;

    float o[NT][4], m[2], l[2];
    int rv = -200, top_rv = -200;  // the sums' value exponent, and the largest seen
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    m[0] = m[1] = -INFINITY;
    l[0] = l[1] = 0.f;

    // scores s of NJ 8-key tiles -> weights in place (f16-ready), sums and references brought up to date.
    // bad(j, e): key column e of tile j is not to be attended; `some`: there are such.
    auto weigh = [&](auto nj, auto& s, float k_scale, int ev, bool some, auto bad) {
      constexpr int NJ = decltype(nj)::value;
      if (some) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (bad(j, e)) s[j][e] = s[j][2 + e] = kLowest;
      }
      float top[2];
      bool grown = false;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float mx = kLowest;
#pragma unroll
        for (int j = 0; j < NJ; ++j) mx = fmaxf(mx, fmaxf(s[j][2 * h], s[j][2 * h + 1]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        top[h] = mx * (cf[h] * k_scale);
        grown |= top[h] > m[h] + kPGrow;
      }
      top_rv = max(top_rv, ev);
      const int want_rv = ev > rv || ev < rv - 10 ? max(ev, top_rv - 40) : rv;
      if (__any_sync(0xffffffffu, grown) || want_rv != rv) {
        const float fv = rv <= -200 ? 0.f : kv8_exp2i(min(max(rv - want_rv, -126), 126));
        rv = want_rv;
        float f[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float mn = top[h] > m[h] + kPGrow ? top[h] : m[h];
          const float a = m[h] == mn ? 1.f : ex2(m[h] - mn);
          m[h] = mn;
          l[h] *= a;
          f[h] = a * fv;
        }
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] *= f[e >> 1];
      }
      const int dv = max(ev - rv, -60);  // <= 0
      const float back = kv8_exp2i(-dv);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float c = cf[h] * k_scale, off = kPScale + float(dv) - m[h];
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) s[j][2 * h + e] = ex2(fmaf(s[j][2 * h + e], c, off));
      }
      if (some) {
#pragma unroll
        for (int j = 0; j < NJ; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (bad(j, e)) s[j][e] = s[j][2 + e] = 0.f;
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < NJ; ++j) sum += s[j][2 * h] + s[j][2 * h + 1];
        l[h] = fmaf(sum, back, l[h]);
      }
    };

    // ---- the block's own rows, 16 at a time: the first by the lane behind the unit's last tile, while the
    // others begin with the cached rows
    if (last && p.blk_k) {
      auto block_tile = [&](int kb) {
        const uint2* kf = reinterpret_cast<const uint2*>(buf) + lane;
        const uint2* vf = kf + 2 * KS * kTerms * 32;
        const float* ex = reinterpret_cast<const float*>(reinterpret_cast<uint32_t*>(buf) + kBlockWords - 32);
        float s[2][4];
        zero(s);
#pragma unroll 4
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int tq = 0; tq < kTerms; ++tq) {
            uint4 q;
            q = my_q[((ks) * kTerms + tq) * 32];
#pragma unroll
            for (int tk = 0; tk < kTerms; ++tk)
#pragma unroll
              for (int j = 0; j < 2; ++j) {
                const uint2 k = kf[((j * KS + ks) * kTerms + tk) * 32];
                mma(s[j], q, k.x, k.y);
              }
          }
        float ev = -200.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) ev = kb + r < p.block ? fmaxf(ev, ex[16 + r]) : ev;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = ex[4 * cq + 2 * j + e];
            s[j][e] *= f;
            s[j][2 + e] *= f;
          }
        weigh(std::integral_constant<int, 2>(), s, 1.f, int(ev), kb + 16 > p.block,
              [&](int j, int e) { return kb + 4 * cq + 2 * j + e >= p.block; });
        uint4 pf[kTerms];
        uint32_t f[4][kTerms];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int j = i >> 1;
          const float f0 = ex2(ex[16 + 4 * cq + 2 * j] - ev), f1 = ex2(ex[16 + 4 * cq + 2 * j + 1] - ev);
          weight_terms(s[j][2 * (i & 1)] * f0, s[j][2 * (i & 1) + 1] * f1, f[i]);
        }
#pragma unroll
        for (int t = 0; t < kTerms; ++t) pf[t] = make_uint4(f[0][t], f[1][t], f[2][t], f[3][t]);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float lo[1][4];
          zero(lo);
#pragma unroll
          for (int tv = 0; tv < kTerms; ++tv) {
            const uint2 v = vf[(n * kTerms + tv) * 32];
            mma(o[n], pf[0], v.x, v.y);
            mma(lo[0], pf[1], v.x, v.y);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) o[n][e] = fmaf(lo[0][e], kWeightLo, o[n][e]);
        }
      };
      for (int kb = 0; kb < p.block; kb += 16) {
        if (kb > 0) {
          __syncthreads();
          float x[2][VB] = {};
          load_block(kb, x[0], x[1]);
          put_block(0, x[0], x[1]);
          __syncthreads();
        }
        if (my_tl == (a1 + kb / 16) % tl) block_tile(kb);
      }
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
      const uint8_t* kt = smem + st * 2 * kKeyBytes;
      const uint8_t* vt = kt + kKeyBytes;
      if (any) {
        float s[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
        // scores: column n of key tile j is key 16 * (n / 2) + 2 j + n % 2, so that a thread ends up with
        // the 16 keys whose codes of one value column lie together
        const uint8_t* krow = kt + (16 * (gq >> 1) + (gq & 1)) * HD;
        // four key tiles at a time: their products are independent, a chain's steps are four products apart
#pragma unroll 1
        for (int ch = 0; ch < CH; ++ch) {
          const uint32_t chunk = HD == 64 ? cq : 2 * cq + (ch & 1);
#pragma unroll
          for (int j4 = 0; j4 < 8; j4 += 4) {
            uint4 k[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int t = 2 * (j4 + j);  // its token is 16 * (gq / 2) + t + gq % 2
              const uint32_t at = HD == 64 ? chunk : (chunk ^ ((t & 7) | (gq & 1))) + (ch >> 1) * 8;
              k[j] = *reinterpret_cast<const uint4*>(krow + t * HD + at * 16);
            }
#pragma unroll
            for (int tq = 0; tq < kTerms; ++tq) {
              float t4[4][4];
              zero(t4);
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint4 q;
                q = my_q[((ch * 4 + w) * kTerms + tq) * 32];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  uint32_t b0, b1;
                  e4m3x4_to_f16(w == 0 ? k[j].x : w == 1 ? k[j].y : w == 2 ? k[j].z : k[j].w, b0, b1);
                  mma(t4[j], q, b0, b1);
                }
              }
#pragma unroll
              for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[j4 + j][e] += t4[j][e];
            }
          }
        }
        if (mg == 1 && refill) {  // the keys are used up
          __syncwarp();
          if (lane == 0) fetch(st, 0, cur, next_pg);
        }
        ok = mbar_wait(full + 2 * st + 1, (i / S) & 1);
        weigh(std::integral_constant<int, 8>(), s, k_scale, kv8_exponent(scales[st].y), nv < kTile,
                                     [&](int j, int e) { return 16 * cq + 2 * j + e >= nv; });
        uint4 pf[4][kTerms];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t f[4][kTerms];
#pragma unroll
          for (int x = 0; x < 4; ++x)
            weight_terms(s[2 * w + (x >> 1)][2 * (x & 1)], s[2 * w + (x >> 1)][2 * (x & 1) + 1], f[x]);
#pragma unroll
          for (int t = 0; t < kTerms; ++t) pf[w][t] = make_uint4(f[0][t], f[1][t], f[2][t], f[3][t]);
        }
        // values: columns 8 n + gq, this thread's 16 keys. Codes behind the length are cleared: a weight of
        // zero would not take a NaN there out
        const uint8_t* vrow = vt + gq * kTile + cq * 16;
#pragma unroll
        for (int n4 = 0; n4 < NT; n4 += 4) {
          uint4 v[4];
#pragma unroll
          for (int n = 0; n < 4; ++n) v[n] = *reinterpret_cast<const uint4*>(vrow + (n4 + n) * 8 * kTile);
          if (nv < kTile) {
            uint32_t keep[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int k = nv - (16 * cq + 4 * w);
              keep[w] = k >= 4 ? 0xffffffffu : k <= 0 ? 0u : (1u << (8 * k)) - 1u;
            }
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              v[n].x &= keep[0];
              v[n].y &= keep[1];
              v[n].z &= keep[2];
              v[n].w &= keep[3];
            }
          }
          float t4[4][4], lo[4][4];
          zero(t4);
          zero(lo);
#pragma unroll
          for (int w = 0; w < 4; ++w)
#pragma unroll
            for (int n = 0; n < 4; ++n) {
              uint32_t b0, b1;
              e4m3x4_to_f16(w == 0 ? v[n].x : w == 1 ? v[n].y : w == 2 ? v[n].z : v[n].w, b0, b1);
              mma(t4[n], pf[w][0], b0, b1);
              mma(lo[n], pf[w][1], b0, b1);
            }
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[n4 + n][e] += fmaf(lo[n][e], kWeightLo, t4[n][e]);
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

    // ---- the unit's sums into those of the first lane that had a tile: lane number x from there
    const int x_tl = (my_tl - a0 % tl + tl) % tl;
    const int busy = min(tl, a1 - a0 + (last && p.blk_k ? (p.block + 15) / 16 : 0));
    const int wrow = warp * kWarpRows;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = l[h];
      x += __shfl_xor_sync(0xffffffffu, x, 1);
      x += __shfl_xor_sync(0xffffffffu, x, 2);
      if (cq == 0) ml[wrow + h * 8 + gq] = make_float4(m[h], x, float(rv), 0.f);
    }
    __syncthreads();
    float M[2], W[2], E = -200.f;
    for (int t = 0; t < tl; ++t) E = fmaxf(E, ml[(my_mg * tl + t) * kWarpRows].z);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4* row = ml + my_mg * tl * kWarpRows + h * 8 + gq;
      float a = -INFINITY, w = 0.f;
      for (int t = 0; t < tl; ++t) a = fmaxf(a, row[t * kWarpRows].x);
      const float ref = a == -INFINITY ? 0.f : a;
      for (int t = 0; t < tl; ++t) w = fmaf(row[t * kWarpRows].y, ex2(row[t * kWarpRows].x - ref), w);
      M[h] = a;
      W[h] = w;
      const float f = ex2(m[h] - ref + fmaxf(float(rv) - E, -126.f));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        o[n][2 * h] *= f;
        o[n][2 * h + 1] *= f;
      }
    }
    for (int half = tl / 2; half >= 1; half /= 2) {
      if (half >= busy) continue;
      float4* slot = reinterpret_cast<float4*>(buf) + (my_mg * half + x_tl % half) * (kWarpRows * HD / 4) + lane;
      if (x_tl >= half && x_tl < min(2 * half, busy)) {
#pragma unroll
        for (int n = 0; n < NT; ++n)
          slot[n * 32] = make_float4(o[n][0], o[n][1], o[n][2], o[n][3]);
      }
      __syncthreads();
      if (x_tl < half && x_tl + half < busy) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          const float4 x = slot[n * 32];
          o[n][0] += x.x;
          o[n][1] += x.y;
          o[n][2] += x.z;
          o[n][3] += x.w;
        }
      }
      __syncthreads();
    }
    if (x_tl == 0) {
      const int slot = 2 * blockIdx.x + (a0 == 0 && un.t > 0 ? 0 : 1);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = my_mg * kWarpRows + h * 8 + gq;
        if (whole) {
          if (r >= n_rows) continue;
          const int rr = r0 + r;
          float* out = static_cast<float*>(p.out) +
                   ((int64_t(un.b) * p.block + rr % p.block) * p.n_heads + g * group + rr / p.block) * HD + 2 * cq;
          const float inv = W[h] == 0.f ? 0.f : 1.f / W[h], fe = kv8_exp2i(max(int(E), -126));
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            const float y0 = W[h] == 0.f ? 0.f : o[n][2 * h] * inv * fe;
            const float y1 = W[h] == 0.f ? 0.f : o[n][2 * h + 1] * inv * fe;
            *reinterpret_cast<float2*>(out + 8 * n) = make_float2(y0, y1);
          }
        } else {
          float* dst = pl.sp.part + (int64_t(slot) * cta_rows + r) * HD + 2 * cq;
#pragma unroll
          for (int n = 0; n < NT; ++n)
            *reinterpret_cast<float2*>(dst + 8 * n) = make_float2(o[n][2 * h], o[n][2 * h + 1]);
          if (cq == 0) pl.sp.ml[int64_t(slot) * cta_rows + r] = make_float4(M[h], W[h], E, 0.f);
        }
      }
    }
    a0 = a1;
  }
}

constexpr int kCombineWarps = 8;

template <int V>
__device__ __forceinline__ void load_part(const float* p, float (&x)[V]) {
#pragma unroll
  for (int i = 0; i < V; i += 2) {
    const float2 v = *reinterpret_cast<const float2*>(p + i);
    x[i] = v.x;
    x[i + 1] = v.y;
  }
}

// Joins the units that were cut: CTA (i, y) looks at the cut between ranges i and i + 1; if it is its unit's
// first, it joins the unit's rows y * 8 .. y * 8 + 7, a warp each: the partial sums of its ranges in
// order, then the division and the one rounding to T.
template <typename T, int HD>
__global__ void __launch_bounds__(kCombineWarps * 32) kv8_attn_combine_kernel(const AttnArgs p, const KvSplit sp) {
  constexpr int V = HD / 32;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x, r = blockIdx.y * kCombineWarps + warp;
  asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the ranges run: see all that they wrote
  // everything that a unit of two ranges needs is asked for at once. Range i's part is its last (slot 2 i + 1),
  // the others' their first (slot 2 k)
  const int4 at = sp.places[i + 1];  // sequence, unit, tile, tiles
  const int x = sp.cuts[i + 1], end = sp.cuts[sp.ctas];
  int c0 = sp.cuts[min(i + lane, sp.ctas)], c1 = sp.cuts[min(i + lane + 1, sp.ctas)];
  const int row = min(r, sp.cta_rows - 1);
  auto slot_of = [&](int k) { return int64_t(k == i ? 2 * i + 1 : 2 * min(k, sp.ctas - 1)) * sp.cta_rows + row; };
  float4 w = sp.ml[slot_of(i + lane)];
  float p0[V], p1[V];
  load_part<V>(sp.part + slot_of(i) * HD + lane * V, p0);
  load_part<V>(sp.part + slot_of(i + 1) * HD + lane * V, p1);
  const int u0 = x - at.z, u1 = u0 + at.w;
  if (x >= end || at.z == 0 || __shfl_sync(0xffffffffu, c0, 0) > u0) return;
  const int g = at.y / sp.row_blocks, r0 = (at.y % sp.row_blocks) * sp.cta_rows;
  if (r >= min(sp.cta_rows, sp.rows - r0)) return;
  // 32 ranges at a time, a lane each; empty ranges have no part
  float M = -INFINITY, E = -200.f, l = 0.f, o[V];
#pragma unroll
  for (int j = 0; j < V; ++j) o[j] = 0.f;
  for (int base = i;;) {
    const bool mine = c0 < c1 && c0 < u1;
    if (!mine) w = make_float4(-INFINITY, 0.f, -200.f, 0.f);
    const float M2 = fmaxf(M, kv8_warp_max(w.x)), E2 = fmaxf(E, kv8_warp_max(w.z));
    const float ref = M2 == -INFINITY ? 0.f : M2;
    const float keep = ex2(M - ref) * ex2(fmaxf(E - E2, -126.f));
    l *= ex2(M - ref);
#pragma unroll
    for (int j = 0; j < V; ++j) o[j] *= keep;
    M = M2;
    E = E2;
    const float f = mine ? ex2(w.x - ref) : 0.f, fo = f * ex2(fmaxf(w.z - E, -126.f));
    l += kv8_warp_sum(w.y * f);
    unsigned parts = __ballot_sync(0xffffffffu, mine);
    if (base == i) {
      const float f0 = __shfl_sync(0xffffffffu, fo, 0), f1 = __shfl_sync(0xffffffffu, fo, 1);
#pragma unroll
      for (int v = 0; v < V; ++v) {
        o[v] = fmaf(p0[v], f0, o[v]);
        if (parts & 2) o[v] = fmaf(p1[v], f1, o[v]);
      }
      parts &= ~3u;
    }
    while (parts) {  // eight parts in flight
      float y[8][V], fj[8];
#pragma unroll
      for (int n = 0; n < 8; ++n) {
        const int j = parts ? __ffs(parts) - 1 : 0;
        fj[n] = __shfl_sync(0xffffffffu, fo, j);
        if (parts) {
          load_part<V>(sp.part + slot_of(base + j) * HD + lane * V, y[n]);
        } else {
          fj[n] = 0.f;
#pragma unroll
          for (int v = 0; v < V; ++v) y[n][v] = 0.f;
        }
        parts &= parts - 1;
      }
#pragma unroll
      for (int n = 0; n < 8; ++n)
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = fmaf(y[n][v], fj[n], o[v]);
    }
    if (__shfl_sync(0xffffffffu, c1, 31) >= u1) break;  // the unit's last tile lies in these ranges
    base += 32;
    c0 = sp.cuts[min(base + lane, sp.ctas)];
    c1 = sp.cuts[min(base + lane + 1, sp.ctas)];
    w = sp.ml[slot_of(base + lane)];
  }
  const int rr = r0 + r, group = p.n_heads / p.n_kv;
  T* out = static_cast<T*>(p.out) +
           ((int64_t(at.x) * p.block + rr % p.block) * p.n_heads + g * group + rr / p.block) * HD + lane * V;
  const float inv = 1.f / l, fe = kv8_exp2i(max(int(E), -126));
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = st_f<T>(l == 0.f ? 0.f : o[j] * inv * fe);
}

constexpr int kMmaSmemMax = 232448;  // 227 KB

struct MmaShape {
  int mg, row_blocks, cta_rows;
};
// Query rows of a KV head -> warps per tile: 16 rows each, up to 128 rows (64 at head_dim 256).
MmaShape mma_shape(int rows, int hd) {
  MmaShape s;
  const int most = hd == 256 ? 64 : 128;
  s.mg = 1;
  while (16 * s.mg < std::min(rows, most)) s.mg *= 2;
  s.cta_rows = 16 * s.mg;
  s.row_blocks = int(ceil_div(rows, s.cta_rows));
  return s;
}

template <int HD>
int launch_mma(const AttnArgs& a, const MmaShape& sh, MmaPlan pl, int ctas, cudaStream_t s) {
  int depth = std::max(kMaxDepth, sh.mg);
  while (depth > 1 && mma_smem(HD, sh.mg, depth, a.batch).bytes > kMmaSmemMax) --depth;
  const int smem = mma_smem(HD, sh.mg, depth, a.batch).bytes;
  if (smem > kMmaSmemMax) return DSM_ERR_UNSUPPORTED;
  pl.depth = depth;
  auto k = kv8_attn_mma_kernel<HD>;
  // all that a CTA may have, whatever this call takes: the kernel's limit is every host thread's
  if (cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kMmaSmemMax) != cudaSuccess)
    return check_launch("gqa_attn_kv8 smem attribute");
  k<<<unsigned(ctas), mma_warps(HD) * 32, size_t(smem), s>>>(a, pl);
  const int st = check_launch("gqa_attn_kv8");
  return st != DSM_OK ? st : kv8_combine(a, pl.sp, HD, DSM_DT_F32, s);
}

size_t mma_ws_bytes(int cta_rows, int hd) { return split_ws_bytes(num_sms(), cta_rows, hd); }

int run_mma(const AttnArgs& a, int hd, void* ws, cudaStream_t s) {
  const MmaShape sh = mma_shape(a.n_heads / a.n_kv * a.block, hd);
  const int64_t most = int64_t(a.batch) * a.max_pages * (a.page / kTile) * a.n_kv * sh.row_blocks;
  const int ctas = int(std::min<int64_t>(num_sms(), most));
  MmaPlan pl;
  pl.mg = sh.mg;
  pl.sp.row_blocks = sh.row_blocks;
  pl.sp.rows = a.n_heads / a.n_kv * a.block;
  pl.sp.cta_rows = sh.cta_rows;
  pl.sp.cost = kUnitCost;
  pl.sp.snap = std::max(1, mma_warps(hd) / sh.mg / 2);
  pl.sp.least = kUnitCost;
  pl.sp.ctas = ctas;
  if (!split_fits(a, pl.sp)) return DSM_ERR_UNSUPPORTED;
  pl.depth = 0;
  pl.vec_q = vec_ok(a.q, a.q_batch, a.q_row, a.q_head, 16);
  pl.vec_blk = a.blk_k && vec_ok(a.blk_k, a.bk_batch, a.bk_head, a.bk_row, 16) &&
               vec_ok(a.blk_v, a.bv_batch, a.bv_head, a.bv_row, 16);
  split_ws(pl.sp, ws, hd);
  switch (hd) {
    case 64: return launch_mma<64>(a, sh, pl, ctas, s);
    case 128: return launch_mma<128>(a, sh, pl, ctas, s);
    default: return launch_mma<256>(a, sh, pl, ctas, s);
  }
}

}  // namespace

int kv8_combine(const AttnArgs& a, const KvSplit& sp, int hd, int dtype, cudaStream_t s) {
  // a unit of up to 2 * snap tiles is never cut
  if (sp.ctas == 1 || a.max_pages * (a.page / kTile) <= 2 * sp.snap) return DSM_OK;
  const dim3 grid(unsigned(sp.ctas - 1), unsigned(ceil_div(std::min(sp.cta_rows, sp.rows), kCombineWarps)));
  const bool bf = dtype == DSM_DT_BF16;
  using B = __nv_bfloat16;
  auto k = hd == 64    ? (bf ? kv8_attn_combine_kernel<B, 64> : kv8_attn_combine_kernel<float, 64>)
           : hd == 128 ? (bf ? kv8_attn_combine_kernel<B, 128> : kv8_attn_combine_kernel<float, 128>)
                       : (bf ? kv8_attn_combine_kernel<B, 256> : kv8_attn_combine_kernel<float, 256>);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(kCombineWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k, a, sp);
  if (e != cudaSuccess) return fail(DSM_ERR_CUDA, std::string("gqa_attn_kv8 combine: ") + cudaGetErrorString(e));
  return check_launch("gqa_attn_kv8 combine");
}

}  // namespace dsm

using namespace dsm;

extern "C" size_t dsm_gqa_attn_kv8_workspace_bytes(int batch, int block, int n_heads, int n_kv, int head_dim) {
  if (batch <= 0 || batch > kKv8MaxBatch || block <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0 ||
      int64_t(block) * n_heads > 0x7fffffff || !kv8_head_dim_ok(head_dim))
    return 0;
  const int rows = n_heads / n_kv * block;
  return std::max(mma_ws_bytes(mma_shape(rows, head_dim).cta_rows, head_dim), kv8_umma_ws_bytes(rows, head_dim));
}

extern "C" int dsm_gqa_attn_kv8(const dsm_kv8_attn_desc* d, const void* q, const int32_t* block_table,
                                const int32_t* lengths, const void* blk_k, const void* blk_v, void* out, void* ws,
                                size_t ws_bytes, void* stream) {
  DSM_REQUIRE(d != nullptr, "dsm_gqa_attn_kv8: desc is NULL");
  DSM_REQUIRE(d->batch >= 0 && d->batch <= kKv8MaxBatch, "dsm_gqa_attn_kv8: batch must be 0..8192");
  DSM_REQUIRE(d->block > 0 && d->n_kv > 0 && d->n_heads > 0 && d->n_heads % d->n_kv == 0,
              "dsm_gqa_attn_kv8: bad shape (n_heads must be a multiple of n_kv)");
  DSM_REQUIRE(int64_t(d->block) * d->n_heads <= 0x7fffffff, "dsm_gqa_attn_kv8: too many rows");
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
  // fp32 results are stored two at a time
  DSM_REQUIRE(d->dtype != DSM_DT_F32 || reinterpret_cast<uintptr_t>(out) % 8 == 0,
              "dsm_gqa_attn_kv8: an fp32 out must be 8-byte aligned");
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
  if (attn_kernel() == 0) {
    int st = DSM_ERR_UNSUPPORTED;
    if (d->dtype == DSM_DT_F32)
      st = run_mma(a, d->head_dim, ws, s);
    else if (d->block <= kUmmaMaxBlock)
      st = kv8_umma(a, d->head_dim, ws, s);
    if (st != DSM_ERR_UNSUPPORTED) return st;
  }
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
