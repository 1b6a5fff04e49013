// The attention over the paged 8-bit cache for bf16 rows, on tcgen05 (dsm_gqa_attn_kv8, layout in
// kv8.cuh).
//
// Mathematics. Everything is taken transposed, so that the keys and the values are the 128-row operands
// as they are stored and the query rows (4 to 64 per KV head) are the narrow one:
//   s [128 keys, rows] = k [128 keys, head_dim] q^T     o [head_dim, rows] += v^T [head_dim, 128 keys] p^T
// kind::f8f6f4 multiplies the e4m3 codes themselves. q, scaled per row by a power of two to at most
// 448, is the sum of two e4m3 terms (hi = e4m3(x), lo = e4m3(x - hi): exact for bf16's 8 bits wherever
// the residual reaches e4m3's normals, 2^-10 of a unit off elsewhere, of a row maximum of 224 to 448).
// The weights are p = 2^(s - m + 8), an e4m3 term and an e5m2 residual: 2^-7 of a weight off at most, and
// nothing above 2^-25 of the largest is lost. m is the row's reference: its maximum when it was last
// set, plus one; it is set again when a weight would pass 2^8.75, and the sums in tensor memory are then
// rescaled. The page's value exponent is folded into the weights relative to a reference rv that moves
// when an exponent leaves [rv - 10, rv]; the scores' page factor is one per thread. Scores, sums and weights'
// sums are fp32. The block's own rows take fp32 products on CUDA cores: they are few.
//
// What bounds it: reading 2 * head_dim bytes per key and KV head. At the copy peak an SM gets 128 keys of
// head_dim 128 per ~1400 cycles; their products take ~300 cycles of the tensor cores for 32 rows, the
// shared-memory traffic ~1000, the softmax ~420 instructions of each of four warps. mma.sync runs e4m3
// operands as f16 products with the conversions around every one, and f16 fragments converted once per warp
// need 1,700 unrolled instructions per 64 keys and 32 rows, which the instruction cache does not hold
// (measured: 116 us for 131,071 keys x 8 heads x 20 rows, against 41 us for the bytes).
//
// Layout. Two CTAs per SM (one at head_dim 256), each over its range of the line of units (kv8_attn.cuh),
// 128 keys a step:
//   warps 0-3  softmax: thread = key for the weights, thread = column for the result
//   warp 4     producer: pages from the block table, 64 keys each; bulk copies (keys of head_dim 128,
//              stored in the operand's 128-byte swizzle) and TMA boxes (the rest, swizzled on the way)
//   warp 5     one thread issues the products: scores of step i + 1 before the sums of step i
#include <algorithm>
#include <mutex>

#include "kv8_attn.cuh"
#include "tcgen05.cuh"

namespace dsm {
namespace {

using B16 = __nv_bfloat16;

constexpr int kThreads = 192;
constexpr int kStepKeys = 128;
constexpr float kPExp = 8.f;   // weights at the reference: 2^8
constexpr float kPMax = 8.75f;  // 2^8.75 = 431 still fits e4m3
constexpr float kPHead = 1.f;  // a new reference lies this much above the maximum

__host__ __device__ constexpr int mma_cols(int nr) { return nr <= 16 ? 16 : nr <= 32 ? 32 : 64; }
__host__ __device__ constexpr int weight_buffers(int nr) { return nr > 32 ? 1 : 2; }

template <int HD, int NR>
struct Cfg {
  static constexpr int NM = mma_cols(NR);               // columns of the products
  static constexpr int NH = HD <= 128 ? 1 : 2;          // 128-row halves of the output
  static constexpr int CTAS = HD == 256 ? 1 : 2;        // per SM
  static constexpr int PB = weight_buffers(NR);         // buffers of weights
  static constexpr int kHalf = kTile * HD;              // bytes of 64 keys, or of their values
  static constexpr int kStage = 4 * kHalf;              // keys, then values, of 128
  static constexpr int kQTerm = NM * HD;                // bytes of one term of q
  static constexpr int kPTerm = NM * kStepKeys;         // bytes of one term of the weights
  static constexpr int kCols = 2 * NM + NH * NM;        // tensor memory: two score buffers, the sums
  static constexpr int kAlloc = kCols <= 64 ? 64 : kCols <= 128 ? 128 : 256;
};

struct UmmaPlan {
  KvSplit sp;
  int stages;
  bool vec_q, vec_blk;
};

struct UmmaSmem {
  int q, p, w, rows, info, bars, sums, P, bytes;
};
// per row: c (score factor), m (reference), a (rescaling), mb / lb (the block's maximum and weight), and four
// warps' partial results
constexpr int kRowFloats = 9;
__host__ __device__ inline UmmaSmem umma_smem(int hd, int nr, int stages, int block, int batch) {
  UmmaSmem s;
  const int nm = mma_cols(nr), pb = weight_buffers(nr);
  s.q = stages * 4 * kTile * hd;
  s.p = s.q + 2 * nm * hd;
  s.w = s.p + pb * 2 * nm * kStepKeys;
  s.rows = s.w + block * nr * 4;
  s.info = s.rows + kRowFloats * nr * 4;
  s.info = (s.info + 15) / 16 * 16;
  s.bars = s.info + stages * 16;
  s.sums = s.bars + (2 * stages + 10) * 8;
  s.P = s.sums + 64;
  s.bytes = 1024 + s.P + (batch + 1) * 4;  // the start is moved to 1024 bytes
  return s;
}

// ---- PTX -------------------------------------------------------------------------------
__device__ __forceinline__ void tma_2d(uint32_t dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(smem_u32(bar))
      : "memory");
}
// K-major operand of 64-byte rows in the 64-byte swizzle: 8-row groups at 512 B
__device__ __forceinline__ uint64_t desc_sw64(uint32_t saddr) {
  return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(1) << 16) | (uint64_t(512 >> 4) << 32) | (uint64_t(1) << 46) |
         (uint64_t(4) << 61);
}
// the weights, rows of 16, 32 or 64 bytes per key (the operand's N dimension contiguous): 16-byte rows
// unswizzled with groups of 8 keys at 128 B (the leading offset), 32- and 64-byte rows in the swizzle of their
// width with groups of 8 keys at 256 and 512 B (the stride)
template <int NM>
__device__ __forceinline__ uint64_t desc_weights(uint32_t saddr) {
  constexpr uint64_t lead = NM == 16 ? 128 >> 4 : 1, stride = NM == 16 ? 128 >> 4 : 8 * NM >> 4;
  constexpr uint64_t swizzle = NM == 16 ? 0 : NM == 32 ? 6 : 4;
  return uint64_t((saddr >> 4) & 0x3FFFu) | (lead << 16) | (stride << 32) | (uint64_t(1) << 46) | (swizzle << 61);
}
// kind::f8f6f4: D f32, A e4m3 K-major, B e4m3 or e5m2, K-major or (b_rows) N-major
__device__ __forceinline__ uint32_t idesc_f8(int n, bool b_e5m2, bool b_rows) {
  return (1u << 4) | (b_e5m2 ? 1u << 10 : 0u) | (b_rows ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) |
         (uint32_t(128 >> 4) << 24);
}
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, bool accumulate) {
  const uint32_t no_mask = 0u, acc = accumulate ? 1u : 0u;
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n}" ::"r"(d_tmem),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(acc), "r"(no_mask)
      : "memory");
}
// this thread's lane: N consecutive columns
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t addr, float* x) {
  if constexpr (N >= 16) {
    uint32_t r[16];
    tc::tmem_ld16(addr, r);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = __uint_as_float(r[i]);
    if constexpr (N > 16) tmem_ld<N - 16>(addr + 16, x + 16);
  } else if constexpr (N >= 8) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(r[i]);
    if constexpr (N > 8) tmem_ld<N - 8>(addr + 8, x + 8);
  } else {
    uint32_t r[4];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = __uint_as_float(r[i]);
  }
}
__device__ __forceinline__ bool any_of_softmax(bool x) {  // over the four softmax warps, with a barrier
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n barrier.cta.red.or.pred q, 1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(x ? 1u : 0u)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void softmax_sync() { asm volatile("barrier.cta.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ float redux_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
// four weights -> an e4m3 term and an e5m2 residual, four bytes each, x0 lowest. They pass through f16,
// whose 11 bits are more than the two terms keep.
__device__ __forceinline__ void weight_terms(float x0, float x1, float x2, float x3, uint32_t& hi, uint32_t& lo) {
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
      " cvt.rn.satfinite.e5m2x2.f16x2 c, x;\n"
      " cvt.rn.satfinite.e5m2x2.f16x2 d, y;\n"
      " mov.b32 %1, {c, d};\n}"
      : "=&r"(hi), "=&r"(lo)
      : "f"(x0), "f"(x1), "f"(x2), "f"(x3));
}
__device__ __forceinline__ void store_words(uint32_t at, const uint32_t (&w)[4], int n) {  // n is a constant
  if (n == 4)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
  else if (n == 2)
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(w[0]), "r"(w[1]) : "memory");
  else
    asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(w[0]) : "memory");
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("add.rn.f32x2 %0, %1, %2;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
// four values of a query row -> two e4m3 terms
__device__ __forceinline__ void q_terms(const float* x, uint32_t& hi, uint32_t& lo) {
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

// One CTA's part of a unit: tiles [t0, t1) of sequence b's KV head g, query rows [r0, r0 + n_rows)
struct Segment {
  Place un;
  int t0, t1, steps, g, r0, n_rows, len;
  bool last, whole;
};

template <int HD, int NR>
__global__ void __launch_bounds__(kThreads, Cfg<HD, NR>::CTAS)
    kv8_umma_kernel(const AttnArgs p, const UmmaPlan pl, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<HD, NR>;
  constexpr int NM = C::NM;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const UmmaSmem L = umma_smem(HD, NR, pl.stages, p.blk_k ? p.block : 0, p.batch);
  const int S = pl.stages;
  float* W = reinterpret_cast<float*>(smem + L.w);  // [block][NR] weights of the block's own rows
  float* row_c = reinterpret_cast<float*>(smem + L.rows);
  float* row_m = row_c + NR;
  float* row_a = row_m + NR;
  float* row_mb = row_a + NR;
  float* row_lb = row_mb + NR;
  float* red = row_lb + NR;  // [4][NR]
  float4* info = reinterpret_cast<float4*>(smem + L.info);  // per stage: key and value scale of each half
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* empty = full + S;
  uint64_t* s_full = empty + S;    // [2]
  uint64_t* s_empty = s_full + 2;  // [2]
  uint64_t* p_full = s_empty + 2;  // [2]
  uint64_t* p_empty = p_full + 2;  // [2]
  uint64_t* q_full = p_empty + 2;
  uint64_t* o_full = q_full + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + L.sums + 32);
  int* P = reinterpret_cast<int*>(smem + L.P);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hr = p.n_kv * pl.sp.row_blocks;
  if (tid == 0) {
    for (int i = 0; i < S; ++i) {
      mbar_init(full + i, 2);  // the copies' expect_tx, and the scales
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(s_full + i, 1);
      mbar_init(s_empty + i, 4);
      mbar_init(p_full + i, 4);
      mbar_init(p_empty + i, 1);
    }
    mbar_init(q_full, 4);
    mbar_init(o_full, 1);
    fence_mbar_init();
  }
  if (warp == 5) tc::tmem_alloc(slot, C::kAlloc);
  scan_tiles<kThreads>(p, P, reinterpret_cast<int*>(smem + L.sums));
  int start;
  const int n_tiles = my_range(p, P, pl.sp, start);
  if (blockIdx.x == 0)
    for (int b = tid; b < p.batch; b += kThreads)
      if (p.lengths[b] > int64_t(p.max_pages) * p.page) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot, t_o = tmem + 2 * NM;

  auto segment = [&](int a0) {
    Segment s;
    s.un = place_of(P, p.batch, hr, start + a0, 0);
    s.t0 = s.un.t;
    s.t1 = min(s.un.T, s.un.t + n_tiles - a0);
    s.last = s.t1 == s.un.T;
    s.whole = s.last && s.t0 == 0;
    s.g = s.un.u / pl.sp.row_blocks;
    s.r0 = (s.un.u % pl.sp.row_blocks) * NR;
    s.n_rows = min(NR, pl.sp.rows - s.r0);
    s.len = seq_len(p, s.un.b);
    s.steps = s.len == 0 ? 0 : (s.t1 - s.t0 + 1) / 2;
    return s;
  };
  bool ok = true;  // no wait has run out; after one has, loops go through without waiting, copying or multiplying

  if (warp == 4) {
    // ---------------------------------------------------------------- producer
    int k = 0;  // steps so far
    for (int a0 = 0; a0 < n_tiles;) {
      const Segment sg = segment(a0);
      a0 += sg.t1 - sg.t0;
      const int tiles = sg.steps == 0 ? 0 : sg.t1 - sg.t0;
      for (int base = 0; base < tiles; base += 32) {
        // a lane per tile: its page, then its scales (used when the first copies are on their way)
        const int t = sg.t0 + base + lane;
        int pg = -1;
        if (base + lane < tiles) {
          pg = __ldg(p.table + int64_t(sg.un.b) * p.table_stride + t * kTile / p.page);
          if (pg < 0 || pg >= p.n_pages) {
            raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
            pg = -1;
          }
        }
        float ks = __int_as_float(0x7fc00000), vs = 1.f;  // NaN marks a half without keys
        if (pg >= 0) {
          ks = __ldg(p.k_scale + int64_t(pg) * p.n_kv + sg.g);
          vs = __ldg(p.v_scale + int64_t(pg) * p.n_kv + sg.g);
        }
        for (int i = 0; i < min(32, tiles - base); i += 2, ++k) {
          const int st = k % S;
          if (ok && k >= S) ok = mbar_wait(empty + st, (k / S - 1) & 1);
          const int pg0 = __shfl_sync(0xffffffffu, pg, i), pg1 = __shfl_sync(0xffffffffu, pg, i + 1);
          if (lane == 0 && ok) {
            mbar_arrive_expect_tx(full + st, ((pg0 >= 0) + (pg1 >= 0)) * 2 * C::kHalf);
            const uint32_t kdst = smem_u32(smem) + st * C::kStage, vdst = kdst + 2 * C::kHalf;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int page = h ? pg1 : pg0;
              if (page < 0) continue;
              const int64_t ph = int64_t(page) * p.n_kv + sg.g;
              const int sub = ((sg.t0 + base + i + h) * kTile % p.page) / kTile;
              const int64_t group = ph * (p.page / kTile) + sub;  // of 64 tokens
              if constexpr (HD == 128) {
                bulk_g2s(smem + st * C::kStage + h * C::kHalf, p.k_codes + group * C::kHalf, C::kHalf, full + st,
                         policy_evict_first());
              } else if constexpr (HD == 64) {
                tma_2d(kdst + h * C::kHalf, &kmap, 0, int(group * kTile), full + st);
              } else {  // two slabs of 128 bytes
                tma_2d(kdst + h * (C::kHalf / 2), &kmap, 0, int(group * kTile), full + st);
                tma_2d(kdst + C::kHalf + h * (C::kHalf / 2), &kmap, 128, int(group * kTile), full + st);
              }
              tma_2d(vdst + h * C::kHalf, &vmap, 0, int(group * HD), full + st);
            }
          }
          const float4 sc = make_float4(__shfl_sync(0xffffffffu, ks, i), __shfl_sync(0xffffffffu, vs, i),
                                        __shfl_sync(0xffffffffu, ks, i + 1), __shfl_sync(0xffffffffu, vs, i + 1));
          if (lane == 0 && ok) {
            info[st] = sc;
            mbar_arrive(full + st);
          }
          __syncwarp();
        }
      }
    }
    // after a wait that ran out, copies may still be on their way: see them land
    if (!ok)
      for (int i = max(0, k - S); i < k; ++i) mbar_wait(full + i % S, (i / S) & 1);
  } else if (warp == 5) {
    // ---------------------------------------------------------------- products
    if (lane == 0) {
      const uint32_t id_s = idesc_f8(NM, false, false), id_hi = idesc_f8(NM, false, true), id_lo = idesc_f8(NM, true, true);
      const uint32_t base = smem_u32(smem), qa = base + L.q, pa = base + L.p;
      int k = 0, seg = 0;  // steps, and units with steps, so far
      for (int a0 = 0; a0 < n_tiles;) {
        const Segment sg = segment(a0);
        a0 += sg.t1 - sg.t0;
        if (sg.steps == 0) continue;
        if (ok) ok = mbar_wait(q_full, seg++ & 1);
        tc::tc_fence_after();
        auto sums = [&](int j, bool first) {  // step j's
          const int pb = C::PB == 2 ? j & 1 : 0, use = C::PB == 2 ? j >> 1 : j;
          if (ok) ok = mbar_wait(p_full + pb, use & 1);
          tc::tc_fence_after();
          if (!ok) return;
          const uint32_t v = base + (j % S) * C::kStage + 2 * C::kHalf, w = pa + pb * 2 * C::kPTerm;
#pragma unroll
          for (int nh = 0; nh < C::NH; ++nh)
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f8(t_o + nh * NM, desc_sw64(v + (ks >> 1) * C::kHalf + nh * 128 * 64 + (ks & 1) * 32),
                        desc_weights<NM>(w + x * C::kPTerm + ks * 32 * NM), x ? id_lo : id_hi, !first || x > 0 || ks > 0);
          tc::umma_commit(empty + j % S);
          tc::umma_commit(p_empty + pb);
        };
        for (int i = 0; i < sg.steps; ++i) {
          const int kk = k + i, st = kk % S, sb = kk & 1;
          if (ok) ok = mbar_wait(full + st, (kk / S) & 1);
          if (ok && kk >= 2) ok = mbar_wait(s_empty + sb, ((kk >> 1) - 1) & 1);
          tc::tc_fence_after();
          if (ok) {
            const uint32_t kt = base + st * C::kStage;
#pragma unroll
            for (int x = 0; x < 2; ++x)
#pragma unroll
              for (int ks = 0; ks < HD / 32; ++ks) {
                const uint64_t a = HD == 64 ? desc_sw64(kt + ks * 32)
                                            : tc::umma_desc_sw128(kt + (ks >> 2) * 2 * 64 * 128 + (ks & 3) * 32);
                const uint32_t qt = qa + x * C::kQTerm;
                const uint64_t b = HD == 64 ? desc_sw64(qt + ks * 32)
                                            : tc::umma_desc_sw128(qt + (ks >> 2) * NM * 128 + (ks & 3) * 32);
                umma_f8(tmem + sb * NM, a, b, id_s, x > 0 || ks > 0);
              }
            tc::umma_commit(s_full + sb);
          }
          if (i > 0) sums(kk - 1, i == 1);
        }
        sums(k + sg.steps - 1, sg.steps == 1);
        if (ok) tc::umma_commit(o_full);
        k += sg.steps;
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax, results
    constexpr int TPR = 8, VB = HD / TPR;  // staging: 16 rows at a time, threads per row, values per thread
    const int half = tid >> 6;             // which 64 keys of a step this thread's key is in
    const int row_r = tid / TPR, row_d = tid % TPR * VB;
    const uint32_t t_lane = uint32_t(warp * 32) << 16;
    const int group = p.n_heads / p.n_kv;
    uint8_t* const q8 = smem + L.q;
    // where this thread's key's weights go, 16 rows at a time
    uint32_t p_at[NM / 16];
#pragma unroll
    for (int c = 0; c < NM / 16; ++c)
      p_at[c] = smem_u32(smem) + L.p + tid * NM + ((c ^ (NM == 32 ? (tid >> 2) & 1 : NM == 64 ? (tid >> 1) & 3 : 0)) << 4);

    int k = 0, outs = 0;  // steps, and units with steps, so far
    for (int a0 = 0; a0 < n_tiles;) {
      const Segment sg = segment(a0);
      const bool blk = sg.last && p.blk_k;
      // ---- q's terms, and the scores of the block's own rows
      softmax_sync();  // the previous unit's row statistics are used up
      const B16* qg = static_cast<const B16*>(p.q) + sg.un.b * p.q_batch;
      const B16* bk = static_cast<const B16*>(p.blk_k) + sg.un.b * p.bk_batch + sg.g * p.bk_head + row_d;
      for (int r = row_r; r < NM; r += 16) {
        float x[VB];
#pragma unroll
        for (int i = 0; i < VB; ++i) x[i] = 0.f;
        const bool live = r < sg.n_rows;
        if (live) {
          const int rr = sg.r0 + r;
          load_vals<B16, VB>(qg + (rr % p.block) * p.q_row + (sg.g * group + rr / p.block) * p.q_head + row_d, pl.vec_q, x);
        }
        if (blk && r < NR) {
          const float f = p.scale * kLog2e;
#pragma unroll 2
          for (int j = 0; j < p.block; ++j) {
            float y[VB], s = 0.f;
            load_vals<B16, VB>(bk + j * p.bk_row, pl.vec_blk, y);
#pragma unroll
            for (int i = 0; i < VB; ++i) s = fmaf(x[i], y[i], s);
#pragma unroll
            for (int w = TPR / 2; w; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
            if (row_d == 0) W[j * NR + r] = live ? s * f : 0.f;
          }
        }
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < VB; ++i) mx = fmaxf(mx, finite_abs(x[i]));
#pragma unroll
        for (int w = TPR / 2; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const int e = kv8_scale_exp(mx);
        const float inv = kv8_exp2i(-e);
#pragma unroll
        for (int i = 0; i < VB; ++i) x[i] = scaled(x[i], inv);
        if (row_d == 0 && r < NR) {
          row_c[r] = live ? p.scale * kLog2e * kv8_exp2i(e) : 0.f;
          row_m[r] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < VB; i += 4) {
          uint32_t hi, lo;
          q_terms(x + i, hi, lo);
          const int d = row_d + i;
          uint8_t* at = HD == 64 ? q8 + r * 64 + ((((d >> 4) & 3) ^ ((r >> 1) & 3)) << 4) + (d & 15)
                                 : q8 + (d >> 7) * NM * 128 + r * 128 + ((((d >> 4) & 7) ^ (r & 7)) << 4) + (d & 15);
          *reinterpret_cast<uint32_t*>(at) = hi;
          *reinterpret_cast<uint32_t*>(at + C::kQTerm) = lo;
        }
      }
      tc::fence_async_smem();
      softmax_sync();
      if (lane == 0 && sg.steps > 0) mbar_arrive(q_full);
      if (blk && tid < NR) {  // the block's weights of row tid, relative to their maximum
        float mb = kLowest, lb = 0.f;
        for (int j = 0; j < p.block; ++j) mb = fmaxf(mb, W[j * NR + tid]);
        for (int j = 0; j < p.block; ++j) {
          const float w = ex2(W[j * NR + tid] - mb);
          W[j * NR + tid] = w;
          lb += w;
        }
        row_mb[tid] = mb;
        row_lb[tid] = lb;
      }

      // ---- the cached rows, 128 a step
      float l[NR];
#pragma unroll
      for (int r = 0; r < NR; ++r) l[r] = 0.f;
      int rv = -200, top_rv = -200;
      for (int i = 0; i < sg.steps; ++i, ++k) {
        const int st = k % S, sb = k & 1;
        if (ok) ok = mbar_wait(full + st, (k / S) & 1);
        const float4 sc = info[st];
        const int t0 = sg.t0 + 2 * i;  // first tile of the step
        const int left = sg.len - t0 * kTile;
        const int n0 = sc.x == sc.x ? max(0, min(kTile, left)) : 0;
        const int n1 = t0 + 1 < sg.t1 && sc.z == sc.z ? max(0, min(kTile, left - kTile)) : 0;
        const bool live = (tid & 63) < (half ? n1 : n0);
        const float ks = half ? sc.z : sc.x;
        const int e0 = n0 ? kv8_exponent(sc.y) : -200, e1 = n1 ? kv8_exponent(sc.w) : -200;
        const int ev = max(e0, e1), low = min(n0 ? e0 : ev, n1 ? e1 : ev);
        top_rv = max(top_rv, ev);
        const int want_rv = ev > rv || low < rv - 10 ? max(ev, top_rv - 40) : rv;
        if (ok) ok = mbar_wait(s_full + sb, (k >> 1) & 1);
        tc::tc_fence_after();
        float y[NR];
        tmem_ld<NR>(tmem + t_lane + sb * NM, y);
        tc::tmem_ld_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty + sb);
        // the weights' exponents: row_m is kPExp less the reference
        float top = kLowest;
#pragma unroll
        for (int r = 0; r < NR; r += 4) {
          const float4 c = *reinterpret_cast<const float4*>(row_c + r), m = *reinterpret_cast<const float4*>(row_m + r);
          const float2 ks2 = make_float2(ks, ks);
          const float2 a = fma2(make_float2(y[r], y[r + 1]), mul2(make_float2(c.x, c.y), ks2), make_float2(m.x, m.y));
          const float2 b = fma2(make_float2(y[r + 2], y[r + 3]), mul2(make_float2(c.z, c.w), ks2), make_float2(m.z, m.w));
          y[r] = a.x;
          y[r + 1] = a.y;
          y[r + 2] = b.x;
          y[r + 3] = b.y;
          top = fmaxf(top, fmaxf(fmaxf(y[r], y[r + 1]), fmaxf(y[r + 2], y[r + 3])));
        }
        if (any_of_softmax((live && top > kPMax) || i == 0 || want_rv != rv)) {
          // new references: every row whose maximum lies above its own (all of them at first)
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float x = redux_max(live ? y[r] : kLowest);
            if (lane == (r & 31)) red[warp * NR + r] = x;
          }
          softmax_sync();
          if (tid < NR) {
            const float x = fmaxf(fmaxf(red[tid], red[NR + tid]), fmaxf(red[2 * NR + tid], red[3 * NR + tid]));
            const float up = x == kLowest ? 0.f : i == 0 || x > kPExp ? x + (kPHead - kPExp) : 0.f;
            row_m[tid] -= up;
            red[tid] = up;
            const float fv = rv <= -200 ? 1.f : kv8_exp2i(min(max(rv - want_rv, -126), 126));
            row_a[tid] = ex2(-up) * fv;
          }
          softmax_sync();
          rv = want_rv;
          if (i > 0) {  // the sums so far, after the products that make them
            const int j = k - 1, pb = C::PB == 2 ? j & 1 : 0, use = C::PB == 2 ? j >> 1 : j;
            if (ok) ok = mbar_wait(p_empty + pb, use & 1);
            tc::tc_fence_after();
#pragma unroll
            for (int nh = 0; nh < C::NH; ++nh)
#pragma unroll 1
              for (int c = 0; c < NM && c < NR; c += 8) {
                float o[8];
                uint32_t u[8];
                const uint32_t at = t_o + t_lane + nh * NM + c;
                tmem_ld<8>(at, o);
                tc::tmem_ld_wait();
#pragma unroll
                for (int x = 0; x < 8; ++x) u[x] = __float_as_uint(o[x] * row_a[c + x]);
                asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(u[0]),
                             "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                             : "memory");
              }
            tc::tmem_st_wait();
          }
#pragma unroll
          for (int r = 0; r < NR; ++r) {
            const float up = red[r];
            if (i > 0) l[r] *= ex2(-up);
            y[r] -= up;
          }
        }
        const int dv = max((half ? e1 : e0) - rv, -60);  // <= 0
        const float fv = kv8_exp2i(dv);
#pragma unroll
        for (int r = 0; r < NR; ++r) y[r] = ex2(y[r]);
        if (!__all_sync(0xffffffffu, live)) {
#pragma unroll
          for (int r = 0; r < NR; ++r) y[r] = live ? y[r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < NR; r += 2) {
          const float2 a = add2(make_float2(l[r], l[r + 1]), make_float2(y[r], y[r + 1]));
          l[r] = a.x;
          l[r + 1] = a.y;
        }
        if (dv != 0) {
#pragma unroll
          for (int r = 0; r < NR; ++r) y[r] *= fv;
        }
        const int pb = C::PB == 2 ? k & 1 : 0, use = C::PB == 2 ? k >> 1 : k;
        if (ok && use > 0) ok = mbar_wait(p_empty + pb, (use - 1) & 1);
#pragma unroll
        for (int r = 0; r < NR; r += 16) {
          constexpr int kWords = NR < 16 ? NR / 4 : 4;
          uint32_t hi[4], lo[4];
#pragma unroll
          for (int w = 0; w < kWords; ++w)
            if (r + 4 * w < NR) weight_terms(y[r + 4 * w], y[r + 4 * w + 1], y[r + 4 * w + 2], y[r + 4 * w + 3], hi[w], lo[w]);
          const uint32_t at = p_at[r / 16] + pb * 2 * C::kPTerm;
          store_words(at, hi, min(4, (NR - r) / 4));
          store_words(at + C::kPTerm, lo, min(4, (NR - r) / 4));
        }
        // value codes without a key (behind the length, or of a page that is none) are cleared: a weight of
        // zero would not take a NaN there out
        if (n0 < kTile || n1 < kTile) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int n = h ? n1 : n0;
            uint8_t* v = smem + st * C::kStage + 2 * C::kHalf + h * C::kHalf;
            for (int d = tid; d < HD; d += 128)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int keep = n - c * 16;
                if (keep >= 16) continue;
                uint4* at = reinterpret_cast<uint4*>(v + d * 64 + ((c ^ ((d >> 1) & 3)) << 4));
                uint4 x = keep > 0 ? *at : make_uint4(0, 0, 0, 0);
                uint32_t* w = reinterpret_cast<uint32_t*>(&x);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                  const int b = keep - 4 * j;
                  w[j] &= b >= 4 ? 0xffffffffu : b <= 0 ? 0u : (1u << (8 * b)) - 1u;
                }
                *at = x;
              }
          }
        }
        tc::fence_async_smem();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full + pb);
      }

      // ---- the unit's result: l over all keys, then thread = column
      if (sg.steps > 0) {
        softmax_sync();  // every warp is done with `red`
        // halves of the rows change hands until a lane holds one row's (two rows') sum over the warp
        constexpr int NP = NR <= 4 ? 4 : NR <= 8 ? 8 : NR <= 16 ? 16 : NR <= 32 ? 32 : 64;
        float x[NP];
#pragma unroll
        for (int r = 0; r < NP; ++r) x[r] = r < NR ? l[r] : 0.f;
        int n = NP;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
          if (n > 1) {
            n /= 2;
#pragma unroll
            for (int r = 0; r < NP / 2; ++r)
              if (r < n) {
                const float give = (lane & off) ? x[r] : x[r + n];
                const float keep = (lane & off) ? x[r + n] : x[r];
                x[r] = keep + __shfl_xor_sync(0xffffffffu, give, off);
              }
          } else {
            x[0] += __shfl_xor_sync(0xffffffffu, x[0], off);
          }
        }
        if constexpr (NP == 64) {
          if (2 * lane < NR) {
            red[warp * NR + 2 * lane] = x[0];
            red[warp * NR + 2 * lane + 1] = x[1];
          }
        } else {
          constexpr int per = 32 / NP;  // lanes that hold the same row
          if (lane % per == 0 && lane / per < NR) red[warp * NR + lane / per] = x[0];
        }
      }
      softmax_sync();
      if (tid < NR) {
        // o and l are relative to row_m, o in units of 2^rv; the block's to mb
        const bool ctx = sg.steps > 0;
        const float lc = ctx ? red[tid] + red[NR + tid] + red[2 * NR + tid] + red[3 * NR + tid] : 0.f;
        const float m = lc == 0.f ? -INFINITY : -row_m[tid], mb = blk ? row_mb[tid] : -INFINITY;
        const float M = fmaxf(m, mb), ref = M == -INFINITY ? 0.f : M;
        const float fa = ex2(m - ref), fb = blk ? ex2(mb - ref) : 0.f;
        const float den = lc * fa + (blk ? row_lb[tid] * fb : 0.f);
        if (sg.whole) {
          const float inv = den == 0.f ? 0.f : 1.f / den;
          row_a[tid] = fa * inv * (rv <= -200 ? 0.f : kv8_exp2i(min(max(rv, -126), 126)));
          row_mb[tid] = fb * inv;
        } else {  // parts are in units of 2^E, E >= rv, and E >= 0 with the block's own rows in them
          const float E = blk ? fmaxf(float(rv), 0.f) : float(rv);
          row_a[tid] = fa * ex2(fmaxf(float(rv) - E, -126.f));
          row_mb[tid] = fb * ex2(-E);
          if (tid < sg.n_rows) {
            const int part = 2 * blockIdx.x + (a0 == 0 && sg.un.t > 0 ? 0 : 1);
            pl.sp.ml[int64_t(part) * NR + tid] = make_float4(M, den, E, 0.f);
          }
        }
      }
      softmax_sync();
      if (blk) {  // the block's weights with their row's factor
        for (int x = tid; x < p.block * NR; x += 128) W[x] *= row_mb[x % NR];
        softmax_sync();
      }
      if (sg.steps > 0) {
        if (ok) ok = mbar_wait(o_full, outs & 1);
        ++outs;
        tc::tc_fence_after();
      }
#pragma unroll 1
      for (int nh = 0; nh < C::NH; ++nh) {
        const int d = nh * 128 + tid;
        float o[NR];
        if (sg.steps > 0) {
          tmem_ld<NR>(t_o + t_lane + nh * NM, o);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int r = 0; r < NR; ++r) o[r] = 0.f;
        }
        if (d >= HD) continue;  // head_dim 64: the other lanes multiplied whatever followed
#pragma unroll
        for (int r = 0; r < NR; ++r) o[r] *= row_a[r];
        if (blk) {
          const B16* bv = static_cast<const B16*>(p.blk_v) + sg.un.b * p.bv_batch + sg.g * p.bv_head + d;
#pragma unroll 4
          for (int j = 0; j < p.block; ++j) {
            const float v = ld_f(bv, j * p.bv_row);
#pragma unroll
            for (int r = 0; r < NR; ++r) o[r] = fmaf(W[j * NR + r], v, o[r]);
          }
        }
        if (sg.whole) {
          B16* out = static_cast<B16*>(p.out) + int64_t(sg.un.b) * p.block * p.n_heads * HD + d;
#pragma unroll
          for (int r = 0; r < NR; ++r)
            if (r < sg.n_rows) {
              const int rr = sg.r0 + r;
              out[(int64_t(rr % p.block) * p.n_heads + sg.g * group + rr / p.block) * HD] = __float2bfloat16_rn(o[r]);
            }
        } else {
          const int part = 2 * blockIdx.x + (a0 == 0 && sg.un.t > 0 ? 0 : 1);
          float* out = pl.sp.part + int64_t(part) * NR * HD + d;
#pragma unroll
          for (int r = 0; r < NR; ++r)
            if (r < sg.n_rows) out[int64_t(r) * HD] = o[r];
        }
      }
      tc::tc_fence_before();
      a0 += sg.t1 - sg.t0;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == 5) tc::tmem_dealloc(tmem, C::kAlloc);
}

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(p);
  });
  return fn;
}

// codes [rows, width] as boxes of [box_rows, box_width] bytes
int byte_map(CUtensorMap* map, const void* base, int64_t rows, int width, int box_width, int box_rows, bool sw64) {
  auto enc = encode_fn();
  if (!enc) return fail(DSM_ERR_CUDA, "dsm_gqa_attn_kv8: cuTensorMapEncodeTiled unavailable");
  const cuuint64_t dims[2] = {cuuint64_t(width), cuuint64_t(rows)}, strides[1] = {cuuint64_t(width)};
  const cuuint32_t box[2] = {cuuint32_t(box_width), cuuint32_t(box_rows)}, one[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, one,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, sw64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(DSM_ERR_CUDA, "dsm_gqa_attn_kv8: cuTensorMapEncodeTiled failed (" + std::to_string(int(r)) + ")");
  return DSM_OK;
}

// query rows per CTA: multiples of 8, since the softmax costs by the row, and 4 for single tokens
int rows_of(int rows) { return rows <= 4 ? 4 : std::min(64, (rows + 7) / 8 * 8); }
int ctas_per_sm(int hd) { return hd == 256 ? 1 : 2; }

template <int HD, int NR>
int launch(const AttnArgs& a, UmmaPlan pl, cudaStream_t s) {
  using C = Cfg<HD, NR>;
  // 227 KB per SM, 1 KB of it taken by each CTA
  const int room = 228 * 1024 / C::CTAS - 1024, block = a.blk_k ? a.block : 0;
  // two stages at least: a step's scores are issued before the previous step's sums. A large batch's prefix
  // and a large block may leave room for one CTA per SM only
  pl.stages = 4;
  while (pl.stages > 2 && umma_smem(HD, NR, pl.stages, block, a.batch).bytes > room) --pl.stages;
  const int smem = umma_smem(HD, NR, pl.stages, block, a.batch).bytes;
  if (smem > 227 * 1024) return DSM_ERR_UNSUPPORTED;
  CUtensorMap kmap{}, vmap{};
  const int64_t groups = int64_t(a.n_pages) * a.n_kv * (a.page / kTile);
  int st = byte_map(&vmap, a.v_codes, groups * HD, kTile, kTile, HD, true);
  if (st == DSM_OK && HD == 64) st = byte_map(&kmap, a.k_codes, groups * kTile, 64, 64, kTile, true);
  if (st == DSM_OK && HD == 256) st = byte_map(&kmap, a.k_codes, groups * kTile, 256, 128, kTile, false);
  if (st != DSM_OK) return st;
  auto kern = kv8_umma_kernel<HD, NR>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
    return check_launch("gqa_attn_kv8 smem attribute");
  kern<<<unsigned(pl.sp.ctas), kThreads, size_t(smem), s>>>(a, pl, kmap, vmap);
  st = check_launch("gqa_attn_kv8");
  return st != DSM_OK ? st : kv8_combine(a, pl.sp, HD, DSM_DT_BF16, s);
}

template <int HD>
int launch_rows(int nr, const AttnArgs& a, const UmmaPlan& pl, cudaStream_t s) {
  switch (nr) {
    case 4: return launch<HD, 4>(a, pl, s);
    case 8: return launch<HD, 8>(a, pl, s);
    case 16: return launch<HD, 16>(a, pl, s);
    case 24: return launch<HD, 24>(a, pl, s);
    case 32: return launch<HD, 32>(a, pl, s);
    case 40: return launch<HD, 40>(a, pl, s);
    case 48: return launch<HD, 48>(a, pl, s);
    case 56: return launch<HD, 56>(a, pl, s);
    default: return launch<HD, 64>(a, pl, s);
  }
}

}  // namespace

size_t kv8_umma_ws_bytes(int rows, int hd) {
  return split_ws_bytes(ctas_per_sm(hd) * num_sms(), rows_of(rows), hd);
}

int kv8_umma(const AttnArgs& a, int hd, void* ws, cudaStream_t s) {
  UmmaPlan pl;
  pl.sp.rows = a.n_heads / a.n_kv * a.block;
  const int nr = rows_of(pl.sp.rows);
  pl.sp.row_blocks = int(ceil_div(pl.sp.rows, nr));
  pl.sp.cta_rows = nr;
  const int64_t groups = int64_t(a.n_pages) * a.n_kv * (a.page / kTile);
  const int64_t most = int64_t(a.batch) * a.max_pages * (a.page / kTile) * a.n_kv * pl.sp.row_blocks;
  // tile numbers, and rows of the TMA maps, stay in 32 bits
  if (most > 0x7fffffff || groups * std::max(hd, kTile) > 0x7fffffff) return DSM_ERR_UNSUPPORTED;
  const int most_ctas = ctas_per_sm(hd) * num_sms();
  pl.sp.ctas = int(std::min<int64_t>(most_ctas, most));
  pl.sp.cost = 6;
  pl.sp.snap = 4;
  pl.sp.least = 12;
  split_ws(pl.sp, ws, hd);
  pl.vec_q = vec_ok(a.q, a.q_batch, a.q_row, a.q_head, 8);
  pl.vec_blk = a.blk_k && vec_ok(a.blk_k, a.bk_batch, a.bk_head, a.bk_row, 8);
  switch (hd) {
    case 64: return launch_rows<64>(nr, a, pl, s);
    case 128: return launch_rows<128>(nr, a, pl, s);
    default: return launch_rows<256>(nr, a, pl, s);
  }
}

}  // namespace dsm
