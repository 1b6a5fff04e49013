// The attention over the paged 8-bit cache for bf16 rows, on tcgen05 (dsm_gqa_attn_kv8, layout in
// kv8.cuh).
//
// Mathematics. Everything is taken transposed, so that the keys and the values are the 128-row operands
// as they are stored and the query rows (4 to 64 per KV head) are the narrow one:
//   s [128 keys, rows] = k [128 keys, head_dim] q^T     o [head_dim, rows] += v^T [head_dim, 128 keys] p^T
// kind::f8f6f4 multiplies the e4m3 codes themselves. q, scaled per row by a power of two to at most
// 448, is the sum of two e4m3 terms (hi = e4m3(x), lo = e4m3(x - hi): exact for bf16's 8 bits wherever
// the residual reaches e4m3's normals, 2^-10 of a unit off elsewhere, of a row maximum of 224 to 448).
// The weights are p = 2^(s - m + 15), rounded to f16 (2^-11 of a weight) and held by three e5m2 terms down to half of
// e5m2's smallest step, 2^-17. m is the row's reference: its maximum when it was last set, plus three, so that the
// largest weight is 2^12 or more, and 2^-29 of it is the most that is lost of any beside its 2^-11. (An e4m3 and
// an e5m2 term, relative to 2^8, left 2^-7 of a weight down to 2^-12 of the largest, an eighth at 2^-16 and nothing
// below 2^-22: a tail behind a heavy key that gives nothing was off by 1 to 7 percent.) m is set again, for every
// row that has risen, when a weight would pass 2^15.75, and the sums in tensor memory are then rescaled (2,200 to
// 3,000 cycles, waiting for the products that make them: with a reference just above the maximum, or moved for
// one row alone, most of a unit's first steps paid that). The page's value exponent is folded into the weights
// relative to a reference rv that moves when an exponent leaves [rv - 10, rv]: the 2^-29 are of the largest weight
// times the largest value that 2^rv stands for, and a page whose values are 2^29 times smaller than its
// neighbour's gives nothing. The scores' page factor is one per thread. Scores, sums and weights'
// sums are fp32. The block's own rows are a unit's first step, in two e4m3 terms per row like q.
//
// What bounds it: reading 2 * head_dim bytes per key and KV head. At the copy peak an SM gets 128 keys of
// head_dim 128 per ~1400 cycles. Of shared memory that takes 256 cycles for the copies and 32 for each product's
// 4 KB of codes, so a weight's terms are columns of one product (N = 3 x rows, a sum each, added at the end): as
// products of their own, 20 a step instead of 12, they cost 210 us instead of 176 for 128 sequences of 4096 keys.
// The softmax is ~420 instructions of each of four warps. mma.sync runs e4m3
// operands as f16 products with the conversions around every one, and f16 fragments converted once per warp
// need 1,700 unrolled instructions per 64 keys and 32 rows, which the instruction cache does not hold
// (measured: 116 us for 131,071 keys x 8 heads x 20 rows, against 41 us for the bytes).
//
// Layout. Two CTAs per SM (one at head_dim 256 or 64 rows), each over its range of the line of units
// (kv8_attn.cuh), 128 keys a step:
//   softmax groups  of four warps, 16 query rows each and independent of one another: thread = key for the
//                   weights, thread = column for the result. Four warps with 32 rows took 3,300 cycles a step at
//                   two CTAs per SM, most of it waiting for their own results
//   producer warp   pages from the block table, 64 keys each; bulk copies (keys of head_dim 128, stored
//                   in the operand's 128-byte swizzle) and TMA boxes (the rest, swizzled on the way)
//   product warp    one thread issues the products: scores of step i + 1 before the sums of step i
// Code that runs once per unit is kept short: a CTA meets it with a cold instruction cache.
//
// Measured (32 query heads on 8 KV heads of 128): 128 sequences of 4096 keys, one row each, 177 us (6.1 TB/s);
// one of 131,071 keys, 5 rows, 70 us (3.8 TB/s); 16 of 2048 keys, 7 rows, 38 us. Where rows are few the copies
// bound it. At 20 to 32 rows a step's instructions and its waits for scores and slots do, and what a unit costs
// beside its steps (ten tiles' time, kv8_umma below).
#include <algorithm>
#include <mutex>

#include "kv8_attn.cuh"
#include "tcgen05.cuh"

namespace dsm {
namespace {

using B16 = __nv_bfloat16;

constexpr int kStepKeys = 128;
constexpr int kGroupRows = 16;  // query rows of a softmax group
constexpr float kPExp = 15.f;    // weights at the reference: 2^15
constexpr float kPMax = 15.75f;  // 2^15.75 = 55,109 still fits e5m2 and f16
constexpr float kPHead = 3.f;    // a new reference lies this much above the maximum: the maximum's own weight is 2^12
constexpr int kPTerms = 3;       // e5m2 terms of a weight

// steps whose weights are held: one where a second would cost a copy's slot (one sequence of 131,071 keys 70.0 us with one, 71.1 with two)
__host__ __device__ constexpr int p_buffers(int hd, int nm) { return hd == 128 && nm <= 32 ? 1 : 2; }

template <int HD, int NR>  // NR query rows per CTA: 4, 8, 16, 32 or 64
struct Cfg {
  static constexpr int NM = NR < 16 ? 16 : NR;  // columns of the products
  static constexpr int G = NM / kGroupRows;     // softmax groups
  static constexpr int RW = NR < 16 ? NR : 16;  // rows that a group computes
  static constexpr int NH = HD <= 128 ? 1 : 2;  // 128-row halves of the output
  static constexpr int CTAS = HD == 256 || NM == 64 ? 1 : 2;  // per SM
  static constexpr int kSoftmax = 128 * G;                    // threads
  static constexpr int kThreads = kSoftmax + 64;
  static constexpr int kHalf = kTile * HD;       // bytes of 64 keys, or of their values
  static constexpr int kSlot = 2 * kHalf;        // a step's keys, or its values
  static constexpr int kQTerm = NM * HD;         // bytes of one term of q
  static constexpr int kPTerm = NM * kStepKeys;  // bytes of one term of the weights
  static constexpr int PB = p_buffers(HD, NM);   // steps' weights in shared memory
  static constexpr int ON = kPTerms * NM;        // columns of the sums: each term of the weights has its own
  static constexpr int kCols = 2 * NM + NH * ON; // tensor memory: two score buffers, the sums
  static constexpr int kAlloc = kCols <= 128 ? 128 : kCols <= 256 ? 256 : 512;
  static_assert(kCols <= 512 && CTAS * kAlloc <= 512);
};

struct UmmaPlan {
  KvSplit sp;
  int k_slots, v_slots;  // steps' keys and values in shared memory: keys are done with earlier
  bool vec_q, vec_blk;   // q's rows / both the block's keys and values can be read 4 values at a time
};

struct UmmaSmem {
  int q, p, rows, keys, info, bars, sums, P, bytes;
};
// per row: c (score factor), m (less its reference), a (rescaling), where its result goes, and four warps' partial
// results
constexpr int kRowFloats = 8;
constexpr int kInfos = 8;  // steps whose scales are noted down: more than there are slots
constexpr int kMaxSlots = 6;
__host__ __device__ inline UmmaSmem umma_smem(int hd, int nm, int slots, int batch) {
  UmmaSmem s;
  s.q = slots * 2 * kTile * hd;
  s.p = s.q + 2 * nm * hd;
  s.rows = s.p + p_buffers(hd, nm) * kPTerms * nm * kStepKeys;
  s.keys = s.rows + kRowFloats * nm * 4;  // the block's rows: key scale and value exponent
  s.info = s.keys + kUmmaMaxBlock * 8;
  s.bars = s.info + kInfos * 16;
  s.sums = s.bars + (4 * kMaxSlots + 2 * kInfos + 10) * 8;
  s.P = s.sums + 128;
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
// the weights, rows of 16, 32 or 64 bytes per key and term (the operand's N dimension contiguous), the terms one
// after another: 16-byte rows unswizzled with groups of 8 keys at 128 B (the leading offset) and terms at the
// stride, 32- and 64-byte rows in the swizzle of their width with groups of 8 keys at 256 and 512 B (the
// stride) and terms at the leading offset
template <int NM>
__device__ __forceinline__ uint64_t desc_weights(uint32_t saddr) {
  constexpr uint64_t keys8 = 8 * NM >> 4, term = NM * kStepKeys >> 4;
  constexpr uint64_t lead = NM == 16 ? keys8 : term, stride = NM == 16 ? term : keys8;
  constexpr uint64_t swizzle = NM == 16 ? 0 : NM == 32 ? 6 : 4;
  return uint64_t((saddr >> 4) & 0x3FFFu) | (lead << 16) | (stride << 32) | (uint64_t(1) << 46) | (swizzle << 61);
}
// kind::f8f6f4: D f32, A e4m3 K-major, B e4m3 K-major (q), or e5m2 N-major (the weights)
__device__ __forceinline__ uint32_t idesc_f8(int n, bool weights) {
  return (1u << 4) | (weights ? 1u << 10 | 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24);
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
// Wait for a phase, for a bounded number of tries (each suspends for a while in the hardware). Short on
// purpose, and no call: it stands in loops that keep their registers.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity) {
  uint32_t tries = 0;
  while (!mbar_try_wait(bar, parity))
    if (++tries == 1u << 24) {
      raise_device_error(DSM_DEV_ERR_PIPELINE_TIMEOUT);
      return false;
    }
  return true;
}
__device__ __forceinline__ bool done(uint64_t* bar, uint32_t parity) {  // without waiting
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}
template <int N>
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[N]) {
  if constexpr (N == 16)
    tc::tmem_st16(addr, r);
  else if constexpr (N == 8)
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
  else
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]),
                 "r"(r[3])
                 : "memory");
}
// barriers of one softmax group (id 1 + group), and of all of them (id 8)
__device__ __forceinline__ bool any_of_group(int group, bool x) {
  uint32_t r;
  asm volatile(
      "{\n .reg .pred p, q;\n setp.ne.u32 p, %2, 0;\n barrier.cta.red.or.pred q, %1, 128, p;\n selp.u32 %0, 1, 0, q;\n}"
      : "=r"(r)
      : "r"(group + 1), "r"(x ? 1u : 0u)
      : "memory");
  return r != 0;
}
__device__ __forceinline__ void group_sync(int group) { asm volatile("barrier.cta.sync %0, 128;" ::"r"(group + 1) : "memory"); }
template <int N>
__device__ __forceinline__ void softmax_sync() {
  asm volatile("barrier.cta.sync 8, %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float redux_max(float x) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
  return r;
}
// Weights of up to 2^15.75 enter in three e5m2 terms. They pass through f16, whose 11 bits the terms hold: a residual
// of 8 bits after the first (3 bits) is at most 8 units after the second, and fits the third.
__device__ __forceinline__ uint32_t to_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// the next term of four weights, a byte each, taken off them. An e5m2 value is the upper byte of its f16.
__device__ __forceinline__ uint32_t weight_term(uint32_t& x, uint32_t& y) {
  uint32_t t;
  asm("{\n .reg .b32 g, h;\n .reg .b16 a, b;\n"
      " cvt.rn.satfinite.e5m2x2.f16x2 a, %1;\n"
      " cvt.rn.satfinite.e5m2x2.f16x2 b, %2;\n"
      " mov.b32 %0, {a, b};\n"
      " prmt.b32 g, %0, 0, 0x1404;\n"
      " prmt.b32 h, %0, 0, 0x3424;\n"
      " sub.rn.f16x2 %1, %1, g;\n"
      " sub.rn.f16x2 %2, %2, h;\n}"
      : "=&r"(t), "+r"(x), "+r"(y));
  return t;
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
  int b, t0, t1, steps, g, r0, n_rows, len;
  bool whole, blk;  // all of the unit; the block's own rows come first, as a step more
};

template <int HD, int NR>
__global__ void __launch_bounds__(Cfg<HD, NR>::kThreads, Cfg<HD, NR>::CTAS)
    kv8_umma_kernel(const AttnArgs p, const UmmaPlan pl, const __grid_constant__ CUtensorMap kmap,
                    const __grid_constant__ CUtensorMap vmap) {
  using C = Cfg<HD, NR>;
  constexpr int NM = C::NM, RW = C::RW, kProducer = 4 * C::G, kProduct = kProducer + 1;
  extern __shared__ uint8_t raw[];
  uint8_t* smem = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
  const int KN = pl.k_slots, VN = pl.v_slots;
  const UmmaSmem L = umma_smem(HD, NM, KN + VN, p.batch);
  uint8_t* const v_slots = smem + KN * C::kSlot;
  float* row_c = reinterpret_cast<float*>(smem + L.rows);
  float* row_m = row_c + NM;
  float* row_a = row_m + NM;
  int* row_out = reinterpret_cast<int*>(row_a + NM);
  float* const reds = row_a + 2 * NM;  // [group][4 warps][16]
  float2* keys = reinterpret_cast<float2*>(smem + L.keys);
  float4* info = reinterpret_cast<float4*>(smem + L.info);  // per step: key and value scale of each half
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L.bars);
  uint64_t* k_empty = k_full + kMaxSlots;
  uint64_t* v_full = k_empty + kMaxSlots;
  uint64_t* v_empty = v_full + kMaxSlots;
  uint64_t* i_full = v_empty + kMaxSlots;  // [kInfos]
  uint64_t* granted = i_full + kInfos;     // [kInfos]: a step's slots wait for the block's own rows
  uint64_t* s_full = granted + kInfos;     // [2]
  uint64_t* s_empty = s_full + 2;          // [2]
  uint64_t* p_full = s_empty + 2;          // [2]
  uint64_t* p_empty = p_full + 2;          // [2]
  uint64_t* q_full = p_empty + 2;
  uint64_t* o_full = q_full + 1;
  uint32_t* slot = reinterpret_cast<uint32_t*>(smem + L.sums + 112);
  int* P = reinterpret_cast<int*>(smem + L.P);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int hr = p.n_kv * pl.sp.row_blocks;
  constexpr int kBars = 4 * kMaxSlots + 2 * kInfos + 10;
  if (tid < kBars) {  // one arrival each, but what the softmax warps arrive on
    const int i = tid - (4 * kMaxSlots + 2 * kInfos);
    const bool by_softmax = i == 2 || i == 3 || i == 4 || i == 5 || i == 8;  // s_empty, p_full, q_full
    mbar_init(k_full + tid, by_softmax ? 4 * C::G : 1);
    fence_mbar_init();
  }
  if (warp == kProduct) tc::tmem_alloc(slot, C::kAlloc);
  scan_tiles<C::kThreads>(p, P, reinterpret_cast<int*>(smem + L.sums));
  asm volatile("griddepcontrol.launch_dependents;");  // the join may take its place and wait
  int start;
  Place un;  // the unit that this warp is at
  const int n_tiles = my_range(p, P, pl.sp, reinterpret_cast<int*>(smem + L.sums) + 20, start, un);
  if (blockIdx.x == 0)
    for (int b = tid; b < p.batch; b += C::kThreads)
      if (p.lengths[b] > int64_t(p.max_pages) * p.page) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = *slot, t_o = tmem + 2 * NM;

  auto segment = [&](int a0) {
    Segment s;
    s.b = un.b;
    s.t0 = un.t;
    s.t1 = min(un.T, un.t + n_tiles - a0);
    s.blk = s.t1 == un.T && p.blk_k;
    s.whole = s.t1 == un.T && s.t0 == 0;
    s.g = un.u;
    s.r0 = 0;
    if (pl.sp.row_blocks > 1) {
      s.g = un.u / pl.sp.row_blocks;
      s.r0 = (un.u - s.g * pl.sp.row_blocks) * NR;
    }
    s.n_rows = min(NR, pl.sp.rows - s.r0);
    s.len = seq_len(p, un.b);
    s.steps = (s.len == 0 ? 0 : (s.t1 - s.t0 + 1) / 2) + s.blk;
    next_unit(P, p.batch, hr, un);
    return s;
  };
  bool ok = true;  // no wait has run out; after one has, loops go through without waiting, copying or multiplying

  if (warp == kProducer) {
    // ---------------------------------------------------------------- producer
    const int per_page = p.page / kTile;
    int k = 0;  // steps so far
    for (int a0 = 0; a0 < n_tiles;) {
      const Segment sg = segment(a0);
      a0 += sg.t1 - sg.t0;
      const int tiles = sg.len == 0 ? 0 : sg.t1 - sg.t0;
      if (sg.blk) {  // the softmax warps fill this step's slots
        if (ok && k >= KN) ok = wait(k_empty + k % KN, (k / KN - 1) & 1);
        if (ok && k >= VN) ok = wait(v_empty + k % VN, (k / VN - 1) & 1);
        if (lane == 0 && ok) {
          mbar_arrive(granted + k % kInfos);
          mbar_arrive(i_full + k % kInfos);
        }
        ++k;
      }
      for (int base = 0; base < tiles; base += 32) {
        // a lane per tile: its page, then its scales (used when the first copies are on their way)
        const int t = sg.t0 + base + lane;
        int pg = -1;
        if (base + lane < tiles) {
          pg = __ldg(p.table + int64_t(sg.b) * p.table_stride + t * kTile / p.page);
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
          const int kn = k % KN, vn = k % VN;
          const int pg0 = __shfl_sync(0xffffffffu, pg, i), pg1 = __shfl_sync(0xffffffffu, pg, i + 1);
          const int live = (pg0 >= 0) + (pg1 >= 0);
          const int64_t ph0 = int64_t(max(pg0, 0)) * p.n_kv + sg.g, ph1 = int64_t(max(pg1, 0)) * p.n_kv + sg.g;
          const int sub = (sg.t0 + base + i) % per_page, sub1 = sub + 1 == per_page ? 0 : sub + 1;
          const int64_t group0 = ph0 * per_page + sub, group1 = ph1 * per_page + sub1;  // of 64 tokens
          if (ok && k >= KN) ok = wait(k_empty + kn, (k / KN - 1) & 1);
          if (lane == 0 && ok) {
            mbar_arrive_expect_tx(k_full + kn, live * C::kHalf);
            uint8_t* const dst = smem + kn * C::kSlot;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              if ((h ? pg1 : pg0) < 0) continue;
              const int64_t g64 = h ? group1 : group0;
              if constexpr (HD == 128) {
                bulk_g2s(dst + h * C::kHalf, p.k_codes + g64 * C::kHalf, C::kHalf, k_full + kn, policy_evict_first());
              } else if constexpr (HD == 64) {
                tma_2d(smem_u32(dst) + h * C::kHalf, &kmap, 0, int(g64 * kTile), k_full + kn);
              } else {  // two slabs of 128 bytes
                tma_2d(smem_u32(dst) + h * (C::kHalf / 2), &kmap, 0, int(g64 * kTile), k_full + kn);
                tma_2d(smem_u32(dst) + C::kHalf + h * (C::kHalf / 2), &kmap, 128, int(g64 * kTile), k_full + kn);
              }
            }
          }
          if (ok && k >= VN) ok = wait(v_empty + vn, (k / VN - 1) & 1);
          if (lane == 0 && ok) {
            mbar_arrive_expect_tx(v_full + vn, live * C::kHalf);
            const uint32_t dst = smem_u32(v_slots + vn * C::kSlot);
            if (pg0 >= 0) tma_2d(dst, &vmap, 0, int(group0 * HD), v_full + vn);
            if (pg1 >= 0) tma_2d(dst + C::kHalf, &vmap, 0, int(group1 * HD), v_full + vn);
          }
          const float4 sc = make_float4(__shfl_sync(0xffffffffu, ks, i), __shfl_sync(0xffffffffu, vs, i),
                                        __shfl_sync(0xffffffffu, ks, i + 1), __shfl_sync(0xffffffffu, vs, i + 1));
          if (lane == 0 && ok) {
            info[k % kInfos] = sc;
            mbar_arrive(i_full + k % kInfos);
          }
          __syncwarp();
        }
      }
    }
    // after a wait that ran out, copies may still be on their way: see them land
    if (!ok) {
      for (int i = max(0, k - KN); i < k; ++i) wait(k_full + i % KN, (i / KN) & 1);
      for (int i = max(0, k - VN); i < k; ++i) wait(v_full + i % VN, (i / VN) & 1);
    }
  } else if (warp == kProduct) {
    // ---------------------------------------------------------------- products
    if (lane == 0) {
      const uint32_t id_s = idesc_f8(NM, false), id_o = idesc_f8(C::ON, true);
      const uint32_t base = smem_u32(smem), qa = base + L.q, pa = base + L.p;
      int k = 0, seg = 0;  // steps, and units with steps, so far
      for (int a0 = 0; a0 < n_tiles;) {
        const Segment sg = segment(a0);
        a0 += sg.t1 - sg.t0;
        if (sg.steps == 0) continue;
        if (ok) ok = wait(q_full, seg++ & 1);
        tc::tc_fence_after();
        auto sums = [&](int j, bool first, bool blk) {  // step j's
          const int pb = j % C::PB;
          if (ok) ok = wait(v_full + j % VN, (j / VN) & 1);
          tc::tc_fence_after();
          if (!ok) return;
          const uint32_t v = base + KN * C::kSlot + (j % VN) * C::kSlot, w = pa + pb * kPTerms * C::kPTerm;
          // 32 keys a product
          const uint64_t av = desc_sw64(v), bw = desc_weights<NM>(w);
          if (!blk) {
#pragma unroll
            for (int nh = 0; nh < C::NH; ++nh)
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
                umma_f8(t_o + nh * C::ON, av + (((ks >> 1) * C::kHalf + nh * 128 * 64 + (ks & 1) * 32) >> 4),
                        bw + (ks * 32 * NM >> 4), id_o, !first || ks > 0);
          } else {  // its values' two terms lie where others have keys 0-63 and 64-127
            const int n = (p.block + 31) / 32;
#pragma unroll 1
            for (int i = 0; i < 2 * C::NH * n; ++i) {
              const int ks = i % n, term = i / n & 1, nh = i / n >> 1;
              umma_f8(t_o + nh * C::ON, av + ((term * C::kHalf + nh * 128 * 64 + ks * 32) >> 4),
                      bw + (ks * 32 * NM >> 4), id_o, !first || i % (2 * n) > 0);
            }
          }
          tc::umma_commit(v_empty + j % VN);
          tc::umma_commit(p_empty + pb);
        };
        // step i's scores, step j's sums: whichever can go
        uint32_t idle = 0;
        for (int i = 0, j = 0; j < sg.steps && ok;) {
          const int kk = k + i, sb = kk & 1, jj = k + j;
          if (i < sg.steps && i < j + 2 && done(k_full + kk % KN, (kk / KN) & 1) &&
              (kk < 2 || done(s_empty + sb, ((kk >> 1) - 1) & 1))) {
            tc::tc_fence_after();
            // the block's step: its keys' hi terms are rows 0-63, their lo terms rows 64-127, multiplied as
            // rows 0-63 once more
            const uint32_t kt = base + (kk % KN) * C::kSlot;
            const uint64_t ak = HD == 64 ? desc_sw64(kt) : tc::umma_desc_sw128(kt);
            const uint64_t bq = HD == 64 ? desc_sw64(qa) : tc::umma_desc_sw128(qa);
#pragma unroll 1
            for (int lo = 0; lo <= (sg.blk && i == 0); ++lo)
#pragma unroll
              for (int x = 0; x < 2; ++x)
#pragma unroll
                for (int ks = 0; ks < HD / 32; ++ks)
                  umma_f8(tmem + sb * NM,
                          ak + (((ks >> 2) * 2 * 64 * 128 + (ks & 3) * 32) >> 4) + lo * ((HD == 64 ? 64 * 64 : 64 * 128) >> 4),
                          bq + ((x * C::kQTerm + (ks >> 2) * NM * 128 + (ks & 3) * 32) >> 4), id_s,
                          lo > 0 || x > 0 || ks > 0);
            tc::umma_commit(s_full + sb);
            tc::umma_commit(k_empty + kk % KN);
            ++i;
            idle = 0;
          } else if (j < i && done(p_full + jj % C::PB, (jj / C::PB) & 1)) {
            sums(jj, j == 0, sg.blk && j == 0);
            ++j;
            idle = 0;
          } else if (++idle == 1u << 24) {
            raise_device_error(DSM_DEV_ERR_PIPELINE_TIMEOUT);
            ok = false;
          }
        }
        if (ok) tc::umma_commit(o_full);
        k += sg.steps;
      }
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax, results
    constexpr int TPR = 8, VB = HD / TPR, kPass = C::kSoftmax / TPR;  // staging: threads per row, values per thread
    const int grp = C::G == 1 ? 0 : warp >> 2, gtid = C::G == 1 ? tid : tid & 127;
    const int g0 = grp * kGroupRows;  // its first row
    const int half = gtid >> 6;       // which 64 keys of a step this thread's key is in
    const int row_r = tid / TPR, row_d = tid % TPR * VB;
    const uint32_t t_lane = uint32_t((warp & 3) * 32) << 16;
    const int group = p.n_heads / p.n_kv;
    // rows of the sums at a time: 8 keep the 96 registers of two CTAs per SM from spilling (one sequence of 131,071 keys
    // 70.0 us, with all 16 74.7), at head_dim 64 their second round costs more (33 sequences of up to 5001, 56 rows:
    // 27.4 us, with 8 rows 29.3)
    constexpr int RP = HD == 64 || RW < 8 ? RW : 8;
    float* const red = reds + grp * 4 * kGroupRows;
    const float* const my_c = row_c + g0;
    const float* const my_m = row_m + g0;
    const float* const my_a = row_a + g0;
    uint8_t* const q8 = smem + L.q;
    // where this thread's key's weights go, 16 rows
    const uint32_t p_at = smem_u32(smem) + L.p + gtid * NM +
                          ((grp ^ (NM == 32 ? (gtid >> 2) & 1 : NM == 64 ? (gtid >> 1) & 3 : 0)) << 4);

    int k = 0, outs = 0;   // steps, and units with steps, so far
    unsigned blocks = 0;  // per step modulo kInfos, whether an odd number of blocks' own rows has been granted
    for (int a0 = 0; a0 < n_tiles;) {
      const Segment sg = segment(a0);
      // ---- q's terms, and the block's own rows: 16 rows at a time, the next ones' loads ahead of this ones' work
      softmax_sync<C::kSoftmax>();  // the previous unit's row statistics are used up
      uint8_t* const kt = smem + (k % KN) * C::kSlot;
      uint8_t* const vt = v_slots + (k % VN) * C::kSlot;
      // the rows in one list: q's (those past n_rows are zero), the block's keys', its values'
      const int n_blk = sg.blk ? p.block : 0, n_list = NR + 2 * n_blk;
      auto load_rows = [&](int r, float(&x)[VB]) {
        const B16* src;
        bool live, vec = pl.vec_blk;
        if (r < NR) {
          const int rr = sg.r0 + r, h = unsigned(rr) / unsigned(p.block);
          src = static_cast<const B16*>(p.q) + sg.b * p.q_batch + (rr - h * p.block) * p.q_row + (sg.g * group + h) * p.q_head;
          live = r < sg.n_rows;
          vec = pl.vec_q;
          if (row_d == 0) row_out[r] = ((rr - h * p.block) * p.n_heads + sg.g * group + h) * HD;
        } else if (r < NR + n_blk) {
          src = static_cast<const B16*>(p.blk_k) + sg.b * p.bk_batch + sg.g * p.bk_head + (r - NR) * p.bk_row;
          live = true;
        } else {
          src = static_cast<const B16*>(p.blk_v) + sg.b * p.bv_batch + sg.g * p.bv_head + (r - NR - n_blk) * p.bv_row;
          live = r < n_list;
        }
#pragma unroll
        for (int i = 0; i < VB; ++i) x[i] = 0.f;
        if (live) load_vals<B16, VB>(src + row_d, vec, x);
      };
      float x[VB];
      load_rows(row_r, x);
      if (sg.blk) {
        if (ok) ok = wait(granted + k % kInfos, blocks >> k % kInfos & 1);
        blocks ^= 1u << k % kInfos;
        // values: columns of 32 (64) keys, zero where there is no key
        const int n = p.block > 32 ? 64 : 32, per = 2 * HD * n / 16;
#pragma unroll 1
        for (int i = tid; i < per; i += C::kSoftmax) {
          const int t = i & 1, d = (i >> 1) % HD, c = (i >> 1) / HD;
          *reinterpret_cast<uint4*>(vt + t * C::kHalf + d * 64 + ((c ^ ((d >> 1) & 3)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        softmax_sync<C::kSoftmax>();
      }
#pragma unroll 1
      for (int at_row = row_r; at_row < (n_list + kPass - 1) / kPass * kPass; at_row += kPass) {
        float next[VB];
        if (at_row + kPass < n_list + row_r) load_rows(at_row + kPass, next);
        const bool of_q = at_row < NR, of_v = at_row >= NR + n_blk;
        const int r = of_q ? at_row : of_v ? at_row - NR - n_blk : at_row - NR;  // among its kind
        const bool live = at_row < n_list;
        // scaled by a power of two to at most 448
        float mx = 0.f;
#pragma unroll
        for (int i = 0; i < VB; ++i) mx = fmaxf(mx, finite_abs(x[i]));
#pragma unroll
        for (int w = TPR / 2; w; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
        const int e = kv8_scale_exp(mx);
        const float inv = kv8_exp2i(-e);
        if (row_d == 0) {
          if (of_q) {
            row_c[r] = r < sg.n_rows ? p.scale * kLog2e * kv8_exp2i(e) : 0.f;
            row_m[r] = 0.f;
          } else if (live) {
            if (of_v)
              keys[r].y = float(e);
            else
              keys[r].x = kv8_exp2i(e);
          }
        }
        // rows of q and of keys: K-major in the swizzle of their width; of values: bytes of its columns
        uint8_t* const at = of_q ? q8 : kt;
        const int rows = of_q ? NM : 128, term = of_q ? C::kQTerm : HD == 64 ? 64 * 64 : 64 * 128;
#pragma unroll
        for (int i = 0; i < VB; i += 4) {
          float y[4];
#pragma unroll
          for (int w = 0; w < 4; ++w) y[w] = scaled(x[i + w], inv);
          uint32_t t[2];
          q_terms(y, t[0], t[1]);
          const int d = row_d + i;
          if (of_v) {
            if (live) {
#pragma unroll
              for (int w = 0; w < 4; ++w) {
                uint8_t* b = vt + (d + w) * 64 + (((r >> 4) ^ (((d + w) >> 1) & 3)) << 4) + (r & 15);
                b[0] = uint8_t(t[0] >> (8 * w));
                b[C::kHalf] = uint8_t(t[1] >> (8 * w));
              }
            }
          } else {
            uint8_t* b = HD == 64 ? at + r * 64 + ((((d >> 4) & 3) ^ ((r >> 1) & 3)) << 4) + (d & 15)
                                  : at + (d >> 7) * rows * 128 + r * 128 + ((((d >> 4) & 7) ^ (r & 7)) << 4) + (d & 15);
            *reinterpret_cast<uint32_t*>(b) = t[0];
            *reinterpret_cast<uint32_t*>(b + term) = t[1];
          }
        }
#pragma unroll
        for (int i = 0; i < VB; ++i) x[i] = next[i];
      }
      tc::fence_async_smem();
      softmax_sync<C::kSoftmax>();
      if (lane == 0 && sg.steps > 0) mbar_arrive(q_full);
      if (sg.blk && tid == 0) {
        mbar_arrive(k_full + k % KN);
        mbar_arrive(v_full + k % VN);
      }

      // ---- the cached rows, 128 a step
      float l[RW];
#pragma unroll
      for (int r = 0; r < RW; ++r) l[r] = 0.f;
      int rv = -200, top_rv = -200;
      for (int i = 0; i < sg.steps; ++i, ++k) {
        const int sb = k & 1;
        if (ok) ok = wait(i_full + k % kInfos, (k / kInfos) & 1);
        const bool own = sg.blk && i == 0;  // the block's own rows: key = thread, a scale each
        int n0 = 0, n1 = 0, e_key = -200, ev = -200, low = 200;
        float ks = 0.f;
        bool live;
        if (own) {
          // a page's exponent is that of many more values than a row's: mostly a step or two above
          for (int j = 0; j < p.block; ++j) ev = max(ev, int(keys[j].y) + 1);
          low = ev;
          live = gtid < p.block;
          if (live) {
            ks = keys[gtid].x;
            e_key = int(keys[gtid].y);
          }
        } else {
          const float4 sc = info[k % kInfos];
          const int t0 = sg.t0 + 2 * (i - sg.blk);  // first tile of the step
          const int left = sg.len - t0 * kTile;
          n0 = sc.x == sc.x ? max(0, min(kTile, left)) : 0;
          n1 = t0 + 1 < sg.t1 && sc.z == sc.z ? max(0, min(kTile, left - kTile)) : 0;
          live = (gtid & 63) < (half ? n1 : n0);
          ks = half ? sc.z : sc.x;
          const int e0 = n0 ? kv8_exponent(sc.y) : -200, e1 = n1 ? kv8_exponent(sc.w) : -200;
          e_key = half ? e1 : e0;
          ev = max(e0, e1);
          low = min(n0 ? e0 : ev, n1 ? e1 : ev);
        }
        top_rv = max(top_rv, ev);
        const int want_rv = ev > rv || low < rv - 10 ? max(ev, top_rv - 40) : rv;
        if (ok) ok = wait(s_full + sb, (k >> 1) & 1);
        tc::tc_fence_after();
        float y[RW];
        tmem_ld<RW>(tmem + t_lane + sb * NM + g0, y);
        tc::tmem_ld_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_empty + sb);
        // the weights' exponents: row_m is kPExp less the reference
        float top = kLowest;
#pragma unroll
        for (int r = 0; r < RW; r += 4) {
          const float4 c = *reinterpret_cast<const float4*>(my_c + r), m = *reinterpret_cast<const float4*>(my_m + r);
          const float2 ks2 = make_float2(ks, ks);
          const float2 a = fma2(make_float2(y[r], y[r + 1]), mul2(make_float2(c.x, c.y), ks2), make_float2(m.x, m.y));
          const float2 b = fma2(make_float2(y[r + 2], y[r + 3]), mul2(make_float2(c.z, c.w), ks2), make_float2(m.z, m.w));
          y[r] = a.x;
          y[r + 1] = a.y;
          y[r + 2] = b.x;
          y[r + 3] = b.y;
          top = fmaxf(top, fmaxf(fmaxf(y[r], y[r + 1]), fmaxf(y[r + 2], y[r + 3])));
        }
        // no step with a key yet (rv is -200 till then): the references are still to be set, the sums are zero
        const bool first = rv <= -200;
        if (any_of_group(grp, (live && top > kPMax) || first || want_rv != rv)) {
          // new references: every row whose maximum has risen since its own was set (all of them at first)
#pragma unroll
          for (int r = 0; r < RW; ++r) {
            const float x = redux_max(live ? y[r] : kLowest);
            if (lane == r) red[(warp & 3) * kGroupRows + r] = x;
          }
          group_sync(grp);
          if (gtid < RW) {
            const float x = fmaxf(fmaxf(red[gtid], red[16 + gtid]), fmaxf(red[32 + gtid], red[48 + gtid]));
            const float up = x == kLowest ? 0.f : first || x > kPExp - kPHead ? x + (kPHead - kPExp) : 0.f;
            row_m[g0 + gtid] -= up;
            red[gtid] = up;
            row_a[g0 + gtid] = first ? 1.f : ex2(-up);  // a first one may lie far below zero: 0 * 2^200 is no 0
          }
          group_sync(grp);
          const float fv = first ? 1.f : kv8_exp2i(min(max(rv - want_rv, -126), 126));
          rv = want_rv;
          if (i > 0) {  // the sums so far, after the products that make them
            const int j = k - 1;
            if (ok) ok = wait(p_empty + j % C::PB, (j / C::PB) & 1);
            tc::tc_fence_after();
#pragma unroll
            for (int r = 0; r < RW; ++r) l[r] *= my_a[r];
#pragma unroll 1
            for (int x = 0; x < C::NH * kPTerms * (RW / RP); ++x) {
              float o[RP];
              uint32_t u[RP];
              const int r0 = x % (RW / RP) * RP;
              const uint32_t at = t_o + t_lane + x / (RW / RP) * NM + g0 + r0;
              tmem_ld<RP>(at, o);
              tc::tmem_ld_wait();
#pragma unroll
              for (int r = 0; r < RP; ++r) u[r] = __float_as_uint(o[r] * (my_a[r0 + r] * fv));
              tmem_st(at, u);
            }
            tc::tmem_st_wait();
          }
#pragma unroll
          for (int r = 0; r < RW; ++r) y[r] -= red[r];
        }
        const int dv = max(e_key - rv, -60);  // <= 0
        const float fv = kv8_exp2i(dv);
#pragma unroll
        for (int r = 0; r < RW; ++r) y[r] = ex2(y[r]);
        if (!__all_sync(0xffffffffu, live)) {
#pragma unroll
          for (int r = 0; r < RW; ++r) y[r] = live ? y[r] : 0.f;
        }
#pragma unroll
        for (int r = 0; r < RW; r += 2) {
          const float2 a = add2(make_float2(l[r], l[r + 1]), make_float2(y[r], y[r + 1]));
          l[r] = a.x;
          l[r + 1] = a.y;
        }
        if (__any_sync(0xffffffffu, dv != 0)) {
#pragma unroll
          for (int r = 0; r < RW; ++r) y[r] *= fv;
        }
        uint32_t w[RW / 2];
#pragma unroll
        for (int r = 0; r < RW; r += 2) w[r / 2] = to_f16x2(y[r], y[r + 1]);
        const int pb = k % C::PB;
        if (ok && k >= C::PB) ok = wait(p_empty + pb, (k / C::PB - 1) & 1);
#pragma unroll
        for (int x = 0; x < kPTerms; ++x) {
          uint32_t t[4];
#pragma unroll
          for (int i = 0; i < RW / 4; ++i) t[i] = weight_term(w[2 * i], w[2 * i + 1]);
          store_words(p_at + (pb * kPTerms + x) * C::kPTerm, t, RW / 4);
        }
        // value codes without a key (behind the length, or of a page that is none) are cleared: a weight of
        // zero would not take a NaN there out
        if (!own && (n0 < kTile || n1 < kTile)) {
          if (ok) ok = wait(v_full + k % VN, (k / VN) & 1);
#pragma unroll 1
          for (int h = 0; h < 2; ++h) {
            const int n = h ? n1 : n0;
            uint8_t* v = v_slots + (k % VN) * C::kSlot + h * C::kHalf;
            for (int d = tid; d < HD; d += C::kSoftmax)
#pragma unroll 1
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
      group_sync(grp);  // every warp is done with `red`
      {
        // halves of the rows change hands until a lane holds one row's sum over the warp
        int n = RW;
#pragma unroll
        for (int off = 16; off >= 1; off >>= 1) {
          if (n > 1) {
            n /= 2;
#pragma unroll
            for (int r = 0; r < RW / 2; ++r)
              if (r < n) {
                const float give = (lane & off) ? l[r] : l[r + n];
                const float keep = (lane & off) ? l[r + n] : l[r];
                l[r] = keep + __shfl_xor_sync(0xffffffffu, give, off);
              }
          } else {
            l[0] += __shfl_xor_sync(0xffffffffu, l[0], off);
          }
        }
        constexpr int per = 32 / RW;  // lanes that hold the same row
        if (lane % per == 0) red[(warp & 3) * kGroupRows + lane / per] = l[0];
      }
      group_sync(grp);
      const int part = 2 * blockIdx.x + (a0 == 0 && sg.t0 > 0 ? 0 : 1);
      if (gtid < RW) {
        // o and l are relative to row_m, o in units of 2^rv (not in row_a: 2^rv / l may fall below fp32's normals)
        const int r = g0 + gtid;
        const float den = red[gtid] + red[16 + gtid] + red[32 + gtid] + red[48 + gtid];
        row_a[r] = den == 0.f ? 0.f : 1.f / den;
        if (!sg.whole && r < sg.n_rows)
          pl.sp.ml[int64_t(part) * NR + r] = make_float4(den == 0.f ? -INFINITY : -row_m[r], den, float(rv), 0.f);
      }
      group_sync(grp);
      if (sg.steps > 0) {
        if (ok) ok = wait(o_full, outs & 1);
        ++outs;
        tc::tc_fence_after();
      }
#pragma unroll 1
      for (int i = 0; i < C::NH * (RW / RP); ++i) {
        const int nh = i / (RW / RP), r0 = g0 + i % (RW / RP) * RP;
        const int d = nh * 128 + gtid;
        float o[RP];
#pragma unroll
        for (int r = 0; r < RP; ++r) o[r] = 0.f;
        if (sg.steps > 0) {
          const uint32_t at = t_o + t_lane + nh * C::ON + r0;  // the terms' sums, small ones first
          constexpr int kAtOnce = RP <= 8 ? kPTerms : 1;
#pragma unroll 1
          for (int x = kPTerms; x > 0; x -= kAtOnce) {
            float t[kAtOnce][RP];
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j) tmem_ld<RP>(at + (x - 1 - j) * NM, t[j]);
            tc::tmem_ld_wait();
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
#pragma unroll
              for (int r = 0; r < RP; ++r) o[r] += t[j][r];
          }
        }
        if (d >= HD) continue;  // head_dim 64: the other lanes multiplied whatever followed
        if (sg.whole) {
          B16* out = static_cast<B16*>(p.out) + int64_t(sg.b) * p.block * p.n_heads * HD + d;
          const float unit = kv8_exp2i(min(max(rv, -126), 126));
#pragma unroll
          for (int r = 0; r < RP; ++r)
            if (r0 + r < sg.n_rows) {
              const float inv = row_a[r0 + r];
              out[row_out[r0 + r]] = __float2bfloat16_rn(inv == 0.f ? 0.f : o[r] * inv * unit);
            }
        } else {
          float* out = pl.sp.part + (int64_t(part) * NR + r0) * HD + d;
#pragma unroll
          for (int r = 0; r < RP; ++r)
            if (r0 + r < sg.n_rows) out[r * HD] = o[r];
        }
      }
      tc::tc_fence_before();
      a0 += sg.t1 - sg.t0;
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  if (warp == kProduct) tc::tmem_dealloc(tmem, C::kAlloc);
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

int rows_of(int rows) { return rows <= 4 ? 4 : rows <= 8 ? 8 : rows <= 16 ? 16 : rows <= 32 ? 32 : 64; }
int ctas_per_sm(int nr, int hd) { return hd == 256 || nr == 64 ? 1 : 2; }

constexpr int kSmemMax = 227 * 1024;

template <int HD, int NR>
int launch(const AttnArgs& a, UmmaPlan pl, cudaStream_t s) {
  using C = Cfg<HD, NR>;
  // 227 KB per SM, 1 KB of it taken by each CTA
  const int room = 228 * 1024 / C::CTAS - 1024;
  // two slots of each at least: a step's scores are issued before the previous step's sums. A large batch's
  // prefix may leave room for one CTA per SM only
  int slots = 2 * kMaxSlots;
  while (slots > 4 && umma_smem(HD, C::NM, slots, a.batch).bytes > room) --slots;
  const int smem = umma_smem(HD, C::NM, slots, a.batch).bytes;
  if (smem > kSmemMax) return DSM_ERR_UNSUPPORTED;
  pl.k_slots = slots / 2;
  pl.v_slots = slots - pl.k_slots;
  // All that a CTA may have, whatever this call takes: the kernel's limit is every host thread's. Before the maps:
  // cuTensorMapEncodeTiled wants a current context, which a host thread's first runtime call makes
  auto kern = kv8_umma_kernel<HD, NR>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemMax) != cudaSuccess)
    return check_launch("gqa_attn_kv8 smem attribute");
  CUtensorMap kmap{}, vmap{};
  const int64_t groups = int64_t(a.n_pages) * a.n_kv * (a.page / kTile);
  int st = byte_map(&vmap, a.v_codes, groups * HD, kTile, kTile, HD, true);
  if (st == DSM_OK && HD == 64) st = byte_map(&kmap, a.k_codes, groups * kTile, 64, 64, kTile, true);
  if (st == DSM_OK && HD == 256) st = byte_map(&kmap, a.k_codes, groups * kTile, 256, 128, kTile, false);
  if (st != DSM_OK) return st;
  kern<<<unsigned(pl.sp.ctas), C::kThreads, size_t(smem), s>>>(a, pl, kmap, vmap);
  st = check_launch("gqa_attn_kv8");
  return st != DSM_OK ? st : kv8_combine(a, pl.sp, HD, DSM_DT_BF16, s);
}

template <int HD>
int launch_rows(int nr, const AttnArgs& a, const UmmaPlan& pl, cudaStream_t s) {
  switch (nr) {
    case 4: return launch<HD, 4>(a, pl, s);
    case 8: return launch<HD, 8>(a, pl, s);
    case 16: return launch<HD, 16>(a, pl, s);
    case 32: return launch<HD, 32>(a, pl, s);
    default: return launch<HD, 64>(a, pl, s);
  }
}

}  // namespace

size_t kv8_umma_ws_bytes(int rows, int hd) {
  const int nr = rows_of(rows);
  return split_ws_bytes(ctas_per_sm(nr, hd) * num_sms(), nr, hd);
}

int kv8_umma(const AttnArgs& a, int hd, void* ws, cudaStream_t s) {
  UmmaPlan pl;
  pl.sp.rows = a.n_heads / a.n_kv * a.block;
  const int nr = rows_of(pl.sp.rows);
  pl.sp.row_blocks = int(ceil_div(pl.sp.rows, nr));
  pl.sp.cta_rows = nr;
  const int64_t groups = int64_t(a.n_pages) * a.n_kv * (a.page / kTile);
  const int64_t most = int64_t(a.batch) * a.max_pages * (a.page / kTile) * a.n_kv * pl.sp.row_blocks;
  if (groups * std::max(hd, kTile) > 0x7fffffff) return DSM_ERR_UNSUPPORTED;  // rows of the TMA maps
  // a row's place in its sequence's result is kept in 32 bits
  if (int64_t(a.block) * a.n_heads * hd > 0x7fffffff) return DSM_ERR_UNSUPPORTED;
  const int most_ctas = ctas_per_sm(nr, hd) * num_sms();
  pl.sp.ctas = int(std::min<int64_t>(most_ctas, most));
  // A unit's staging, first step and result take as long as ten tiles. Measured at 28 rows of head_dim 128 for 61 ragged
  // sequences and for 16 equal ones: cost 6 / 10 / 14 92, 81, 74 us and 37, 38, 39; at head_dim 64 and 256 and 4, 16, 28
  // and 56 rows, ragged, cost 6 is up to 22% slower than 10, and 14 from 4% faster to 8% slower (4 rows of 256).
  // Cuts that move further leave uneven ranges (snap 0 / 2 / 4 / 8: 81, 81, 79, 78 us and 39, 38, 40, 47; 4 instead of
  // 2 is 1% faster to 9% slower at the other widths), none at all leave one short request's units in pieces (11.4 us ->
  // 13.3). Ranges of at least 4, 8 or 12 tiles' cost differ by 2%, but at 16 rows, where 12 is 9 to 13% slower.
  pl.sp.cost = 10;
  pl.sp.snap = 2;
  pl.sp.least = 8;
  if (!split_fits(a, pl.sp)) return DSM_ERR_UNSUPPORTED;
  split_ws(pl.sp, ws, hd);
  pl.vec_q = vec_ok(a.q, a.q_batch, a.q_row, a.q_head, 8);
  pl.vec_blk = a.blk_k && vec_ok(a.blk_k, a.bk_batch, a.bk_head, a.bk_row, 8) &&
               vec_ok(a.blk_v, a.bv_batch, a.bv_head, a.bv_row, 8);
  switch (hd) {
    case 64: return launch_rows<64>(nr, a, pl, s);
    case 128: return launch_rows<128>(nr, a, pl, s);
    default: return launch_rows<256>(nr, a, pl, s);
  }
}

}  // namespace dsm
