// dsm_kv8_append: rows k, v [n_rows, n_kv, head_dim] into the slots of a slot map of the paged 8-bit
// cache (layout in kv8.cuh), as e4m3 codes with one power-of-two scale per page and KV head:
// s = 2^e, e the least with max|x| <= 448 * 2^e over the page's rows so far. No reference
// counterpart: the reference keeps its context K/V in the activation dtype
// (dspark_mlx/arch/qwen3.py:122-143).
//
// The scale is exact (a maximum and its exponent), a code is rounded once, to nearest even; a scale that
// grows shifts the codes already there by whole octaves, which rounds again only what falls into e4m3's
// subnormals.
//
// What bounds it: a long prompt by reading the rows and writing half as many bytes (bf16), a decode step by
// latency: the slots, the rows, the scale and the codes wait for one another. Hence a run's rows are read
// once and kept in registers where one tile holds them, short runs go to a warp each, side by side, and the
// two passes share one loop, since each instruction that runs once costs a fetch. 30,705 rows x 8 heads of
// 128 in bf16 take 46 us (3.0 TB/s; 290 us with a CTA per row and byte stores), half of it issue, half
// latency at 24 warps per SM; 64 runs of up to 8 rows x 8 heads 6.4 us, 5 runs of 300 fp32 rows 7.4 us. With 4
// CTAs per SM the compiler spills (50 us), with one window for all sizes a decode step's runs wait in line.
#include "kv8.cuh"

namespace dsm {
namespace {

constexpr int kAppendThreads = 256;
constexpr int kAppendWarps = kAppendThreads / 32;

// x + 0 y, for both halves: NaN where y is not finite, else x
__device__ __forceinline__ uint64_t nan_unless_finite(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(y), "l"(0ull), "l"(x));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t x, uint64_t y) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
  return r;
}
__device__ __forceinline__ uint64_t pair(uint32_t lo, uint32_t hi) { return lo | uint64_t(hi) << 32; }
__device__ __forceinline__ float lo_of(uint64_t x) { return __uint_as_float(uint32_t(x)); }
__device__ __forceinline__ float hi_of(uint64_t x) { return __uint_as_float(uint32_t(x >> 32)); }

struct AppendArgs {
  const void *k, *v;
  int64_t n_rows;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  const int64_t* slots;
  int n_kv, page, n_pages;
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  int window;         // rows per CTA, at most 64
  uint32_t per_page;  // kv8_per_page
};

// The page of slot s, -1 for a row that is skipped (slot < 0, or outside the pool).
__device__ __forceinline__ int slot_page(const AppendArgs& p, int64_t s) {
  if (s < 0 || s >= int64_t(p.n_pages) * p.page) return -1;
  const uint64_t u = uint64_t(s) / kKv8Group;
  if (p.per_page == 0) return int(u);
  return u < (1u << 28) ? int(__umulhi(unsigned(u), p.per_page)) : int(u / (unsigned(p.page) / kKv8Group));
}

// eight neighbouring values of a row
template <typename T>
struct Eight {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < int(sizeof(T) / 2); ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  template <bool VEC>
  __device__ __forceinline__ void load(const T* src) {
    if constexpr (VEC) {
#pragma unroll
      for (int i = 0; i < int(sizeof(T) / 2); ++i) w[i] = __ldg(reinterpret_cast<const uint4*>(src) + i);
    } else {
      uint32_t x[2 * sizeof(T)];
      if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __float_as_uint(src[i]);
      } else {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(src);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = h[2 * i] | uint32_t(h[2 * i + 1]) << 16;
      }
#pragma unroll
      for (int i = 0; i < int(sizeof(T) / 2); ++i) w[i] = make_uint4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
    }
  }
  __device__ __forceinline__ void get(uint64_t (&x)[4]) const {
    const uint4 u = w[0], v = w[sizeof(T) / 4];
    if constexpr (sizeof(T) == 4) {
      x[0] = pair(u.x, u.y);
      x[1] = pair(u.z, u.w);
      x[2] = pair(v.x, v.y);
      x[3] = pair(v.z, v.w);
    } else {
      x[0] = pair(u.x << 16, u.x & 0xffff0000u);
      x[1] = pair(u.y << 16, u.y & 0xffff0000u);
      x[2] = pair(u.z << 16, u.z & 0xffff0000u);
      x[3] = pair(u.w << 16, u.w & 0xffff0000u);
    }
  }
  // the largest |x| and m: what is not finite takes no part in it (fmaxf drops a NaN)
  __device__ __forceinline__ float amax(float m) const {
    uint64_t x[4];
    get(x);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[i] = nan_unless_finite(x[i], x[i]);
      m = fmaxf(m, fmaxf(fabsf(lo_of(x[i])), fabsf(hi_of(x[i]))));
    }
    return m;
  }
  // bf16: the largest |x| and m as bits, in two halves
  __device__ __forceinline__ uint32_t top_bits(uint32_t m) const {
    const uint32_t u[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) asm("max.u16x2 %0, %0, %1;" : "+r"(m) : "r"(u[i] & 0x7fff7fffu));
    return m;
  }
  // the codes of x / scale: what is not finite becomes NaN (e4m3 has no infinity)
  __device__ __forceinline__ uint2 codes(float inv) const {
    uint64_t x[4];
    get(x);
    const uint64_t f = pair(__float_as_uint(inv), __float_as_uint(inv));
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = nan_unless_finite(mul2(x[i], f), x[i]);
    return make_uint2(kv8_from_f32(lo_of(x[0]), hi_of(x[0]), lo_of(x[1]), hi_of(x[1])),
                      kv8_from_f32(lo_of(x[2]), hi_of(x[2]), lo_of(x[3]), hi_of(x[3])));
  }
};

// the largest finite |x| of them and m
template <typename T, int N>
__device__ __forceinline__ float amax_of(const Eight<T>* x, float m) {
  if constexpr (sizeof(T) == 2) {
    uint32_t b = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) b = x[i].top_bits(b);
    const uint32_t lo = b & 0xffffu, hi = b >> 16;
    if (max(lo, hi) < 0x7f80u) return fmaxf(m, __uint_as_float(max(lo, hi) << 16));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) m = x[i].amax(m);
  return m;
}

// rows r0 .. r0 + n - 1 of one page; `straight`: they are tokens t0, t0 + 1, ... of it
struct Run {
  int64_t r0;
  int n, page, t0;
  bool fresh, straight;
};

// A team of TEAM threads (a warp, or the CTA) writes a run, TEAM / 4 tokens at a time: the largest finite |x|,
// the scale (and the shift of the codes that are there), the codes. A run of one tile stays in registers
// between the two passes. A thread of the keys holds eight columns of a row, neighbouring threads the row; a
// thread of the values holds eight columns of four tokens, neighbouring threads the next tokens, so that
// after a 4 x 4 byte transposition a column's 64-byte row of the cache is written by neighbouring threads.
template <typename T, int HD, bool VEC, int TEAM>
__device__ __forceinline__ void append_run(const AppendArgs& p, const Run run, int h, int tid, float* red) {
  constexpr int kTokens = TEAM / 4, kChunks = HD / 8, kQuads = kTokens / 4;
  constexpr int NK = kChunks / 4, NV = (kChunks + 15) / 16;  // items per thread
  const int64_t ph = int64_t(run.page) * p.n_kv + h;
  const float old_k = p.k_scale[ph], old_v = p.v_scale[ph];
  // tile i holds rows i * kTokens - lead ...: a straight run's tiles begin at multiples of four tokens, the
  // CTA's at groups of the values
  const int lead = run.straight ? run.t0 % (TEAM == 32 ? 4 : kTokens) : 0;
  const int tiles = (run.n + lead + kTokens - 1) / kTokens;
  const int kr = tid / kChunks - lead, vr = tid % kQuads * 4 - lead;  // the thread's first row of tile 0
  constexpr int kStep = TEAM / kChunks;  // rows between its items of the keys; of the values, columns
  const T* const k0 = static_cast<const T*>(p.k) + (run.r0 + kr) * p.k_row + h * p.k_head + tid % kChunks * 8;
  const T* const v0 = static_cast<const T*>(p.v) + (run.r0 + vr) * p.v_row + h * p.v_head + tid / kQuads * 8;
  Eight<T> kx[NK], vx[NV * 4];
  auto load = [&](int first) {
    const T* k = k0 + first * p.k_row;
#pragma unroll
    for (int j = 0; j < NK; ++j, k += kStep * p.k_row) {
      kx[j].zero();
      if (unsigned(first + kr + j * kStep) < unsigned(run.n)) kx[j].template load<VEC>(k);
    }
    const T* v = v0 + first * p.v_row;
#pragma unroll
    for (int i = 0; i < 4; ++i, v += p.v_row) {
      const bool in = unsigned(first + vr + i) < unsigned(run.n);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        vx[j * 4 + i].zero();
        if (in && (kChunks >= 16 || tid / kQuads < kChunks)) vx[j * 4 + i].template load<VEC>(v + j * (TEAM / kQuads * 8));
      }
    }
  };
  auto token = [&](int r) {
    return run.straight ? run.t0 + r : int(p.slots[run.r0 + r] - int64_t(run.page) * p.page);
  };
  float mk = 0.f, mv = 0.f, ik = 0.f, iv = 0.f;
  uint8_t* const kc = p.k_codes + ph * p.page * HD;
  uint8_t* const vc = p.v_codes + ph * p.page * HD;
  // the tiles twice, in one loop: cold instructions cost more than its branches
#pragma unroll 1
  for (int it = 0; it < 2 * tiles; ++it) {
    const int first = (it < tiles ? it : it - tiles) * kTokens;
    if (it == 0 || tiles > 1) load(first);
    if (it < tiles) {
      mk = amax_of<T, NK>(kx, mk);
      mv = amax_of<T, 4 * NV>(vx, mv);
      if (it < tiles - 1) continue;
      mk = kv8_warp_max(mk);
      mv = kv8_warp_max(mv);
      auto sync = [] {
        if constexpr (TEAM == 32)
          __syncwarp();
        else
          __syncthreads();
      };
      if constexpr (TEAM > 32) {
        if ((tid & 31) == 0) {
          red[tid >> 5] = mk;
          red[TEAM / 32 + (tid >> 5)] = mv;
        }
        sync();
#pragma unroll
        for (int w = 0; w < TEAM / 32; ++w) {
          mk = fmaxf(mk, red[w]);
          mv = fmaxf(mv, red[TEAM / 32 + w]);
        }
      }
      int ek = kv8_scale_exp(mk), ev = kv8_scale_exp(mv);
      if (!run.fresh) {  // rows are there already: their scale holds, or grows and their codes shrink with it
        const int ok = min(max(kv8_exponent(old_k), kKv8MinExp), kKv8MaxExp);
        const int ov = min(max(kv8_exponent(old_v), kKv8MinExp), kKv8MaxExp);
#pragma unroll 1
        for (int which = 0; which < 2; ++which) {
          const int was = which ? ov : ok, now = which ? ev : ek;
          if (now <= was) continue;
          const float ratio = was - now < -126 ? 0.f : kv8_exp2i(was - now);
          uint4* c = reinterpret_cast<uint4*>(which ? vc : kc);
#pragma unroll 2
          for (int i = tid; i < p.page * HD / 16; i += TEAM) {
            uint4 w = c[i];
            uint32_t* u = &w.x;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              float x[4];
              kv8_to_f32(u[j], x);
              u[j] = kv8_from_f32(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
            }
            c[i] = w;
          }
        }
        ek = max(ek, ok);
        ev = max(ev, ov);
      }
      if (tid == 0) {
        p.k_scale[ph] = kv8_exp2i(ek);
        p.v_scale[ph] = kv8_exp2i(ev);
      }
      sync();  // the old codes are rewritten before new ones land among them, the scales read before the next run's
      ik = kv8_exp2i(-ek);
      iv = kv8_exp2i(-ev);
      continue;
    }
#pragma unroll
    for (int j = 0; j < NK; ++j) {
      const int r = first + kr + j * kStep, c = tid % kChunks;
      if (unsigned(r) >= unsigned(run.n)) continue;
      const int t = token(r);
      *reinterpret_cast<uint2*>(kc + t * HD + kv8_key_chunk<HD>(c / 2, t) * 16 + c % 2 * 8) = kx[j].codes(ik);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int r = first + vr, c = tid / kQuads + j * (TEAM / kQuads);
      if (c >= kChunks || r + 3 < 0 || r >= run.n) continue;
      uint2 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = vx[j * 4 + i].codes(iv);
      uint32_t col[8];  // a column's four tokens
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint32_t w0 = m ? w[0].y : w[0].x, w1 = m ? w[1].y : w[1].x, w2 = m ? w[2].y : w[2].x,
                       w3 = m ? w[3].y : w[3].x;
        const uint32_t a = __byte_perm(w0, w1, 0x5140), b = __byte_perm(w2, w3, 0x5140);
        const uint32_t d = __byte_perm(w0, w1, 0x7362), e = __byte_perm(w2, w3, 0x7362);
        col[4 * m] = __byte_perm(a, b, 0x5410);
        col[4 * m + 1] = __byte_perm(a, b, 0x7632);
        col[4 * m + 2] = __byte_perm(d, e, 0x5410);
        col[4 * m + 3] = __byte_perm(d, e, 0x7632);
      }
      if (run.straight && r >= 0 && r + 3 < run.n) {
        const int t = run.t0 + r;
        uint8_t* dst = vc + t / kKv8Group * HD * kKv8Group + c * 8 * kKv8Group + t % kKv8Group;
#pragma unroll
        for (int d = 0; d < 8; ++d) *reinterpret_cast<uint32_t*>(dst + d * kKv8Group) = col[d];
      } else {
        const int to = min(4, run.n - r);
#pragma unroll 1
        for (int i = max(-r, 0); i < to; ++i) {
          const int t = token(r + i);
          uint8_t* dst = vc + t / kKv8Group * HD * kKv8Group + c * 8 * kKv8Group + t % kKv8Group;
#pragma unroll
          for (int d = 0; d < 8; ++d) dst[d * kKv8Group] = uint8_t(col[d] >> (8 * i));
        }
      }
    }
  }
}

// The CTA of (window, KV head) writes the runs (consecutive rows of one page) that start in its window: a run is
// one team's, which alone owns the page's scale. Runs of up to kShort rows go to a warp each, side by side; a
// longer one takes the CTA.
constexpr int kShort = 16;

template <typename T, int HD, bool VEC>
__global__ void __launch_bounds__(kAppendThreads, sizeof(T) == 2 && HD <= 128 ? 3 : HD * sizeof(T) <= 512 ? 2 : 1)
    kv8_append_kernel(const AppendArgs p) {
  __shared__ float red[2 * kAppendWarps];
  __shared__ unsigned change_sm[kAppendWarps], bent_sm[kAppendWarps], zero_sm[kAppendWarps], start_sm[2];
  __shared__ int run_end[kAppendWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int h = int(blockIdx.x % unsigned(p.n_kv));
  const int64_t w0 = int64_t(blockIdx.x / unsigned(p.n_kv)) * p.window;
  {  // the rows from the window's first on, one per thread
    const int64_t r = w0 + tid;
    const int64_t s = r < p.n_rows ? p.slots[r] : -1;
    const int64_t s0 = lane == 0 && r > 0 && r < p.n_rows ? p.slots[r - 1] : -1;
    const int pg = slot_page(p, s);
    const int64_t s1 = __shfl_up_sync(0xffffffffu, s, 1);
    const int p1 = __shfl_up_sync(0xffffffffu, pg, 1);
    const int64_t before = lane == 0 ? s0 : s1;
    const int pb = lane == 0 ? slot_page(p, s0) : p1;
    if (tid < p.window && s >= 0 && pg < 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
    const unsigned start = __ballot_sync(0xffffffffu, tid < p.window && pg >= 0 && pg != pb);
    const unsigned change = __ballot_sync(0xffffffffu, pg < 0 || pg != pb);
    const unsigned bent = __ballot_sync(0xffffffffu, s != before + 1);
    const unsigned zero = __ballot_sync(0xffffffffu, pg >= 0 && s == int64_t(pg) * p.page);
    if (lane == 0) {
      if (warp < 2) start_sm[warp] = start;
      change_sm[warp] = change;
      bent_sm[warp] = bent;
      zero_sm[warp] = zero;
    }
  }
  __syncthreads();
  uint64_t starts = start_sm[0] | uint64_t(start_sm[1]) << 32;
  if (starts == 0) return;
  auto end_of = [&](int b) {  // the row behind the run that starts at row b, kAppendThreads where none is seen
    int w = b >> 5;
    unsigned m = change_sm[w] & (0xfffffffeu << (b & 31));
    while (m == 0 && ++w < kAppendWarps) m = change_sm[w];
    return m ? w * 32 + __ffs(m) - 1 : kAppendThreads;
  };
  auto run_at = [&](int b, int e) {
    const int64_t s = p.slots[w0 + b];
    Run run;
    run.r0 = w0 + b;
    run.n = e - b;
    run.page = slot_page(p, s);
    run.t0 = int(s - int64_t(run.page) * p.page);
    unsigned fresh = 0, bent = 0;
    for (int w = b >> 5; w * 32 < e; ++w) {
      const unsigned mine = (w == b >> 5 ? 0xffffffffu << (b & 31) : 0xffffffffu) &
                            (e - w * 32 < 32 ? (1u << (e - w * 32)) - 1 : 0xffffffffu);
      fresh |= zero_sm[w] & mine;
      bent |= bent_sm[w] & mine & ~(w == b >> 5 ? 1u << (b & 31) : 0u);
    }
    run.fresh = fresh != 0;
    run.straight = bent == 0;
    return run;
  };
  uint64_t wide = 0;  // the runs that take the CTA
  for (int i = 0; starts; starts &= starts - 1) {
    const int b = __ffsll(starts) - 1;
    const int e = end_of(b);
    if (e - b > kShort)
      wide |= 1ull << b;
    else if (i++ % kAppendWarps == warp)
      append_run<T, HD, VEC, 32>(p, run_at(b, e), h, lane, nullptr);
  }
  for (; wide; wide &= wide - 1) {
    const int b = __ffsll(wide) - 1, e = end_of(b);
    Run run = run_at(b, e);
    if (e == kAppendThreads) {  // it may go on behind them
      for (int64_t base = w0 + kAppendThreads;; base += kAppendThreads) {
        const int64_t r = base + tid;
        const int64_t s = r < p.n_rows ? p.slots[r] : -1;
        const bool in = slot_page(p, s) == run.page;
        const unsigned vote = __ballot_sync(0xffffffffu, in);
        if (lane == 0) run_end[warp] = vote == 0xffffffffu ? 32 : __ffs(~vote) - 1;
        __syncthreads();
        int len = 0;
        for (int w = 0; w < kAppendWarps; ++w) {
          len += run_end[w];
          if (run_end[w] < 32) break;
        }
        const bool counts = tid < len;
        run.fresh |= __syncthreads_or(counts && s == int64_t(run.page) * p.page) != 0;
        run.straight &= __syncthreads_and(!counts || s == p.slots[r - 1] + 1) != 0;
        run.n += len;
        if (len < kAppendThreads) break;
      }
    }
    append_run<T, HD, VEC, kAppendThreads>(p, run, h, tid, red);
  }
}

}  // namespace
}  // namespace dsm

using namespace dsm;

extern "C" int dsm_kv8_append(const void* k, const void* v, int dtype, int64_t n_rows, int n_kv, int head_dim,
                              int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                              int64_t v_head_stride, const int64_t* slot_map, int page_size, int n_pages,
                              uint8_t* k_codes, uint8_t* v_codes, float* k_scale, float* v_scale, void* stream) {
  DSM_REQUIRE(n_rows >= 0 && n_rows <= 0x7fffffff && n_kv > 0 && n_kv <= 65535 && n_pages > 0,
              "dsm_kv8_append: bad shape");
  DSM_REQUIRE(kv8_head_dim_ok(head_dim), "dsm_kv8_append: head_dim must be 64, 128 or 256");
  DSM_REQUIRE(kv8_page_ok(page_size), "dsm_kv8_append: page_size must be a multiple of 64, at most 1024");
  DSM_REQUIRE(dtype == DSM_DT_F32 || dtype == DSM_DT_BF16, "dsm_kv8_append: dtype must be F32 or BF16");
  DSM_REQUIRE(k_row_stride >= 0 && k_head_stride >= 0 && v_row_stride >= 0 && v_head_stride >= 0,
              "dsm_kv8_append: bad strides");
  if (n_rows == 0) return DSM_OK;
  DSM_REQUIRE(k && v && slot_map && k_codes && v_codes && k_scale && v_scale, "dsm_kv8_append: NULL pointer");
  DSM_REQUIRE(kv8_aligned16(k_codes) && kv8_aligned16(v_codes), "dsm_kv8_append: codes must be 16-byte aligned");
  const size_t bytes = dtype == DSM_DT_F32 ? 4 : 2;
  const bool vec = kv8_aligned16(k) && kv8_aligned16(v) && k_row_stride * bytes % 16 == 0 &&
                   k_head_stride * bytes % 16 == 0 && v_row_stride * bytes % 16 == 0 && v_head_stride * bytes % 16 == 0;
  // Windows of a page's least rows where that makes CTAs enough (8 rows there: four times as many CTAs that
  // find no run to write); of 8 rows where it does not
  const int window = ceil_div(n_rows, int64_t(64)) * n_kv >= 4 * num_sms() ? 64 : 8;
  const uint32_t per_page = kv8_per_page(page_size);
  const AppendArgs a = {k,       v,       n_rows,  k_row_stride, k_head_stride, v_row_stride, v_head_stride, slot_map, n_kv,
                        page_size, n_pages, k_codes, v_codes,      k_scale,       v_scale,      window,   per_page};
  const int64_t grid = ceil_div(n_rows, int64_t(window)) * n_kv;  // a window's heads are neighbours: so are their rows
  DSM_REQUIRE(grid <= 0x7fffffff, "dsm_kv8_append: more rows and heads than one launch holds");
  cudaStream_t s = as_stream(stream);
  auto pick = [&](auto hd) {
    constexpr int HD = decltype(hd)::value;
    using B = __nv_bfloat16;
    if (dtype == DSM_DT_BF16) return vec ? kv8_append_kernel<B, HD, true> : kv8_append_kernel<B, HD, false>;
    return vec ? kv8_append_kernel<float, HD, true> : kv8_append_kernel<float, HD, false>;
  };
  auto kernel = head_dim == 64    ? pick(std::integral_constant<int, 64>())
                : head_dim == 128 ? pick(std::integral_constant<int, 128>())
                                  : pick(std::integral_constant<int, 256>());
  kernel<<<unsigned(grid), kAppendThreads, 0, s>>>(a);
  return check_launch("kv8_append");
}

