// dsm_kv8_append: rows k, v [n_rows, n_kv, head_dim] into the slots of a slot map of the paged 8-bit
// cache (layout in kv8.cuh), as e4m3 codes with one power-of-two scale per page and KV head:
// s = 2^e, e the least with max|x| <= 448 * 2^e over the page's rows so far. No reference
// counterpart: the reference keeps its context K/V in the activation dtype
// (dspark_mlx/arch/qwen3.py:122-143).
#include "kv8.cuh"

namespace dsm {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendWarps = kAppendThreads / 32;

// |x| for the scale: what is not finite takes no part in it
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a <= 3.402823466e38f ? a : 0.f;
}
// x / scale for the code: what is not finite becomes NaN (e4m3 has no infinity)
__device__ __forceinline__ float scaled(float x, float inv) {
  return fabsf(x) <= 3.402823466e38f ? x * inv : __int_as_float(0x7fffffff);
}

struct AppendArgs {
  const void *k, *v;
  int64_t n_rows;
  int64_t k_row, k_head, v_row, v_head;  // strides in elements
  const int64_t* slots;
  int n_kv, page, n_pages;
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
};

// The page of row r, -1 for a row that is skipped (slot < 0, or outside the pool).
__device__ __forceinline__ int row_page(const AppendArgs& p, int64_t r) {
  const int64_t s = p.slots[r];
  return s >= 0 && s < int64_t(p.n_pages) * p.page ? int(s / p.page) : -1;
}

// One CTA per (row, KV head). The CTA of a run's first row (consecutive rows of one page) writes
// the whole run: it alone owns the page's scale. The others leave at once.
template <typename T, int HD>
__global__ void __launch_bounds__(kAppendThreads) kv8_append_kernel(const AppendArgs p) {
  __shared__ float red[2][kAppendWarps];
  __shared__ int run_end[kAppendWarps];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t r0 = blockIdx.x;
  const int h = blockIdx.y;
  const int pg = row_page(p, r0);
  if (pg < 0) {
    if (p.slots[r0] >= 0 && tid == 0) raise_device_error(DSM_DEV_ERR_PAGE_RANGE);
    return;
  }
  if (r0 > 0 && row_page(p, r0 - 1) == pg) return;
  // the run's length, and whether it starts the page afresh (token 0 is among its rows)
  int64_t n = 0;
  bool fresh = false;
  for (int64_t base = r0;; base += kAppendThreads) {
    const int64_t r = base + tid;
    const bool in = r < p.n_rows && row_page(p, r) == pg;
    const unsigned vote = __ballot_sync(0xffffffffu, in);
    if (lane == 0) run_end[warp] = vote == 0xffffffffu ? 32 : __ffs(~vote) - 1;
    __syncthreads();
    int len = 0;
    for (int w = 0; w < kAppendWarps; ++w) {
      len += run_end[w];
      if (run_end[w] < 32) break;
    }
    fresh |= __syncthreads_or(in && tid < len && p.slots[r] % p.page == 0);
    n += len;
    if (len < kAppendThreads) break;
  }
  const T* k = static_cast<const T*>(p.k) + r0 * p.k_row + h * p.k_head;
  const T* v = static_cast<const T*>(p.v) + r0 * p.v_row + h * p.v_head;
  float mk = 0.f, mv = 0.f;
  for (int64_t i = tid; i < n * HD; i += kAppendThreads) {
    const int64_t r = i / HD;
    const int d = int(i % HD);
    mk = fmaxf(mk, finite_abs(ld_f(k, r * p.k_row + d)));
    mv = fmaxf(mv, finite_abs(ld_f(v, r * p.v_row + d)));
  }
  mk = kv8_warp_max(mk);
  mv = kv8_warp_max(mv);
  if (lane == 0) {
    red[0][warp] = mk;
    red[1][warp] = mv;
  }
  const int64_t ph = int64_t(pg) * p.n_kv + h;
  const float old_k = p.k_scale[ph], old_v = p.v_scale[ph];
  __syncthreads();
  for (int w = 0; w < kAppendWarps; ++w) {
    mk = fmaxf(mk, red[0][w]);
    mv = fmaxf(mv, red[1][w]);
  }
  int ek = kv8_scale_exp(mk), ev = kv8_scale_exp(mv);
  uint8_t* kc = p.k_codes + ph * p.page * HD;
  uint8_t* vc = p.v_codes + ph * p.page * HD;
  if (!fresh) {  // rows are there already: their scale holds, or grows and their codes shrink with it
    const int ok = min(max(kv8_exponent(old_k), kKv8MinExp), kKv8MaxExp);
    const int ov = min(max(kv8_exponent(old_v), kKv8MinExp), kKv8MaxExp);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int was = which ? ov : ok, now = which ? ev : ek;
      if (now <= was) continue;
      const float ratio = was - now < -126 ? 0.f : kv8_exp2i(was - now);
      uint32_t* c = reinterpret_cast<uint32_t*>(which ? vc : kc);
      for (int i = tid; i < p.page * HD / 4; i += kAppendThreads) {
        float x[4];
        kv8_to_f32(c[i], x);
        c[i] = kv8_from_f32(x[0] * ratio, x[1] * ratio, x[2] * ratio, x[3] * ratio);
      }
    }
    ek = max(ek, ok);
    ev = max(ev, ov);
  }
  if (tid == 0) {
    p.k_scale[ph] = kv8_exp2i(ek);
    p.v_scale[ph] = kv8_exp2i(ev);
  }
  __syncthreads();  // the old codes are rewritten before new ones land among them
  const float ik = kv8_exp2i(-ek), iv = kv8_exp2i(-ev);
  for (int64_t i = tid; i < n * (HD / 4); i += kAppendThreads) {
    const int64_t r = i / (HD / 4);
    const int d = int(i % (HD / 4)) * 4;
    const int t = int(p.slots[r0 + r] % p.page);
    const int64_t ok = r * p.k_row + d, ov = r * p.v_row + d;
    *reinterpret_cast<uint32_t*>(kc + t * HD + kv8_key_chunk<HD>(d / 16, t) * 16 + d % 16) =
        kv8_from_f32(scaled(ld_f(k, ok), ik), scaled(ld_f(k, ok + 1), ik), scaled(ld_f(k, ok + 2), ik),
                     scaled(ld_f(k, ok + 3), ik));
    const uint32_t w = kv8_from_f32(scaled(ld_f(v, ov), iv), scaled(ld_f(v, ov + 1), iv), scaled(ld_f(v, ov + 2), iv),
                                    scaled(ld_f(v, ov + 3), iv));
    uint8_t* dst = vc + (t / kKv8Group) * HD * kKv8Group + d * kKv8Group + t % kKv8Group;
#pragma unroll
    for (int j = 0; j < 4; ++j) dst[j * kKv8Group] = uint8_t(w >> (8 * j));
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
  const AppendArgs a = {k,    v,         n_rows,  k_row_stride, k_head_stride, v_row_stride, v_head_stride, slot_map,
                        n_kv, page_size, n_pages, k_codes,      v_codes,       k_scale,      v_scale};
  const dim3 grid(unsigned(n_rows), unsigned(n_kv), 1);
  cudaStream_t s = as_stream(stream);
  const bool bf = dtype == DSM_DT_BF16;
  if (head_dim == 64)
    bf ? kv8_append_kernel<__nv_bfloat16, 64><<<grid, kAppendThreads, 0, s>>>(a)
       : kv8_append_kernel<float, 64><<<grid, kAppendThreads, 0, s>>>(a);
  else if (head_dim == 128)
    bf ? kv8_append_kernel<__nv_bfloat16, 128><<<grid, kAppendThreads, 0, s>>>(a)
       : kv8_append_kernel<float, 128><<<grid, kAppendThreads, 0, s>>>(a);
  else
    bf ? kv8_append_kernel<__nv_bfloat16, 256><<<grid, kAppendThreads, 0, s>>>(a)
       : kv8_append_kernel<float, 256><<<grid, kAppendThreads, 0, s>>>(a);
  return check_launch("kv8_append");
}

