// The 8-bit KV cache's two users (layout in kv8.cuh; no reference counterpart: the reference keeps
// its context K/V in the activation dtype, dspark_mlx/arch/qwen3.py:122-143).
//
//   dsm_kv8_append    rows k, v [n_rows, n_kv, head_dim] into the slots of a slot map, as e4m3 codes
//                     with one power-of-two scale per page and KV head: s = 2^e, e the least with
//                     max|x| <= 448 * 2^e over the page's rows so far.
//   dsm_gqa_attn_kv8  grouped-query attention of q [batch, block, n_heads, head_dim] over each
//                     sequence's cached rows and then the block's own rows.
#include "kv8.cuh"

namespace dsm {
namespace {

constexpr int kAppendThreads = 128;
constexpr int kAppendWarps = kAppendThreads / 32;

__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

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
  mk = warp_max(mk);
  mv = warp_max(mv);
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

// ------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------
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
    const float m_new = fmaxf(m, warp_max(x));
    const float ref = m_new == -INFINITY ? 0.f : m_new;
    const float alpha = expf(m - ref), w = expf(x - ref);
    l = l * alpha + warp_sum(w);
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
      const float m_new = fmaxf(m, warp_max(x));
      const float ref = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = expf(m - ref), w = expf(x - ref);
      l = l * alpha + warp_sum(w);
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

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool head_dim_ok(int hd) { return hd == 64 || hd == 128 || hd == 256; }
bool page_ok(int page) { return page > 0 && page % kKv8Group == 0 && page <= kKv8MaxPage; }

}  // namespace
}  // namespace dsm

using namespace dsm;

extern "C" int dsm_kv8_append(const void* k, const void* v, int dtype, int64_t n_rows, int n_kv, int head_dim,
                              int64_t k_row_stride, int64_t k_head_stride, int64_t v_row_stride,
                              int64_t v_head_stride, const int64_t* slot_map, int page_size, int n_pages,
                              uint8_t* k_codes, uint8_t* v_codes, float* k_scale, float* v_scale, void* stream) {
  DSM_REQUIRE(n_rows >= 0 && n_rows <= 0x7fffffff && n_kv > 0 && n_kv <= 65535 && n_pages > 0,
              "dsm_kv8_append: bad shape");
  DSM_REQUIRE(head_dim_ok(head_dim), "dsm_kv8_append: head_dim must be 64, 128 or 256");
  DSM_REQUIRE(page_ok(page_size), "dsm_kv8_append: page_size must be a multiple of 64, at most 1024");
  DSM_REQUIRE(dtype == DSM_DT_F32 || dtype == DSM_DT_BF16, "dsm_kv8_append: dtype must be F32 or BF16");
  DSM_REQUIRE(k_row_stride >= 0 && k_head_stride >= 0 && v_row_stride >= 0 && v_head_stride >= 0,
              "dsm_kv8_append: bad strides");
  if (n_rows == 0) return DSM_OK;
  DSM_REQUIRE(k && v && slot_map && k_codes && v_codes && k_scale && v_scale, "dsm_kv8_append: NULL pointer");
  DSM_REQUIRE(aligned16(k_codes) && aligned16(v_codes), "dsm_kv8_append: codes must be 16-byte aligned");
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

extern "C" size_t dsm_gqa_attn_kv8_workspace_bytes(int batch, int block, int n_heads, int n_kv, int head_dim) {
  if (batch <= 0 || batch > kKv8MaxBatch || block <= 0 || n_kv <= 0 || n_heads <= 0 || n_heads % n_kv != 0 ||
      !head_dim_ok(head_dim))
    return 0;
  return 16;
}

extern "C" int dsm_gqa_attn_kv8(const dsm_kv8_attn_desc* d, const void* q, const int32_t* block_table,
                                const int32_t* lengths, const void* blk_k, const void* blk_v, void* out, void* ws,
                                size_t ws_bytes, void* stream) {
  DSM_REQUIRE(d != nullptr, "dsm_gqa_attn_kv8: desc is NULL");
  DSM_REQUIRE(d->batch >= 0 && d->batch <= kKv8MaxBatch, "dsm_gqa_attn_kv8: batch must be 0..8192");
  DSM_REQUIRE(d->block > 0 && d->n_kv > 0 && d->n_heads > 0 && d->n_heads % d->n_kv == 0,
              "dsm_gqa_attn_kv8: bad shape (n_heads must be a multiple of n_kv)");
  DSM_REQUIRE(head_dim_ok(d->head_dim), "dsm_gqa_attn_kv8: head_dim must be 64, 128 or 256");
  DSM_REQUIRE(page_ok(d->page_size), "dsm_gqa_attn_kv8: page_size must be a multiple of 64, at most 1024");
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
  DSM_REQUIRE(aligned16(d->k_codes) && aligned16(d->v_codes), "dsm_gqa_attn_kv8: codes must be 16-byte aligned");
  DSM_REQUIRE(aligned16(ws), "dsm_gqa_attn_kv8: workspace must be 16-byte aligned");
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
