// Latent attention: every token's keys and values come from one shared latent
// row (512 values at the model's shape) and one rotary row (64).
//
// Absorbed form (decode).  The queries are already in the latent space, so
// for token t and head h over the request's cached rows c_j, r_j
//   s_j = scale (q_latent . c_j + q_rope . r_j),  o = sum_j softmax(s)_j c_j.
// Expanded form (prefill).  Keys [k_nope_h | k_rope] and values v_h of every
// head are given; causal rows see the keys up to their own position.
//
// One block per (token, head): eight warps walk the keys, each with its own
// running maximum and sum, and the eight results are joined in shared memory.
#include <algorithm>
#include <cmath>

#include "latent.cuh"

namespace glm53 {
namespace latent {
namespace {

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxDim = 640;    // query values of a head (nope or latent, and rotary)
constexpr int kMaxValue = 512;  // two 8-value pieces a lane

struct Joined {
  float q[kMaxDim];
  float o[kWarps][kMaxValue];
  float m[kWarps], l[kWarps];
};

// One (token, head): keys(j, a, b, v) gives key j's two parts and value row.
template <typename E, typename Keys>
__device__ __forceinline__ void attend(Joined& sm, const uint16_t* qa, int da, const uint16_t* qb, int db, int dv,
                                       int64_t visible, float scale, uint16_t* out, float* lse, Keys keys) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < da + db; i += kThreads)
    sm.q[i] = Elem<E>::to_float(i < da ? qa[i] : qb[i - da]);
  __syncthreads();
  float m = -INFINITY, l = 0.f, acc[2][8] = {};
  for (int64_t j = warp; j < visible; j += kWarps) {
    const uint16_t *ka, *kb, *kv;
    keys(j, ka, kb, kv);
    float s = 0.f;
    for (int v = lane; v < (da + db) >> 3; v += 32) {
      const int e = v * 8;
      float f[8];
      unpack8<E>(*reinterpret_cast<const uint4*>(e < da ? ka + e : kb + e - da), f);
#pragma unroll
      for (int i = 0; i < 8; ++i) s = fmaf(sm.q[e + i], f[i], s);
    }
    s = warp_sum(s) * scale;
    const float top = fmaxf(m, s);
    const float base = top == -INFINITY ? 0.f : top;
    const float keep = __expf(m - base), p = __expf(s - base);
    l = l * keep + p;
    m = top;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int v = lane + 32 * i;
      if (v * 8 < dv) {
        float f[8];
        unpack8<E>(*reinterpret_cast<const uint4*>(kv + v * 8), f);
#pragma unroll
        for (int k = 0; k < 8; ++k) acc[i][k] = fmaf(p, f[k], acc[i][k] * keep);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int v = lane + 32 * i;
    if (v * 8 < dv)
      for (int k = 0; k < 8; ++k) sm.o[warp][v * 8 + k] = acc[i][k];
  }
  if (lane == 0) {
    sm.m[warp] = m;
    sm.l[warp] = l;
  }
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
  for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm.m[w]);
  const float base = top == -INFINITY ? 0.f : top;
  for (int w = 0; w < kWarps; ++w) sum += sm.l[w] * __expf(sm.m[w] - base);
  const float inv = visible > 0 ? 1.f / sum : 0.f;
  for (int i = threadIdx.x; i < dv; i += kThreads) {
    float o = 0.f;
    for (int w = 0; w < kWarps; ++w) o = fmaf(sm.o[w][i], __expf(sm.m[w] - base), o);
    out[i] = visible > 0 ? Elem<E>::from_float(o * inv) : (uint16_t)0;
  }
  if (lse && threadIdx.x == 0) *lse = visible > 0 ? top + logf(sum) : -INFINITY;
}

// Largest i with starts[i] <= t among starts[0..n - 1].
__device__ __forceinline__ int request_of(const int32_t* starts, int n, int t) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= t)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

struct AbsorbedArgs {
  const uint16_t *ql, *qr;
  int64_t ql_t, ql_h, qr_t, qr_h;
  int64_t T;
  int H, R, r;
  const uint16_t* cache;
  int64_t pages;
  int page;
  const int32_t* table;
  int64_t table_stride, table_width;
  const int32_t* lens;
  int B;
  const int32_t* starts;
  float scale;
  uint16_t* out;
  float* lse;
  int fill_tail;
  uint32_t *status, *status_host;
};

template <typename E>
__global__ void __launch_bounds__(kThreads) absorbed_kernel(AbsorbedArgs a) {
  __shared__ Joined sm;
  const int t = blockIdx.x, h = blockIdx.y;
  int i = t;
  int64_t len = 0, back = 0;
  bool tail = false;
  if (a.starts) {
    tail = a.B == 0 || t >= a.starts[a.B];
    if (!tail) {
      i = request_of(a.starts, a.B, t);
      back = (int64_t)a.starts[i + 1] - 1 - t;
      if (back < 0) tail = true;  // starts that do not ascend
    }
  }
  if (tail && !a.fill_tail) return;
  if (!tail) {
    len = a.lens[i];
    if (len < 0 || len > a.table_width * a.page) {
      if (threadIdx.x == 0) report(a.status, a.status_host, kStatusBadGeometry);
      len = 0;
    }
  }
  const int64_t visible = len - back;
  const int width = a.R + a.r;
  const int32_t* row = a.table + (tail ? 0 : i * a.table_stride);
  attend<E>(sm, a.ql + t * a.ql_t + h * a.ql_h, a.R, a.qr + t * a.qr_t + h * a.qr_h, a.r, a.R,
            visible > 0 ? visible : 0, a.scale, a.out + ((int64_t)t * a.H + h) * a.R,
            a.lse ? a.lse + (int64_t)t * a.H + h : nullptr,
            [&](int64_t j, const uint16_t*& ka, const uint16_t*& kb, const uint16_t*& kv) {
              const int64_t at = j / a.page;
              int32_t id = row[at];
              if (id < 0 || id >= a.pages) {
                report(a.status, a.status_host, kStatusBadPage);
                id = 0;
              }
              ka = a.cache + ((int64_t)id * a.page + (j - at * a.page)) * width;
              kb = ka + a.R;
              kv = ka;
            });
}

bool stride_ok(int64_t s) { return s >= 0 && s % 8 == 0 && s < (int64_t)1 << 38; }

}  // namespace
}  // namespace latent
}  // namespace glm53

using namespace glm53;
using namespace glm53::latent;

extern "C" size_t glm53_latent_absorbed_workspace_bytes(int64_t tokens, int64_t heads, int64_t latent_dim) {
  (void)tokens;
  (void)heads;
  (void)latent_dim;
  return 256;
}

extern "C" int glm53_latent_absorbed(const void* q_latent, int64_t ql_stride_t, int64_t ql_stride_h,
                                     const void* q_rope, int64_t qr_stride_t, int64_t qr_stride_h, int64_t tokens,
                                     int64_t heads, int64_t latent_dim, int64_t rope_dim, int dtype, const void* cache,
                                     int64_t pages, int64_t page_size, const int32_t* block_table,
                                     int64_t table_stride, int64_t table_width, const int32_t* seq_lens,
                                     int64_t requests, const int32_t* query_starts, float scale, void* out, float* lse,
                                     int fill_tail, void* workspace, size_t workspace_bytes, uint32_t* status,
                                     uint32_t* status_host, void* stream) {
  const char* fn = "glm53_latent_absorbed";
  if (dtype != GLM53_DTYPE_BF16 && dtype != GLM53_DTYPE_FP16) {
    set_last_error("%s: unknown element type %d", fn, dtype);
    return GLM53_ERR_INVALID;
  }
  if (latent_dim <= 0 || latent_dim % 128 != 0 || latent_dim > 512 || (rope_dim != 0 && rope_dim != 64)) {
    set_last_error("%s: latent size %lld must be 128, 256, 384 or 512 and the rotary size %lld 0 or 64", fn,
                   (long long)latent_dim, (long long)rope_dim);
    return GLM53_ERR_INVALID;
  }
  if (tokens < 0 || tokens > INT32_MAX || heads < 1 || heads > 1024 || requests < 0 || requests > INT32_MAX ||
      pages < 0 || page_size < 8 || page_size % 8 != 0 || page_size > INT32_MAX || pages > INT32_MAX / page_size ||
      table_width < 0 || table_stride < table_width || table_width > INT32_MAX / page_size) {
    set_last_error("%s: %lld heads (1 to 1024), pages of %lld rows (a multiple of 8), %lld pages and a table of %lld: "
                   "cache rows and positions are 32-bit",
                   fn, (long long)heads, (long long)page_size, (long long)pages, (long long)table_width);
    return GLM53_ERR_INVALID;
  }
  if (!std::isfinite(scale) || !stride_ok(ql_stride_t) || !stride_ok(ql_stride_h) || ql_stride_h < latent_dim ||
      (rope_dim && (!stride_ok(qr_stride_t) || !stride_ok(qr_stride_h) || qr_stride_h < rope_dim))) {
    set_last_error("%s: the scale must be finite and strides non-negative multiples of 8", fn);
    return GLM53_ERR_INVALID;
  }
  if (!query_starts && tokens != requests) {
    set_last_error("%s: without query_starts there is one token a request (%lld tokens, %lld requests)", fn,
                   (long long)tokens, (long long)requests);
    return GLM53_ERR_INVALID;
  }
  if (tokens == 0) return GLM53_OK;
  if (!q_latent || (rope_dim && !q_rope) || !out || (requests && !seq_lens) ||
      (requests && table_width && !block_table) || (pages && !cache) ||
      (((uintptr_t)q_latent | (uintptr_t)q_rope | (uintptr_t)cache | (uintptr_t)out) & 15)) {
    set_last_error("%s: tensors must be non-NULL and 16-byte aligned", fn);
    return GLM53_ERR_INVALID;
  }
  if (!workspace || workspace_bytes < glm53_latent_absorbed_workspace_bytes(tokens, heads, latent_dim)) {
    set_last_error("%s: the workspace is too small", fn);
    return GLM53_ERR_INVALID;
  }
  AbsorbedArgs a{(const uint16_t*)q_latent, (const uint16_t*)q_rope, ql_stride_t, ql_stride_h, qr_stride_t, qr_stride_h,
                 tokens, (int)heads, (int)latent_dim, (int)rope_dim, (const uint16_t*)cache, pages, (int)page_size,
                 block_table, table_stride, table_width, seq_lens, (int)requests, query_starts, scale, (uint16_t*)out,
                 lse, fill_tail, status, status_host};
  const dim3 grid((unsigned)tokens, (unsigned)heads);
  if (dtype == GLM53_DTYPE_BF16)
    absorbed_kernel<__nv_bfloat16><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a);
  else
    absorbed_kernel<__half><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a);
  return check_launch(fn);
}
