// Page planning and row stores of the paged latent cache.
//
// glm53_plan_pages.  With P rows a page, request i holds ceil(cached_i / P)
// pages and needs ceil((cached_i + new_i) / P); two exclusive prefix sums over
// the requests (new tokens, new pages) place every token and every page, so
// token t of request i at position p = cached_i + t - start_i goes to row
// table[i][p / P] * P + p % P of the cache, and new page j of the batch is
// free[count - 1 - j].  A few KB are read and 12 bytes a token written: the
// call is bound by latency, so it is one launch.  Every block scans all
// requests itself (two loads a request from L2) instead of waiting for
// another block, and a token on a new page takes its page from the free list
// rather than from the table another block is writing.
//
// glm53_latent_cache_write.  One row a token: [x[:R] * rsqrt(mean(x[:R]^2) +
// eps) * w | x[R:] turned by position * inv_freq], rounded once, stored at the
// token's slot; the queries' rotary parts turn by the same angles in the same
// launch.  Bound by HBM: every value is read and written once, in 16-byte
// pieces.
#include <algorithm>

#include "latent.cuh"

namespace glm53 {
namespace latent {
namespace {

constexpr int kPlanThreads = 256;
constexpr int64_t kPlanMaxRequests = 8192;  // two prefix arrays of this length fit shared memory
constexpr int kWriteThreads = 256;
constexpr int64_t kMaxLatent = 1024;
constexpr int64_t kMaxRope = 256;

struct PlanArgs {
  const int32_t* cached;
  const int32_t* fresh;  // new tokens
  int B;
  int32_t* table;
  int64_t table_stride, table_width;
  const int32_t* free_pages;
  int64_t free_capacity;
  const int32_t* free_count;
  int page;
  int64_t tokens;
  int64_t* slots;
  int32_t* positions;
  int32_t* query_starts;
  int32_t* seq_lens;
  int32_t* free_count_out;
  uint32_t* status;
  uint32_t* status_host;
};

__device__ __forceinline__ int64_t pages_of(int64_t rows, int page) { return (rows + page - 1) / page; }

// Largest i with start[i] <= v, over start[0..n] ascending with start[0] = 0
// and v < start[n].
__device__ __forceinline__ int find_run(const int32_t* start, int n, int32_t v) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= v)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

__global__ void __launch_bounds__(kPlanThreads) plan_pages_kernel(PlanArgs a) {
  extern __shared__ int32_t plan_smem[];
  int32_t* tok = plan_smem;               // [B + 1] first token of each request
  int32_t* pgs = plan_smem + (a.B + 1);   // [B + 1] first new page of each request
  __shared__ int64_t warp_tok[kPlanThreads / 32], warp_pg[kPlanThreads / 32];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (a.B + kPlanThreads - 1) / kPlanThreads;
  const int i0 = min(a.B, tid * per), i1 = min(a.B, i0 + per);
  const int64_t count = *a.free_count;
  int64_t ntok = 0, npg = 0;
  bool bad = count < 0 || count > a.free_capacity;
  for (int i = i0; i < i1; ++i) {
    const int64_t c = a.cached[i], n = a.fresh[i];
    if (c < 0 || n < 0 || c + n > a.table_width * a.page) {
      bad = true;
      continue;
    }
    ntok += n;
    npg += pages_of(c + n, a.page) - pages_of(c, a.page);
  }
  // block-wide exclusive scan of both sums, in request order
  int64_t st = ntok, sp = npg;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t t = __shfl_up_sync(0xffffffffu, st, o), p = __shfl_up_sync(0xffffffffu, sp, o);
    if (lane >= o) {
      st += t;
      sp += p;
    }
  }
  if (lane == 31) {
    warp_tok[warp] = st;
    warp_pg[warp] = sp;
  }
  __syncthreads();
  int64_t tok_total = 0, pg_total = 0, tok0 = 0, pg0 = 0;
#pragma unroll
  for (int w = 0; w < kPlanThreads / 32; ++w) {
    if (w == warp) {
      tok0 = tok_total;
      pg0 = pg_total;
    }
    tok_total += warp_tok[w];
    pg_total += warp_pg[w];
  }
  bad = __syncthreads_or(bad || tok_total > a.tokens || pg_total > count);
  if (!bad) {
    int64_t t = tok0 + st - ntok, p = pg0 + sp - npg;
    for (int i = i0; i < i1; ++i) {
      tok[i] = (int32_t)t;
      pgs[i] = (int32_t)p;
      const int64_t c = a.cached[i], n = a.fresh[i];
      t += n;
      p += pages_of(c + n, a.page) - pages_of(c, a.page);
    }
    if (tid == kPlanThreads - 1) {
      tok[a.B] = (int32_t)tok_total;
      pgs[a.B] = (int32_t)pg_total;
    }
  }
  __syncthreads();

  const int64_t stride = (int64_t)gridDim.x * blockDim.x, first = (int64_t)blockIdx.x * blockDim.x + tid;
  if (blockIdx.x == 0 && tid == 0) {
    *a.free_count_out = (int32_t)(bad ? count : count - pg_total);
    if (bad) report(a.status, a.status_host, kStatusNoPages);
  }
  for (int64_t i = first; i <= a.B; i += stride) {
    a.query_starts[i] = bad ? 0 : tok[i];
    if (i < a.B) a.seq_lens[i] = bad ? a.cached[i] : a.cached[i] + a.fresh[i];
  }
  if (bad) {
    for (int64_t t = first; t < a.tokens; t += stride) {
      a.slots[t] = -1;
      a.positions[t] = 0;
    }
    return;
  }
  for (int64_t j = first; j < pg_total; j += stride) {
    const int i = find_run(pgs, a.B, (int32_t)j);
    a.table[i * a.table_stride + pages_of(a.cached[i], a.page) + (j - pgs[i])] = a.free_pages[count - 1 - j];
  }
  for (int64_t t = first; t < a.tokens; t += stride) {
    int64_t slot = -1;
    int32_t pos = 0;
    if (t < tok_total) {
      const int i = find_run(tok, a.B, (int32_t)t);
      const int32_t c = a.cached[i];
      pos = c + (int32_t)t - tok[i];
      const int64_t held = pages_of(c, a.page), at = pos / a.page;
      const int32_t id = at < held ? a.table[i * a.table_stride + at]
                                   : a.free_pages[count - 1 - (pgs[i] + (at - held))];
      if (id >= 0)
        slot = (int64_t)id * a.page + (pos - at * a.page);
      else
        report(a.status, a.status_host, kStatusBadPage);
    }
    a.slots[t] = slot;
    a.positions[t] = pos;
  }
}

struct WriteArgs {
  const uint16_t* kv;
  int64_t T, kv_stride;
  int latent, rope;
  const uint16_t* weight;  // nullptr: stored unnormalised
  float eps;
  const int32_t* positions;  // nullptr: stored unrotated
  const double* inv_freq;
  int interleaved;
  const int64_t* slots;
  uint16_t* cache;
  int64_t cache_rows;
  const uint16_t* q;  // nullptr: no queries
  int heads;
  int64_t q_stride_t, q_stride_h;
  uint16_t* q_out;
  uint32_t* status;
  uint32_t* status_host;
};

// cos and sin of position * inv_freq.  A position of 10^6 leaves a 32-bit
// angle 0.06 rad off, so the turn count is formed and reduced in 64 bits and
// only its fraction goes to 32.
__device__ __forceinline__ float2 turn_of(int32_t position, double inv_freq) {
  const double turns = (double)position * inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  const float f = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.0f * f, &s, &c);
  return make_float2(c, s);
}

// What a warp loads of token t's row, all at once: the slot, the first 512
// latent values and the first rotary pair a lane, raw.
struct Row {
  int64_t slot;
  uint4 raw[2];
  uint16_t u, w;
};
// where rotary pair p lies in a row
__device__ __forceinline__ int2 pair_at(const WriteArgs& a, int p) {
  const int e = a.latent + (a.interleaved ? 2 * p : p);
  return make_int2(e, e + (a.interleaved ? 1 : a.rope >> 1));
}
__device__ __forceinline__ Row load_row(const WriteArgs& a, int64_t t, int lane) {
  Row row;
  const uint16_t* x = a.kv + t * a.kv_stride;
  row.slot = a.slots[t];
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 32 * i < a.latent >> 3) row.raw[i] = reinterpret_cast<const uint4*>(x)[lane + 32 * i];
  if (lane < a.rope >> 1) {
    const int2 e = pair_at(a, lane);
    row.u = x[e.x];
    row.w = x[e.y];
  }
  return row;
}

template <typename E>
__device__ __forceinline__ void write_row(const WriteArgs& a, int64_t t, int lane, const float2* turns,
                                          const Row& row) {
  if (row.slot < 0) return;
  if (row.slot >= a.cache_rows) {
    if (lane == 0) report(a.status, a.status_host, kStatusBadPage);
    return;
  }
  const uint16_t* x = a.kv + t * a.kv_stride;
  uint16_t* y = a.cache + row.slot * (a.latent + a.rope);
  const uint4* xv = reinterpret_cast<const uint4*>(x);
  const int vecs = a.latent >> 3;
  // what is beyond the first 512 values is read again
  float sq = 0.f;
  auto square = [&](uint4 w) {
    float f[8];
    unpack8<E>(w, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) sq = fmaf(f[j], f[j], sq);
  };
  float r = 1.f;
  if (a.weight) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 32 * i < vecs) square(row.raw[i]);
    for (int v = lane + 64; v < vecs; v += 32) square(xv[v]);
    r = 1.0f / sqrtf(warp_sum(sq) / (float)a.latent + a.eps);
  }
  auto store = [&](int v, uint4 p) {
    if (a.weight) {
      float f[8], w[8];
      unpack8<E>(p, f);
      unpack8<E>(__ldg(reinterpret_cast<const uint4*>(a.weight) + v), w);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = f[j] * r * w[j];
      p = pack8<E>(f);
    }
    reinterpret_cast<uint4*>(y)[v] = p;
  };
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (lane + 32 * i < vecs) store(lane + 32 * i, row.raw[i]);
  for (int v = lane + 64; v < vecs; v += 32) store(v, xv[v]);
  for (int p = lane; p < a.rope >> 1; p += 32) {
    const int2 e = pair_at(a, p);
    const uint16_t u16 = p == lane ? row.u : x[e.x], w16 = p == lane ? row.w : x[e.y];
    if (a.positions) {
      const float u = Elem<E>::to_float(u16), w = Elem<E>::to_float(w16);
      const float2 cs = turns ? turns[p] : turn_of(a.positions[t], a.inv_freq[p]);
      y[e.x] = Elem<E>::from_float(u * cs.x - w * cs.y);
      y[e.y] = Elem<E>::from_float(w * cs.x + u * cs.y);
    } else {
      y[e.x] = u16;
      y[e.y] = w16;
    }
  }
}

// Without queries: a warp a token.  With queries: a block a token, whose last
// warp forms the angles for all heads and stores the row while the others'
// loads are on their way (4,096 tokens of 64 heads, 77 MB: 29.3 us when the
// loads waited for the angles, 16.1 us so).  A piece pair a thread is quickest
// while the blocks run at once, blocks of fewer threads when they take turns,
// with more tokens' angles and loads on their way.  64 heads, 256 / 64 threads
// beside that warp: 1 token 2.9 / 3.3 us, 888 (6 blocks an SM) 4.6 / 4.8, 1,500
// 7.2 / 6.1, 4,096 16.1 / 12.7, 16,384 68 / 53; 16 heads, 64 pairs: 600 3.4 / 3.1.
constexpr int kWideQueries = 256, kWideBlocks = 6;
constexpr int kNarrowQueries = 64, kNarrowBlocks = 16;

template <typename E>
__global__ void __launch_bounds__(kWriteThreads) latent_write_kernel(WriteArgs a) {
  const int64_t t = (int64_t)blockIdx.x * (kWriteThreads / 32) + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (t < a.T) write_row<E>(a, t, lane, nullptr, load_row(a, t, lane));
}

// The two 8-value pieces that piece pair v of a head turns: values 8 v and
// rope / 2 + 8 v, or 16 v and 16 v + 8 when neighbours pair up.
template <typename E>
__device__ __forceinline__ void turn_pieces(const WriteArgs& a, const float2* turns, int v, uint4& p, uint4& q) {
  float x[8], y[8];
  unpack8<E>(p, x);
  unpack8<E>(q, y);
  if (a.interleaved) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 c0 = turns[8 * v + j], c1 = turns[8 * v + 4 + j];
      const float u0 = x[2 * j], w0 = x[2 * j + 1], u1 = y[2 * j], w1 = y[2 * j + 1];
      x[2 * j] = u0 * c0.x - w0 * c0.y;
      x[2 * j + 1] = w0 * c0.x + u0 * c0.y;
      y[2 * j] = u1 * c1.x - w1 * c1.y;
      y[2 * j + 1] = w1 * c1.x + u1 * c1.y;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float2 cs = turns[8 * v + j];
      const float u = x[j], w = y[j];
      x[j] = u * cs.x - w * cs.y;
      y[j] = w * cs.x + u * cs.y;
    }
  }
  p = pack8<E>(x);
  q = pack8<E>(y);
}

// QUERIES: threads that turn queries
template <typename E, int QUERIES, int BLOCKS>
__global__ void __launch_bounds__(QUERIES + 32, BLOCKS) latent_write_queries_kernel(WriteArgs a) {
  __shared__ float2 turns[kMaxRope / 2];
  const int64_t t = blockIdx.x;
  const int half = a.rope >> 1;
  if (threadIdx.x >= QUERIES) {
    const int lane = threadIdx.x & 31;
    const int32_t position = a.positions[t];
    const Row row = load_row(a, t, lane);
    for (int p = lane; p < half; p += 32) turns[p] = turn_of(position, a.inv_freq[p]);
    __syncthreads();
    write_row<E>(a, t, lane, turns, row);
    return;
  }
  const int pieces = a.rope >> 4, items = a.heads * pieces;  // pairs of pieces: of a head, in all
  const uint16_t* q = a.q + t * a.q_stride_t;
  uint16_t* out = a.q_out + t * a.heads * a.rope;
  auto at = [&](int v, int second) { return a.interleaved ? 16 * v + 8 * second : 8 * v + half * second; };
  auto load = [&](int i, uint4& x, uint4& y) {
    const int h = i / pieces, v = i - h * pieces;
    const uint16_t* src = q + h * a.q_stride_h;
    x = ldg_stream(reinterpret_cast<const uint4*>(src + at(v, 0)));
    y = ldg_stream(reinterpret_cast<const uint4*>(src + at(v, 1)));
  };
  uint4 x, y;
  int i = threadIdx.x;
  if (i < items) load(i, x, y);
  __syncthreads();
  while (i < items) {
    const int h = i / pieces, v = i - h * pieces;
    turn_pieces<E>(a, turns, v, x, y);
    uint16_t* dst = out + h * a.rope;
    *reinterpret_cast<uint4*>(dst + at(v, 0)) = x;
    *reinterpret_cast<uint4*>(dst + at(v, 1)) = y;
    i += QUERIES;
    if (i < items) load(i, x, y);
  }
}

template <typename E>
void launch_write(const WriteArgs& a, cudaStream_t st) {
  if (a.q) {
    if ((int64_t)a.heads * (a.rope >> 4) > kNarrowQueries && a.T <= (int64_t)kWideBlocks * sm_count())
      latent_write_queries_kernel<E, kWideQueries, kWideBlocks><<<(unsigned)a.T, kWideQueries + 32, 0, st>>>(a);
    else
      latent_write_queries_kernel<E, kNarrowQueries, kNarrowBlocks><<<(unsigned)a.T, kNarrowQueries + 32, 0, st>>>(a);
  } else {
    const int64_t blocks = (a.T + kWriteThreads / 32 - 1) / (kWriteThreads / 32);
    latent_write_kernel<E><<<(unsigned)blocks, kWriteThreads, 0, st>>>(a);
  }
}

}  // namespace
}  // namespace latent
}  // namespace glm53

using namespace glm53;
using namespace glm53::latent;

extern "C" int glm53_plan_pages(const int32_t* cached_lens, const int32_t* new_lens, int64_t requests,
                                int32_t* block_table, int64_t table_stride, int64_t table_width,
                                const int32_t* free_pages, int64_t free_capacity, const int32_t* free_count,
                                int64_t page_size, int64_t tokens, int64_t* slots, int32_t* positions,
                                int32_t* query_starts, int32_t* seq_lens, int32_t* free_count_out, uint32_t* status,
                                uint32_t* status_host, void* stream) {
  const char* fn = "glm53_plan_pages";
  if (requests < 0 || requests > kPlanMaxRequests) {
    set_last_error("%s: %lld requests are outside [0, %lld]", fn, (long long)requests, (long long)kPlanMaxRequests);
    return GLM53_ERR_INVALID;
  }
  if (page_size < 1 || table_width < 0 || table_stride < table_width || free_capacity < 0 || tokens < 0 ||
      page_size > INT32_MAX || table_width > INT32_MAX / page_size || tokens > INT32_MAX) {
    set_last_error("%s: page size %lld, table width %lld, tokens %lld: sizes are non-negative and positions 32-bit", fn,
                   (long long)page_size, (long long)table_width, (long long)tokens);
    return GLM53_ERR_INVALID;
  }
  if (!query_starts || !free_count || !free_count_out || free_count == free_count_out ||
      (requests && (!cached_lens || !new_lens || !seq_lens)) || (requests && table_width && !block_table) ||
      (free_capacity && !free_pages) || (tokens && (!slots || !positions))) {
    set_last_error("%s: missing tensor, or free_count_out is free_count", fn);
    return GLM53_ERR_INVALID;
  }
  PlanArgs a{cached_lens, new_lens, (int)requests, block_table, table_stride, table_width, free_pages, free_capacity,
             free_count, (int)page_size, tokens, slots, positions, query_starts, seq_lens, free_count_out, status,
             status_host};
  const size_t smem = 2 * (size_t)(requests + 1) * sizeof(int32_t);
  const int rc = ensure_max_smem((const void*)plan_pages_kernel, 2 * (kPlanMaxRequests + 1) * sizeof(int32_t));
  if (rc) return rc;
  // a thread a token or request, at most one block an SM: each block repeats the
  // scan, and a thread's chain of loads is long (512 requests, 8,600 tokens: 8.3 us
  // with four tokens a thread, 5.0 with one)
  const int64_t items = std::max(tokens, requests);
  const int64_t blocks =
      std::min<int64_t>(sm_count(), std::max<int64_t>(1, (items + kPlanThreads - 1) / kPlanThreads));
  plan_pages_kernel<<<(unsigned)blocks, kPlanThreads, smem, (cudaStream_t)stream>>>(a);
  return check_launch(fn);
}

extern "C" int glm53_latent_cache_write(const void* kv, int64_t tokens, int64_t kv_stride, int64_t latent_dim,
                                        int64_t rope_dim, int dtype, const void* norm_weight, float eps,
                                        const int32_t* positions, const double* inv_freq, int interleaved,
                                        const int64_t* slots, void* cache, int64_t cache_rows, const void* queries,
                                        int64_t heads, int64_t q_stride_t, int64_t q_stride_h, void* queries_out,
                                        uint32_t* status, uint32_t* status_host, void* stream) {
  const char* fn = "glm53_latent_cache_write";
  if (dtype != GLM53_DTYPE_BF16 && dtype != GLM53_DTYPE_FP16) {
    set_last_error("%s: unknown element type %d", fn, dtype);
    return GLM53_ERR_INVALID;
  }
  if (tokens < 0 || tokens > INT32_MAX || latent_dim <= 0 || latent_dim % 8 != 0 || latent_dim > kMaxLatent ||
      rope_dim < 0 || rope_dim % 16 != 0 || rope_dim > kMaxRope || kv_stride < latent_dim + rope_dim ||
      kv_stride % 8 != 0 || cache_rows < 0) {
    set_last_error("%s: latent %lld (a multiple of 8, at most %lld), rotary %lld (a multiple of 16, at most %lld), row "
                   "stride %lld (a multiple of 8)",
                   fn, (long long)latent_dim, (long long)kMaxLatent, (long long)rope_dim, (long long)kMaxRope,
                   (long long)kv_stride);
    return GLM53_ERR_INVALID;
  }
  if ((positions != nullptr) != (inv_freq != nullptr) || (positions && rope_dim == 0)) {
    set_last_error("%s: positions and inv_freq come together, with a rotary part", fn);
    return GLM53_ERR_INVALID;
  }
  if (queries && (!positions || !queries_out || heads < 1 || heads > 4096 || q_stride_h < 0 ||
                  q_stride_t < 0 || q_stride_h % 8 != 0 || q_stride_t % 8 != 0)) {
    set_last_error("%s: queries need positions, an output, 1 to 4096 heads and strides that are multiples of 8 from 0 on",
                   fn);
    return GLM53_ERR_INVALID;
  }
  if (tokens == 0) return GLM53_OK;
  if (!kv || !slots || !cache ||
      (((uintptr_t)kv | (uintptr_t)cache | (uintptr_t)norm_weight | (uintptr_t)queries | (uintptr_t)queries_out) & 15)) {
    set_last_error("%s: tensors must be non-NULL and 16-byte aligned", fn);
    return GLM53_ERR_INVALID;
  }
  WriteArgs a{(const uint16_t*)kv, tokens, kv_stride, (int)latent_dim, (int)rope_dim, (const uint16_t*)norm_weight,
              eps, positions, inv_freq, interleaved, slots, (uint16_t*)cache, cache_rows, (const uint16_t*)queries,
              (int)heads, q_stride_t, q_stride_h, (uint16_t*)queries_out, status, status_host};
  if (dtype == GLM53_DTYPE_BF16)
    launch_write<__nv_bfloat16>(a, (cudaStream_t)stream);
  else
    launch_write<__half>(a, (cudaStream_t)stream);
  return check_launch(fn);
}
