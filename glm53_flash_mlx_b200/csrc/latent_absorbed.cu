// Latent attention, absorbed form (decode): the queries are in the latent
// space already, so for a token's head h over its request's cached rows
// [c_j | r_j]
//   s_j = scale (q_latent . c_j + q_rope . r_j),  o = sum_j softmax(s)_j c_j.
//
// All heads read the same rows: a row (1,152 bytes at 512 + 64) is used for
// 64 x 2 x 1,088 FLOPs, 121 FLOP a byte against the 259 where this GPU's
// tensor cores and memory balance, so the floor is one pass over the cache.
// The products are formed with the keys on the M side,
//   S^T [64 keys x 64 heads]    = rows . Q^T        (M64 N64, K = 576)
//   O^T [latent x 64 heads]    += c^T . P^T         (4 x M128 N64, K = 64)
// so that 64 heads fill N instead of half of M, O^T needs only 256 of the 512
// TMEM columns, and a row's latent part is the operand of both products from
// one copy in shared memory (K-major for the first, MN-major for the second).
// Measured alone, one thread issuing: 32 cycles an M64 N64 MMA, 48 an M128
// N64, so a tile of 64 rows is 1,920 cycles against ~3,070 of its share of the
// memory bandwidth.
//
// Shared memory holds Q (72 KB), two tiles of 64 rows (72 KB each, filled and
// freed in two halves of the row) and P^T (8 KB).  Inside a half, eight rows
// of each 64-value chunk are one swizzle atom and the chunks of eight rows lie
// side by side, so that one TMA (a 4-D view: 64 values, 8 rows, chunks, row
// groups) brings a half of all rows that are contiguous in the cache, whatever
// the page size.
//
// A CTA per SM takes an equal run of the flattened list of (token, 64 heads,
// tile) units, whatever the lengths: the number of tiles is summed on the
// device, so a captured graph follows its lengths.  A unit that lies within
// one CTA's run is finished there; others leave FP32 partial results (at most
// two a CTA) that a second kernel joins.
//
// Roles: warps 0-7 softmax (a strip of 16 keys and half of the heads each) and
// epilogue, warp 8 TMA, warp 9 issues S^T, warp 10 issues O^T; in the last
// three one lane waits and issues, since a lane that spins must not hold up one
// with work.  Row maxima are replaced only when a score passes them by 2^8
// (latent.cuh).  A token never shares a unit with one that sees fewer rows, so
// only rows behind its own last one are masked: their scores are replaced, and
// their values cleared in shared memory (a zero weight does not remove a NaN)
// up to the 16 rows that an MMA takes.  Every mbarrier wait is bounded, as in
// the expanded form.
//
// 64 requests of 6,000-8,192 rows, 64 heads: 112 us, 4.75 TB/s of rows (72% of
// the measured copy); bound by the life of a stage: load, S^T, softmax and O^T
// of a tile follow one another, and two tiles fit beside Q.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemv_tile.cuh"
#include "kernels.cuh"
#include "latent.cuh"
#include "tcgen05.cuh"

namespace glm53 {
namespace latent {
namespace {

using namespace tc;

constexpr int kKeys = 64;                  // cache rows a tile
constexpr int kMaxHeads = 64;              // heads a unit, at most
constexpr int kChunkBytes = kKeys * 128;   // 64 rows of 64 values
constexpr int kMaxChunks = 9;
constexpr int kAtomBytes = 1024;           // 8 rows of a chunk
constexpr int kStageBytes = kMaxChunks * kChunkBytes;
constexpr int kSoftWarps = 8;
constexpr int kSoftThreads = kSoftWarps * 32;
constexpr int kThreads = kSoftThreads + 96;
constexpr int kMaxGrid = 256;              // CTAs, and so parts of a result, at most
constexpr int kFewTokens = 64;             // of a request, planned by one thread
constexpr int kSCol = 256;                 // TMEM: O^T at 0..255, two S^T tiles behind

struct Args {
  int64_t T;
  int H, R, r, G;  // G groups of 64 heads
  const uint16_t* cache;
  int64_t pages;
  int page, box;   // rows of a page, rows of a TMA box: gcd(page, 64)
  int half[2];     // chunks of the two halves of a row: whole 128-value groups, the rotary part last
  const int32_t* table;
  int64_t table_stride, table_width;
  const int32_t* lens;
  int B;
  const int32_t* starts;
  float c;  // scale log2(e)
  uint16_t* out;
  float* lse;
  int fill_tail;
  uint32_t *status, *status_host;
  // workspace
  int32_t* plan;     // [0] tiles a CTA; then the first tile of every token (-1: outside every request)
  int32_t* counts;   // tiles of every token, one group of heads
  float *po, *pm, *pl;  // partial results [2 grid][64][R], their maxima and sums [2 grid][64]
};

struct Request {
  int q0, nq, len;
  bool bad, disorder;  // disorder: bounds outside the tokens or descending
};
__device__ __forceinline__ Request request_at(const Args& a, int i) {
  Request q{i, 1, a.lens[i], false, false};
  if (a.starts) {
    q.q0 = a.starts[i];
    const int64_t n = (int64_t)a.starts[i + 1] - q.q0;
    q.nq = (int)n;
    if (q.q0 < 0 || n < 0 || q.q0 + n > a.T) {
      q.bad = q.disorder = true;
      q.nq = 0;
    }
  }
  if (q.len < 0 || q.len > a.table_width * a.page) {
    q.bad = true;
    q.len = 0;
  }
  return q;
}
__device__ __forceinline__ int visible_of(const Request& q, int j) { return max(0, q.len - (q.nq - 1 - j)); }
__device__ __forceinline__ int tiles_of(int visible) { return (visible + kKeys - 1) / kKeys; }
// sum over v = 1..n of ceil(v / 64)
__device__ __forceinline__ int64_t tiles_up_to(int64_t n) {
  if (n <= 0) return 0;
  const int64_t q = n / kKeys, r = n % kKeys;
  return kKeys * (q * (q + 1) / 2) + r * (q + 1);
}
// Tiles of all of a request's units (the host checks that the sum over all
// requests stays below 2^31).
__device__ __forceinline__ int tiles_of(const Request& q, int G) {
  const int n = q.nq == 1 ? tiles_of(q.len) : (int)(tiles_up_to(q.len) - tiles_up_to((int64_t)q.len - q.nq));
  return n * G;
}

// A CTA's place in the flattened list: request i, its token j, head group g,
// tile of that unit, and tiles left in the run.
struct Cursor {
  int i, j, g, tile, left;
};
struct Segment {
  int token, g, tile, n, tiles, visible, request;
};
__device__ __forceinline__ bool next_segment(const Args& a, Cursor& c, Segment& s) {
  while (c.left > 0 && c.i < a.B) {
    const Request q = request_at(a, c.i);
    while (c.j < q.nq) {
      const int vis = visible_of(q, c.j), n = tiles_of(vis);
      if (n == 0) {
        ++c.j;
        continue;
      }
      s.token = q.q0 + c.j;
      s.g = c.g;
      s.tile = c.tile;
      s.tiles = n;
      s.visible = vis;
      s.request = c.i;
      s.n = min(c.left, n - c.tile);
      c.left -= s.n;
      c.tile = 0;
      if (++c.g == a.G) {
        c.g = 0;
        ++c.j;
      }
      return true;
    }
    ++c.i;
    c.j = 0;
  }
  return false;
}

struct Bars {
  uint64_t q_full, q_empty, full[2][2], empty[2][2], s_full[2], p_full[2], o_done, drain[2];
  uint32_t tmem_base;
  int abort_flag;
  Cursor cursor;
  int warp_sum[kThreads / 32];
  alignas(16) float factor[kMaxHeads];  // read four at a time
  float top[kMaxHeads];
  float xchg[4][kMaxHeads];
};
// alignment slack, Q, two stages, P^T, barriers
constexpr size_t kSmemBytes = 1024 + 3 * (size_t)kStageBytes + kChunkBytes + 2048;
static_assert(sizeof(Bars) <= 2048, "barriers share two KB");
static_assert((3 * kStageBytes + kChunkBytes) % alignof(Bars) == 0, "where the barriers lie, behind P^T");
static_assert(kSmemBytes <= 232448, "227 KB a CTA");

__device__ __forceinline__ bool mbar_wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  __syncwarp();
  return __all_sync(0xffffffffu, mbar_wait_fast(bar, parity, abort_flag));
}

// N: heads a unit, 16, 32 or 64
template <typename E, int N>
__global__ void __launch_bounds__(kThreads, 1)
    absorbed_kernel(const __grid_constant__ CUtensorMap ql_map, const __grid_constant__ CUtensorMap qr_map,
                    const __grid_constant__ CUtensorMap kv0_map, const __grid_constant__ CUtensorMap kv1_map,
                    Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_smem = smem;
  uint8_t* kv_smem = smem + kStageBytes;
  uint8_t* p_smem = kv_smem + 2 * kStageBytes;
  Bars* bars = reinterpret_cast<Bars*>(p_smem + kChunkBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  auto bar = [&](uint64_t* p) { return smem_addr(p); };

  // the join kernel may be set up beside this one; it waits for its end
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // tiles of all requests, this CTA's run of them, and where it begins
  {
    const int per = (a.B + kThreads - 1) / kThreads;
    const int i0 = min(a.B, tid * per);
    int i1 = min(a.B, i0 + per);
    int n = 0;
    bool disorder = false;
    for (int i = i0; i < i1; ++i) {
      const Request q = request_at(a, i);
      n += tiles_of(q, a.G);
      disorder |= q.disorder;
      if (q.bad && blockIdx.x == 0) report(a.status, a.status_host, kStatusBadGeometry);
    }
    if (warp == 9) {
      tmem_alloc_all<false>(smem_addr(&bars->tmem_base));
    } else if (warp == 8 && lane == 0) {
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&ql_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qr_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kv0_map)) : "memory");
      asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kv1_map)) : "memory");
    } else if (tid == 0) {
      bars->cursor.left = 0;
      bars->abort_flag = 0;
      mbar_init(bar(&bars->q_full), 1);
      mbar_init(bar(&bars->q_empty), 1);
      for (int b = 0; b < 2; ++b) {
        for (int h = 0; h < 2; ++h) {
          mbar_init(bar(&bars->full[b][h]), 1);
          mbar_init(bar(&bars->empty[b][h]), 1);
        }
        mbar_init(bar(&bars->s_full[b]), 1);
        mbar_init(bar(&bars->p_full[b]), kSoftWarps);
        mbar_init(bar(&bars->drain[b]), 1);
      }
      mbar_init(bar(&bars->o_done), 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += x;
    }
    if (lane == 31) bars->warp_sum[warp] = s;
    if (blockIdx.x == 0)
      for (int64_t t = tid; t < a.T; t += kThreads) a.plan[1 + t] = -1;
    // starts out of order, with which two requests could hold one token: no plan
    const bool none = __syncthreads_or(disorder);
    int total = 0, before = s - n;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += bars->warp_sum[w];
      total += bars->warp_sum[w];
    }
    if (none) {
      total = 0;
      i1 = i0;
    }
    const int run = max(1, (int)(((uint32_t)total + gridDim.x - 1) / gridDim.x));
    const int64_t begin = (int64_t)blockIdx.x * run;
    if (blockIdx.x == 0) {
      // what the join looks up: every token's first tile and tiles.  A request
      // with many tokens leaves only its first one's, and the block fills the rest.
      if (tid == 0) a.plan[0] = run;
      bool many = false;
      int f = before;
      for (int i = i0; i < i1; ++i) {
        const Request q = request_at(a, i);
        if (q.nq > kFewTokens) {
          many = true;
          a.plan[1 + q.q0] = f;
          f += tiles_of(q, a.G);
          continue;
        }
        for (int j = 0; j < q.nq; ++j) {
          const int k = tiles_of(visible_of(q, j));
          a.plan[1 + q.q0 + j] = f;
          a.counts[q.q0 + j] = k;
          f += k * a.G;
        }
      }
      if (__syncthreads_or(many)) {
        for (int i = 0; i < a.B; ++i) {
          const Request q = request_at(a, i);
          if (q.nq <= kFewTokens) continue;
          const int at = *(volatile int32_t*)(a.plan + 1 + q.q0);
          const int64_t skipped = tiles_up_to((int64_t)q.len - q.nq);
          __syncthreads();
          for (int j = tid; j < q.nq; j += kThreads) {
            a.plan[1 + q.q0 + j] = at + (int)(tiles_up_to((int64_t)q.len - q.nq + j) - skipped) * a.G;
            a.counts[q.q0 + j] = tiles_of(visible_of(q, j));
          }
        }
      }
    }
    if (begin < total && before <= begin && begin < (int64_t)before + n) {
      int f = before;
      for (int i = i0; i < i1; ++i) {
        const Request q = request_at(a, i);
        const int all = tiles_of(q, a.G);
        if (begin >= f + all) {
          f += all;
          continue;
        }
        // the last token whose first tile is not behind `begin`
        const int64_t skipped = tiles_up_to((int64_t)q.len - q.nq);
        auto first_of = [&](int j) { return f + (int)(tiles_up_to((int64_t)q.len - q.nq + j) - skipped) * a.G; };
        int j = 0, hi = q.nq;
        while (hi - j > 1) {
          const int mid = (j + hi) >> 1;
          if (first_of(mid) <= begin)
            j = mid;
          else
            hi = mid;
        }
        f = first_of(j);
        const int k = tiles_of(visible_of(q, j)), rest = (int)(begin - f);
        const int g = a.G == 1 ? 0 : rest / k;
        bars->cursor = Cursor{i, j, g, rest - g * k, min(run, total - (int)begin)};
        break;
      }
    }
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  volatile int* abort_flag = &bars->abort_flag;
  constexpr bool bf16 = std::is_same<E, __nv_bfloat16>::value;
  const int groups = a.R / 128, halves = a.half[1] ? 2 : 1;
  const int half_bytes = a.half[0] * kChunkBytes;  // of the first half of a tile
  Cursor cur = bars->cursor;
  Segment sg;
  uint32_t n = 0;  // tiles so far, over all segments

  if (warp == 8) {
    // ---------------- TMA ----------------
    // Lane 0 waits and issues; the lanes look up a tile's boxes side by side.
    const int boxes = kKeys / a.box, box_groups = a.box / 8;
    bool ok = true;
    uint32_t queries = 0;  // Q tiles asked for
    int at_half = 0;
    while (next_segment(a, cur, sg)) {
      // lane k looks up box k of a tile: rows pos .. pos + box of the request
      const int32_t* row = a.table + sg.request * a.table_stride;
      auto place = [&](int t) {  // group of eight rows in the cache, -1 for none
        const int pos = t * kKeys + lane * a.box;
        if (lane >= boxes || pos >= sg.visible || t >= sg.tile + sg.n) return -1;
        const int at = pos / a.page;
        const int32_t id = row[at];
        if (id < 0 || id >= a.pages) {
          report(a.status, a.status_host, kStatusBadPage);
          return (int)(a.pages * a.page / 8);  // outside the map: zeros
        }
        return (id * a.page + (pos - at * a.page)) / 8;
      };
      int next = place(sg.tile);
      if (lane == 0) {
        if (queries) ok = ok && mbar_wait_fast(bar(&bars->q_empty), (queries - 1) & 1u, abort_flag);
        if (ok) {
          ++queries;
          mbar_expect_tx(bar(&bars->q_full), (a.R + a.r) / 64 * (N * 128));
          for (int c = 0; c < a.R / 64; ++c)
            tma_load_3d(smem_addr(q_smem + c * (N * 128)), &ql_map, c * 64, sg.g * N, sg.token, bar(&bars->q_full));
          if (a.r)
            tma_load_3d(smem_addr(q_smem + a.R / 64 * (N * 128)), &qr_map, 0, sg.g * N, sg.token,
                        bar(&bars->q_full));
        }
      }
      __syncwarp();
      for (int t = sg.tile; t < sg.tile + sg.n; ++t) {
        const int count = __popc(__ballot_sync(0xffffffffu, next >= 0));
        int y[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) y[k] = __shfl_sync(0xffffffffu, next, k);
        // The next tile is looked up ahead of the waits below, and its rows, one
        // run of memory a box, go into L2 by then: a freed stage is refilled from
        // there, and memory is read in order (64 requests of 6,000-8,192 rows:
        // 119.4 -> 111.7 us; two tiles ahead 115.4, three 122.2; as tensor boxes,
        // 128 bytes of a row at a time, no gain).
        next = place(t + 1);
        if (next >= 0 && next < a.pages * a.page / 8)
          prefetch_l2(a.cache + (int64_t)next * 8 * (a.R + a.r), a.box * (a.R + a.r) * 2);
        if (lane == 0 && ok) {
          const uint32_t b = n & 1, use = n >> 1;
          for (at_half = 0; at_half < halves; ++at_half) {
            const int h = at_half;
            if (use) ok = mbar_wait_fast(bar(&bars->empty[b][h]), (use - 1) & 1u, abort_flag);
            if (!ok) break;
            const int box_bytes = a.half[h] * kAtomBytes * box_groups;
            mbar_expect_tx(bar(&bars->full[b][h]), count * box_bytes);
            const uint32_t dst = smem_addr(kv_smem + b * kStageBytes + h * half_bytes);
#pragma unroll
            for (int k = 0; k < 8; ++k)
              if (k < count)
                tma_load_4d(dst + k * box_bytes, h ? &kv1_map : &kv0_map, 0, 0, h ? a.half[0] : 0, y[k],
                            bar(&bars->full[b][h]));
          }
          if (ok) {
            at_half = 0;
            ++n;
          }
        }
        __syncwarp();
      }
    }
    if (!ok) {
      // copies still in flight write this CTA's shared memory: wait for them
      volatile int never = 0;
      if (queries) mbar_wait(bar(&bars->q_full), (queries - 1) & 1u, &never);
      for (int b = 0; b < 2; ++b)
        for (int h = 0; h < halves; ++h) {
          // the last tile of this stage whose half h was asked for
          const int64_t last = (int64_t)n - ((n & 1) == (uint32_t)b ? (h < at_half ? 0 : 2) : 1);
          never = 0;
          if (last >= 0) mbar_wait(bar(&bars->full[b][h]), (uint32_t)(last >> 1) & 1u, &never);
        }
    }
    __syncwarp();
  } else if (warp == 9) {
    // ---------------- S^T = rows . Q^T ----------------
    // All lanes walk the loops, so that descriptors stay uniform; one waits and issues.
    const bool leader = elect_one();
    constexpr uint32_t id_s = make_idesc_f16(kKeys, N, bf16, false, false);
    const uint64_t qd0 = make_sw128_desc(smem_addr(q_smem));
    bool ok = true;
    for (uint32_t segments = 0; next_segment(a, cur, sg); ++segments) {
      if (leader) ok = ok && mbar_wait_fast(bar(&bars->q_full), segments & 1u, abort_flag);
      for (int t = 0; t < sg.n; ++t, ++n) {
        const uint32_t b = n & 1, use = n >> 1, d = kSCol + b * N;
        // softmax has read the buffer's last tile
        if (leader && use) ok = ok && mbar_wait_fast(bar(&bars->p_full[b]), (use - 1) & 1u, abort_flag);
        for (int h = 0; h < halves; ++h) {
          const uint64_t kd = make_sw128_desc(smem_addr(kv_smem) + b * kStageBytes + h * half_bytes,
                                              a.half[h] * kAtomBytes);
          const uint64_t qd = qd0 + (uint64_t)((h * a.half[0] * N * 128) >> 4);
          const int chunks = a.half[h];
          if (leader) {
            ok = ok && mbar_wait_fast(bar(&bars->full[b][h]), use & 1u, abort_flag);
            tmem_fence_after();
            if (ok) {
              for (int c = 0; c < chunks; ++c) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  mma_f16_ss(d, kd + c * (kAtomBytes >> 4) + 2 * k, qd + c * (N * 128 >> 4) + 2 * k, id_s,
                             (h | c | k) != 0);
              }
            }
          }
        }
        if (leader && ok) mma_commit(bar(&bars->s_full[b]));
      }
      if (leader && ok) mma_commit(bar(&bars->q_empty));
    }
    // no MMA is in flight when TMEM is freed; a lane that spins must not keep its
    // warp from one with work, so the lane that issued waits alone
    if (leader) {
      volatile int never = 0;
      mma_commit(bar(&bars->drain[0]));
      if (!mbar_wait(bar(&bars->drain[0]), 0, &never)) *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp == 10) {
    // ---------------- O^T += c^T . P^T ----------------
    const bool leader = elect_one();
    constexpr uint32_t id_o = make_idesc_f16(128, N, bf16, true, true);
    const uint64_t pd = make_sw128_mn_desc(smem_addr(p_smem), kChunkBytes);
    const int groups0 = min(groups, a.half[0] / 2);
    bool ok = true;
    while (next_segment(a, cur, sg)) {
      for (int t = 0; t < sg.n; ++t, ++n) {
        const uint32_t b = n & 1, use = n >> 1;
        const int valid = min(kKeys, sg.visible - (sg.tile + t) * kKeys);
        const int steps = (valid + 15) >> 4;
        if (leader) {
          ok = ok && mbar_wait_fast(bar(&bars->p_full[b]), use & 1u, abort_flag);
          tmem_fence_after();
        }
        for (int h = 0; h < halves; ++h) {
          const int g0 = h ? groups0 : 0, g1 = h ? groups : groups0;
          const uint64_t vd = make_sw128_mn_desc(smem_addr(kv_smem) + b * kStageBytes + h * half_bytes, kAtomBytes,
                                                 a.half[h] * kAtomBytes);
          const uint32_t step = a.half[h] * (2 * kAtomBytes >> 4);  // 16 keys
          if (leader && ok) {
            for (int g = g0; g < g1; ++g) {
              const uint64_t v = vd + (uint64_t)((g - g0) * (2 * kAtomBytes >> 4));
              if (steps == 4) {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16_ss(g * N, v + k * step, pd + 128 * k, id_o, (t | k) != 0);
              } else {
                for (int k = 0; k < steps; ++k)
                  mma_f16_ss(g * N, v + k * step, pd + 128 * k, id_o, (t | k) != 0);
              }
            }
            mma_commit(bar(&bars->empty[b][h]));
          }
        }
        if (leader && ok) mma_commit(bar(&bars->o_done));
      }
    }
    // no MMA is in flight when TMEM is freed; a lane that spins must not keep its
    // warp from one with work, so the lane that issued waits alone
    if (leader) {
      volatile int never = 0;
      mma_commit(bar(&bars->drain[1]));
      if (!mbar_wait(bar(&bars->drain[1]), 0, &never)) *abort_flag = 1;
    }
    __syncwarp();
  } else {
    // ---------------- softmax, epilogue ----------------
    // this thread's keys of a tile: k0 and k0 + 8; its heads: h0 + 8 j + {0, 1}
    constexpr int kHalf = N / 2, kOwn = N / 8;  // heads of a warp, of a thread
    const int strip = warp & 3, side = warp >> 2;
    const int k0 = 16 * strip + (lane >> 2), h0 = side * kHalf + 2 * (lane & 3);
    const uint32_t lanes = (uint32_t)(strip * 32) << 16;
    bool stop = false;
    for (int segment = 0; !stop && next_segment(a, cur, sg); ++segment) {
      float m[kOwn], l[kOwn];  // m: the maximum in use less kWeightShift, from which weights are counted
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        m[i] = -INFINITY;
        l[i] = 0.f;
      }
      for (int t = 0; t < sg.n; ++t, ++n) {
        const uint32_t b = n & 1, use = n >> 1;
        if (!mbar_wait_warp(bar(&bars->s_full[b]), use & 1u, abort_flag)) stop = true;
        const int valid = min(kKeys, sg.visible - (sg.tile + t) * kKeys);
        float v[2 * kOwn];
        bool grow = stop;
        if (!stop) {
          tmem_fence_after();
          uint32_t w[2 * kOwn];
          tmem_ld16_frag(lanes + kSCol + b * N + side * kHalf, w);
          tmem_wait_ld();
          const bool in0 = k0 < valid, in1 = k0 + 8 < valid;
#pragma unroll
          for (int i = 0; i < 2 * kOwn; ++i)
            v[i] = ((i & 2) ? in1 : in0) ? __uint_as_float(w[i]) * a.c : -INFINITY;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            const int e = (i >> 1) * 4 + (i & 1);
            grow |= fmaxf(v[e], v[e + 2]) - m[i] > kMaxSlack + kWeightShift<E>;
          }
          if (valid < kKeys) {
            // clear the value rows that the last MMA step takes beyond the end
            const int r16 = (valid + 15) & ~15, pieces = a.R / 8;
            for (int i = tid; i < (r16 - valid) * pieces; i += kSoftThreads) {
              const int row = valid + i / pieces, p = i % pieces, c = p >> 3;
              const int h = c >= a.half[0] ? 1 : 0;
              uint8_t* at = kv_smem + b * kStageBytes + h * half_bytes +
                            ((row >> 3) * a.half[h] + c - h * a.half[0]) * kAtomBytes;
              *reinterpret_cast<uint4*>(at + (row & 7) * 128 + (p & 7) * 16) = make_uint4(0, 0, 0, 0);
            }
          }
        }
        if (any_of(grow, 1, kSoftThreads)) {
          stop = any_of(stop, 1, kSoftThreads);
          if (stop) break;
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            const int e = (i >> 1) * 4 + (i & 1);
            float x = fmaxf(v[e], v[e + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            if (lane < 4) bars->xchg[strip][8 * (i >> 1) + h0 + (i & 1)] = x;
          }
          bar_sync(1, kSoftThreads);
#pragma unroll
          for (int i = 0; i < kOwn; ++i) {
            const int h = 8 * (i >> 1) + h0 + (i & 1);
            const float top = fmaxf(m[i], fmaxf(fmaxf(bars->xchg[0][h], bars->xchg[1][h]),
                                                fmaxf(bars->xchg[2][h], bars->xchg[3][h])) - kWeightShift<E>);
            const float f = top == m[i] ? 1.f : ex2(m[i] - top);
            m[i] = top;
            l[i] *= f;
            if (strip == 0 && lane < 4) bars->factor[h] = f;
          }
          bar_sync(1, kSoftThreads);
          if (t > 0 && mbar_wait_warp(bar(&bars->o_done), (n - 1) & 1u, abort_flag)) {
            tmem_fence_after();
            for (int o = 16 * side; o < groups * N; o += 32) {
              uint32_t w[16];
              tmem_ld16(lanes + o, w);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i)
                w[i] = __float_as_uint(__uint_as_float(w[i]) * bars->factor[(o & (N - 1)) + i]);
              tmem_st16(lanes + o, w);
            }
            tmem_wait_st();
          }
        }
        // P^T: rows of keys, 64 heads of 2 bytes, 128-byte swizzle
        uint32_t p0[kOwn / 2], p1[kOwn / 2];
#pragma unroll
        for (int j = 0; j < kOwn / 2; ++j) {
          const float s0 = m[2 * j] == -INFINITY ? 0.f : m[2 * j], s1 = m[2 * j + 1] == -INFINITY ? 0.f : m[2 * j + 1];
          const float a0 = ex2(v[4 * j] - s0), a1 = ex2(v[4 * j + 1] - s1);
          const float b0 = ex2(v[4 * j + 2] - s0), b1 = ex2(v[4 * j + 3] - s1);
          l[2 * j] += a0 + b0;
          l[2 * j + 1] += a1 + b1;
          p0[j] = Elem<E>::pack(a0, a1);
          p1[j] = Elem<E>::pack(b0, b1);
        }
        if (n > 0) mbar_wait_warp(bar(&bars->o_done), (n - 1) & 1u, abort_flag);  // P^T of the last tile is read
#pragma unroll
        for (int j = 0; j < kOwn / 2; ++j) {
          uint8_t* at = p_smem + k0 * 128 + (((side * (kHalf / 8) + j) ^ (k0 & 7)) << 4) + 4 * (lane & 3);
          *reinterpret_cast<uint32_t*>(at) = p0[j];
          *reinterpret_cast<uint32_t*>(at + 8 * 128) = p1[j];
        }
        fence_async_shared();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(&bars->p_full[b]));
      }
      if (!stop) stop = !mbar_wait_warp(bar(&bars->o_done), (n - 1) & 1u, abort_flag);
      stop = any_of(stop, 1, kSoftThreads);
      if (stop) break;
      // row sums over the 64 keys of every strip
#pragma unroll
      for (int i = 0; i < kOwn; ++i) {
        float x = l[i];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (lane < 4) bars->xchg[strip][8 * (i >> 1) + h0 + (i & 1)] = x;
      }
      bar_sync(1, kSoftThreads);
      if (strip == 0 && lane < 4) {
#pragma unroll
        for (int i = 0; i < kOwn; ++i) bars->top[8 * (i >> 1) + h0 + (i & 1)] = m[i];
      }
      bar_sync(1, kSoftThreads);
      const int heads = min(N, a.H - sg.g * N);
      const bool whole = sg.n == sg.tiles;
      const int64_t slot = 2 * (int64_t)blockIdx.x + (segment ? 1 : 0);
      const int64_t first = (int64_t)sg.token * a.H + sg.g * N;  // row of out
      if (tid < N) {
        const float sum = (bars->xchg[0][tid] + bars->xchg[1][tid]) + (bars->xchg[2][tid] + bars->xchg[3][tid]);
        const float top = bars->top[tid];
        bars->factor[tid] = inverse_sum(sum);
        if (!whole) {
          a.pm[slot * N + tid] = top;
          a.pl[slot * N + tid] = sum;
        } else if (a.lse && tid < heads) {
          a.lse[first + tid] = ((top == -INFINITY ? 0.f : top) + log2f(sum)) * kLn2;
        }
      }
      bar_sync(1, kSoftThreads);
      tmem_fence_after();
      // a thread holds 16 heads of one latent index: a store of one head is 128
      // bytes a warp in FP32; for the 16-bit result lane pairs exchange values
      const int odd = lane & 1;
#pragma unroll 2
      for (int o = 16 * side; o < groups * N; o += 32) {
        uint32_t w[16];
        tmem_ld16(lanes + o, w);
        const int hb = o & (N - 1), lim = heads - hb;
        const int64_t col = (int64_t)(o / N) * 128 + strip * 32 + lane;
        tmem_wait_ld();
        if (!whole) {
          float* part = a.po + (slot * N + hb) * a.R + col;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (i < lim) part[i * a.R] = __uint_as_float(w[i]);
        } else {
          uint16_t* dst = a.out + (first + hb + odd) * a.R + (col - odd);
          float f[16];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 x = reinterpret_cast<const float4*>(bars->factor + hb)[i];
            f[4 * i] = x.x;
            f[4 * i + 1] = x.y;
            f[4 * i + 2] = x.z;
            f[4 * i + 3] = x.w;
          }
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const float x0 = __uint_as_float(w[i]) * f[i], x1 = __uint_as_float(w[i + 1]) * f[i + 1];
            const float got = __shfl_xor_sync(0xffffffffu, odd ? x0 : x1, 1);
            if (i + odd < lim)
              *reinterpret_cast<uint32_t*>(dst + i * a.R) = odd ? Elem<E>::pack(got, x1) : Elem<E>::pack(x0, got);
          }
        }
      }
      tmem_fence_before();
      bar_sync(1, kSoftThreads);  // factor, top and xchg are free again
    }
  }
  __syncthreads();
  if (tid == 0 && bars->abort_flag) report(a.status, a.status_host, kStatusWaitTimeout);
  if (warp == 9) {
    tmem_fence_after();
    tmem_free_all<false>(bars->tmem_base);
  }
}

// Joins the partial results of units that several CTAs shared:
//   o = sum_p 2^(m_p - M) o_p / sum_p 2^(m_p - M) l_p,  M the largest m_p,
// and fills what no CTA wrote: tokens that see nothing, and of those outside
// every request the log-sums, with fill_tail the results too.  Bound by latency:
// the plan is one round to L2, all maxima, sums and the first rows a second.

// Where the parts of unit (t, h) are; false when there is nothing to join.
struct Parts {
  int c0, count, row;  // first CTA, parts, row of a slot
  bool late;           // the first part is not its CTA's first segment
  __device__ __forceinline__ int64_t slot(int p, int heads) const {
    return (int64_t)(2 * (c0 + p) + (p == 0 && late ? 1 : 0)) * heads + row;
  }
};
__device__ __forceinline__ bool find_parts(const Args& a, int t, int h, int heads, Parts& q, bool& empty, bool& fill) {
  const int first = a.plan[1 + t], run = a.plan[0], n = first < 0 ? 0 : a.counts[t];
  empty = n == 0;
  fill = first >= 0 || a.fill_tail;
  if (empty) return false;
  const int g = h / heads, f = first + g * n, c1 = (f + n - 1) / run;
  q.c0 = f / run;
  q.count = c1 - q.c0 + 1;
  q.row = h - g * heads;
  q.late = f != q.c0 * run;
  return q.count > 1;
}

// One warp's weights of all parts into `weight`; returns (1 / sum, lse).
constexpr int kPartRounds = kMaxGrid / 32;
__device__ __forceinline__ float2 part_weights(const Args& a, const Parts& q, int heads, float* weight, bool store) {
  const int lane = threadIdx.x & 31;
  float m[kPartRounds], l[kPartRounds], top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int k = 0; k < kPartRounds; ++k) {
    const int p = lane + 32 * k;
    m[k] = p < q.count ? a.pm[q.slot(p, heads)] : -INFINITY;
    l[k] = p < q.count ? a.pl[q.slot(p, heads)] : 0.f;
  }
#pragma unroll
  for (int k = 0; k < kPartRounds; ++k) top = fmaxf(top, m[k]);
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int k = 0; k < kPartRounds; ++k) {
    const int p = lane + 32 * k;
    const float w = ex2(m[k] - base);
    if (store && p < q.count) weight[p] = w;
    sum = fmaf(l[k], w, sum);
  }
  sum = warp_sum(sum);
  return make_float2(inverse_sum(sum), (base + log2f(sum)) * kLn2);
}

__device__ __forceinline__ void add_part(float4& o, float w, const float4& x) {
  o.x = fmaf(w, x.x, o.x);
  o.y = fmaf(w, x.y, o.y);
  o.z = fmaf(w, x.z, o.z);
  o.w = fmaf(w, x.w, o.w);
}
template <typename E>
__device__ __forceinline__ void store_joined(uint16_t* dst, const float4& o, float inv) {
  *reinterpret_cast<uint2*>(dst) = make_uint2(Elem<E>::pack(o.x * inv, o.y * inv), Elem<E>::pack(o.z * inv, o.w * inv));
}

// Few results: a block takes 128 values of one (token, head), and each of its
// WAYS warps every WAYS-th part of them.
template <typename E, int WAYS>
__global__ void __launch_bounds__(32 * WAYS) join_few_kernel(Args a, int heads) {
  __shared__ float weight[kMaxGrid];
  __shared__ float4 part[WAYS][32];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int t = blockIdx.x, h = blockIdx.y, way = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = 4 * (blockIdx.z * 32 + lane);
  const int64_t at = (int64_t)t * a.H + h;
  const bool mine = col < a.R;
  Parts q;
  bool empty, fill;
  if (!find_parts(a, t, h, heads, q, empty, fill)) {
    if (!empty) return;
    if (fill && way == 0 && mine) *reinterpret_cast<uint2*>(a.out + at * a.R + col) = make_uint2(0, 0);
    if (a.lse && threadIdx.x == 0 && blockIdx.z == 0) a.lse[at] = -INFINITY;
    return;
  }
  constexpr int kBatch = 5;
  float4 x[kBatch], o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int k = 0; k < kBatch; ++k) {
    const int p = way + WAYS * k;
    x[k] = mine && p < q.count ? *reinterpret_cast<const float4*>(a.po + q.slot(p, heads) * a.R + col) : o;
  }
  const float2 total = part_weights(a, q, heads, weight, way == 0);
  __syncthreads();
  for (int p0 = way; p0 < q.count; p0 += kBatch * WAYS) {
#pragma unroll
    for (int k = 0; k < kBatch; ++k) {
      const int p = p0 + WAYS * k, next = p + WAYS * kBatch;
      if (p < q.count) add_part(o, weight[p], x[k]);
      if (mine && next < q.count) x[k] = *reinterpret_cast<const float4*>(a.po + q.slot(next, heads) * a.R + col);
    }
  }
  part[way][lane] = o;
  __syncthreads();
  if (way) return;
#pragma unroll
  for (int k = 1; k < WAYS; ++k) add_part(o, 1.f, part[k][lane]);
  if (mine) store_joined<E>(a.out + at * a.R + col, o, total.x);
  if (a.lse && threadIdx.x == 0 && blockIdx.z == 0) a.lse[at] = total.y;
}

// Many results: a warp takes one (token, head), 16 values a lane.
template <typename E>
__global__ void __launch_bounds__(128) join_many_kernel(Args a, int heads) {
  __shared__ float weights[4][kMaxGrid];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, h = blockIdx.y * 4 + warp;
  if (h >= a.H) return;
  const int64_t at = (int64_t)t * a.H + h;
  uint16_t* dst = a.out + at * a.R + 4 * lane;
  Parts q;
  bool empty, fill;
  if (!find_parts(a, t, h, heads, q, empty, fill)) {
    if (!empty) return;
    for (int c = 0; c < a.R && fill; c += 128) *reinterpret_cast<uint2*>(dst + c) = make_uint2(0, 0);
    if (a.lse && lane == 0) a.lse[at] = -INFINITY;
    return;
  }
  const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
  float4 x[2][4], o[4];
  auto load = [&](int p, float4 (&y)[4]) {
    const float* src = a.po + q.slot(p, heads) * a.R + 4 * lane;
#pragma unroll
    for (int c = 0; c < 4; ++c) y[c] = 128 * c < a.R ? *reinterpret_cast<const float4*>(src + 128 * c) : zero;
  };
  load(0, x[0]);
  load(1, x[1]);
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] = zero;
  const float2 total = part_weights(a, q, heads, weights[warp], true);
  __syncwarp();
  for (int p0 = 0; p0 < q.count; p0 += 2) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int p = p0 + k;
      if (p < q.count) {
        const float w = weights[warp][p];
#pragma unroll
        for (int c = 0; c < 4; ++c) add_part(o[c], w, x[k][c]);
        if (p + 2 < q.count) load(p + 2, x[k]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (128 * c < a.R) store_joined<E>(dst + 128 * c, o[c], total.x);
  if (a.lse && lane == 0) a.lse[at] = total.y;
}

int grid_size() { return std::min(sm_count(), kMaxGrid); }
size_t plan_bytes(int64_t tokens) { return align_up((size_t)(2 * tokens + 1) * 4, 256); }
size_t part_bytes(int64_t latent_dim) {
  return 2 * (size_t)grid_size() * kMaxHeads * ((size_t)latent_dim + 2) * sizeof(float);
}

bool stride_ok(int64_t s, int64_t count) {
  return s % 8 == 0 && s < (int64_t)1 << 38 && (count > 1 ? s > 0 : s >= 0);
}

int make_map(CUtensorMap* map, const void* base, bool bf16, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
             const cuuint32_t* box) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("glm53_latent_absorbed: cuTensorMapEncodeTiled is unavailable");
    return GLM53_ERR_CUDA;
  }
  const cuuint32_t step[4] = {1, 1, 1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, rank, const_cast<void*>(base),
         dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("glm53_latent_absorbed: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return GLM53_ERR_CUDA;
  }
  return GLM53_OK;
}

template <typename E, int N>
int launch(const CUtensorMap& ql, const CUtensorMap& qr, const CUtensorMap& kv0, const CUtensorMap& kv1, const Args& a,
           cudaStream_t st) {
  int rc = ensure_max_smem((const void*)absorbed_kernel<E, N>, kSmemBytes);
  if (rc) return rc;
  absorbed_kernel<E, N><<<grid_size(), kThreads, kSmemBytes, st>>>(ql, qr, kv0, kv1, a);
  if ((rc = check_launch("absorbed_kernel"))) return rc;
  // How many warps share a result: many while there are few results, which then
  // have many parts.  1,000 / 12,000 rows each, whole calls, us by warps:
  //   results         16           8            4            2            1
  //   1 x 64      15.5 / 20.8  15.5 / 22.1  15.9 / 25.4  16.6 / 28.9  20.3 / 70.3
  //   2 x 64      18.6 / 29.3  15.5 / 25.3  16.1 / 27.8  16.8 / 31.6  20.5 / 58.4
  //   4 x 64      24.0 / 38.3  18.4 / 32.1  16.4 / 30.5  17.5 / 33.0  23.8 / 47.7
  //   8 x 64      35.4 / 61.6  23.9 / 50.0  18.8 / 44.7  17.9 / 45.0  25.6 / 52.1
  //   16 x 64     52.6 / 96.2  34.6 / 77.5  24.7 / 67.5  20.5 / 62.6  21.9 / 65.9
  //   24 x 64     75.2 / 132   48.7 / 104   35.3 / 90.1  29.0 / 83.8  26.5 / 82.0
  //   16 x 16     21.9 / 57.9  17.3 / 52.7  15.5 / 51.5  15.7 / 50.8  18.4 / 56.1
  //   4 x 128     35.2 / 57.2  23.9 / 46.0  18.8 / 40.6  17.9 / 39.9  25.9 / 49.2
  // Two warps no longer pay where a unit has two or three parts: 64 x 16 27.4 / 148
  // with two, 25.8 / 146 with one.
  const int64_t results = a.T * a.H;
  const dim3 pieces((unsigned)a.T, (unsigned)a.H, (unsigned)(a.R / 128));
  if (results <= 64)
    launch_programmatic(join_few_kernel<E, 16>, pieces, dim3(512), 0, st, a, N);
  else if (results <= 128)
    launch_programmatic(join_few_kernel<E, 8>, pieces, dim3(256), 0, st, a, N);
  else if (results <= 384)
    launch_programmatic(join_few_kernel<E, 4>, pieces, dim3(128), 0, st, a, N);
  else if (results <= 1024 && 3 * a.T * a.G <= grid_size())
    launch_programmatic(join_few_kernel<E, 2>, pieces, dim3(64), 0, st, a, N);
  else
    launch_programmatic(join_many_kernel<E>, dim3((unsigned)a.T, (unsigned)((a.H + 3) / 4)), dim3(128), 0, st, a, N);
  return check_launch("join_kernel");
}

// Heads a unit: the fewest of 16, 32 and 64 that hold all heads, else 64.  A
// unit of 16 heads pays a third of the MMA cycles of one of 64.
int unit_heads(int64_t heads) { return heads <= 16 ? 16 : heads <= 32 ? 32 : 64; }

}  // namespace
}  // namespace latent
}  // namespace glm53

using namespace glm53;
using namespace glm53::latent;

extern "C" size_t glm53_latent_absorbed_workspace_bytes(int64_t tokens, int64_t heads, int64_t latent_dim) {
  if (tokens < 0 || heads < 1 || latent_dim < 1 || latent_dim > 512) return 0;
  return plan_bytes(tokens) + part_bytes(latent_dim);
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
  if (!std::isfinite(scale) || !stride_ok(ql_stride_t, tokens) || !stride_ok(ql_stride_h, heads) ||
      (rope_dim && (!stride_ok(qr_stride_t, tokens) || !stride_ok(qr_stride_h, heads)))) {
    set_last_error("%s: the scale must be finite and strides positive multiples of 8", fn);
    return GLM53_ERR_INVALID;
  }
  if (!query_starts && tokens != requests) {
    set_last_error("%s: without query_starts there is one token a request (%lld tokens, %lld requests)", fn,
                   (long long)tokens, (long long)requests);
    return GLM53_ERR_INVALID;
  }
  if ((double)tokens * (double)((heads + 63) / 64) * (double)((table_width * page_size + 63) / 64) >= 2147483648.0) {
    set_last_error("%s: %lld tokens over a table of %lld rows: 2^31 tiles of 64 rows at most", fn, (long long)tokens,
                   (long long)(table_width * page_size));
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
  if ((uintptr_t)workspace & 255) {
    set_last_error("%s: the workspace must be 256-byte aligned", fn);
    return GLM53_ERR_INVALID;
  }
  const bool bf16 = dtype == GLM53_DTYPE_BF16;
  CUtensorMap ql, qr, kv0, kv1;
  const cuuint64_t ql_dims[3] = {(cuuint64_t)latent_dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  const cuuint64_t ql_strides[2] = {(cuuint64_t)(ql_stride_h ? ql_stride_h : 8) * 2,
                                    (cuuint64_t)(ql_stride_t ? ql_stride_t : 8) * 2};
  const int unit = unit_heads(heads);
  const cuuint32_t q_box[3] = {64, (cuuint32_t)unit, 1};
  int rc = make_map(&ql, q_latent, bf16, 3, ql_dims, ql_strides, q_box);
  if (rc) return rc;
  qr = kv0 = kv1 = ql;  // maps that no load reads (no rotary part, no pages, no second half)
  if (rope_dim) {
    const cuuint64_t dims[3] = {(cuuint64_t)rope_dim, (cuuint64_t)heads, (cuuint64_t)tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)(qr_stride_h ? qr_stride_h : 8) * 2,
                                   (cuuint64_t)(qr_stride_t ? qr_stride_t : 8) * 2};
    if ((rc = make_map(&qr, q_rope, bf16, 3, dims, strides, q_box))) return rc;
  }
  // rows of a TMA box: the largest divisor of 64 that divides a page
  int box = 64;
  while (page_size % box) box >>= 1;
  // the two halves of a row, in 64-value chunks: whole 128-value groups first
  const int groups = (int)latent_dim / 128;
  const int half[2] = {2 * ((groups + 1) / 2), 2 * (groups / 2) + (rope_dim ? 1 : 0)};
  if (pages) {
    const cuuint64_t width = 2 * (cuuint64_t)(latent_dim + rope_dim);  // bytes
    const cuuint64_t dims[4] = {64, 8, (cuuint64_t)(latent_dim + rope_dim) / 64, (cuuint64_t)(pages * page_size / 8)};
    const cuuint64_t strides[3] = {width, 128, 8 * width};
    cuuint32_t kv_box[4] = {64, 8, (cuuint32_t)half[0], (cuuint32_t)box / 8};
    if ((rc = make_map(&kv0, cache, bf16, 4, dims, strides, kv_box))) return rc;
    kv_box[2] = (cuuint32_t)half[1];
    if (half[1] && (rc = make_map(&kv1, cache, bf16, 4, dims, strides, kv_box))) return rc;
  }
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const int64_t slots = 2 * (int64_t)grid_size() * kMaxHeads;
  Args a{};
  a.T = tokens;
  a.H = (int)heads;
  a.R = (int)latent_dim;
  a.r = (int)rope_dim;
  a.G = (int)((heads + unit - 1) / unit);
  a.cache = (const uint16_t*)cache;
  a.pages = pages;
  a.page = (int)page_size;
  a.box = box;
  a.table = block_table;
  a.table_stride = table_stride;
  a.table_width = pages ? table_width : 0;  // no page can be named
  a.lens = seq_lens;
  a.B = (int)requests;
  a.starts = query_starts;
  a.c = scale * kLog2e;
  a.out = (uint16_t*)out;
  a.lse = lse;
  a.fill_tail = fill_tail;
  a.status = status;
  a.status_host = status_host;
  a.half[0] = half[0];
  a.half[1] = half[1];
  a.plan = reinterpret_cast<int32_t*>(ws);
  a.counts = a.plan + tokens + 1;
  a.po = reinterpret_cast<float*>(ws + plan_bytes(tokens));
  a.pm = a.po + slots * latent_dim;
  a.pl = a.pm + slots;
  const cudaStream_t st = (cudaStream_t)stream;
  if (bf16)
    return unit == 16   ? launch<__nv_bfloat16, 16>(ql, qr, kv0, kv1, a, st)
           : unit == 32 ? launch<__nv_bfloat16, 32>(ql, qr, kv0, kv1, a, st)
                        : launch<__nv_bfloat16, 64>(ql, qr, kv0, kv1, a, st);
  return unit == 16   ? launch<__half, 16>(ql, qr, kv0, kv1, a, st)
         : unit == 32 ? launch<__half, 32>(ql, qr, kv0, kv1, a, st)
                      : launch<__half, 64>(ql, qr, kv0, kv1, a, st);
}
