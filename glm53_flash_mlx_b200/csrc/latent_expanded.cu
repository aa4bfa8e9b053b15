// Latent attention, expanded form (prefill): softmax(scale q k^T) v over a
// ragged batch, with keys [k_nope_h | k_rope] whose rotary part all heads share
// and causal rows that see the keys up to their own position.
//
// One CTA takes 128 queries of one head and walks their keys 128 at a time:
//   S = Q K^T   tcgen05 M128 N128, operands in shared memory, FP32 in TMEM;
//   P = 2^(S c - m), c = scale log2(e), rounded to the element type into the
//               columns of S (the second product's A operand comes from TMEM);
//   O += P V    tcgen05 M128, N up to 128 a 128-value half, FP32 in TMEM.
// m is a running maximum per row that is replaced only when a score exceeds it
// by more than 2^8 (O in TMEM is rescaled then, rarely after the first tile);
// the row sums use the unrounded weights in FP32.
//
// Bound by the tensor cores: 2 x 128 x 128 x (dqk + dv) FLOPs a tile, 2,048
// MMA cycles at 256 + 256 against 1,024 cycles of exponentials (16 a cycle and
// SM).  So S is double buffered and the MMA warp issues S of tile i + 1 before
// P V of tile i: the softmax of one tile runs under the products of another.
// TMEM is full: O 256 columns, two S tiles of 128.  Shared memory too: Q
// 64 KB, and one ring of five 32 KB slots that K and V halves (128 keys x 128
// values) share in the order the MMAs take them.
//
// One CTA alone moves 128 KB into shared memory a tile and its MMAs read
// 192 KB there: 2,560 cycles at 128 bytes each, more than the MMAs need.  For
// long requests two CTAs work as a pair (cta_group::2, M = 256): each holds its
// 128 queries, half the keys of a K tile and half the values of a V tile, and
// rank 0 issues for both (2,048 queries over 8,192 keys, 64 heads of 256 + 256:
// 856 us alone, 715 to 771 as pairs by the clock that the power limit leaves,
// 1,250 to 1,345 TFLOP/s).  For short ones a CTA an SM walks
// the units instead, so that the set-up of one runs under the results of the
// last.  Both rules are at the launch.
//
// Roles: warps 0-7 softmax (two threads a row, 64 keys each) and epilogue,
// warp 8 TMA, warp 9 MMA, warps 10 and 11 clean values (below).  Every mbarrier
// wait is bounded; a CTA that gives up sets GLM53_STATUS_WAIT_TIMEOUT, waits for
// its copies and MMAs, frees its TMEM and exits.
//
// Masked places must not enter, whatever they hold.  Masked scores are
// replaced before the maximum.  A masked weight is 0, but 0 x NaN is not, so on
// the tiles that the mask cuts two warps clear value rows behind the request's
// last key and values that are not finite, under the softmax and before the
// product reads them; the epilogue then adds the latter to the rows that do
// see them.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "gemv_tile.cuh"
#include "latent.cuh"
#include "tcgen05.cuh"

namespace glm53 {
namespace latent {
namespace {

using namespace tc;

constexpr int kTile = 128;                 // queries a CTA, keys a step
constexpr int kChunkBytes = kTile * 128;   // 128 rows of 64 values
constexpr int kSlotBytes = 2 * kChunkBytes;
constexpr int kSlots = 5;
constexpr int kSoftWarps = 8;
constexpr int kSoftThreads = kSoftWarps * 32;
constexpr int kCleanWarps = 2;
constexpr int kThreads = kSoftThreads + 128;
constexpr int kFillCtas = 512;             // CTAs that fill rows outside every request, at most
constexpr int kOCol = 0;     // TMEM: O at 0..255, S tiles at 256 and 384
constexpr int kSCol = 256;

struct Args {
  int64_t Tq, Tk;
  int H, dn, dr, dv;
  const int32_t *q_starts, *k_starts;
  int B;
  float c;       // |scale| log2(e), not 0: a masked score is -inf and stays that
  int negative;  // the scale's sign
  int causal;
  const uint16_t* v;
  int64_t v_t, v_h;
  uint16_t* out;
  float* lse;
  int fill_tail;
  int persistent;  // CTAs walk the units; else one a CTA (pair), units in x, heads in y
  uint32_t *status, *status_host;
};

// One head's queries [first, first + rows of a unit) of a request, and what
// they see.  A unit is 128 queries, 256 for a pair of CTAs.
struct Unit {
  int q0, nq, k0, nk;
  int first, head;

  // keys that query j of the request sees
  __device__ __forceinline__ int seen(const Args& a, int j) const {
    return a.causal ? max(0, (int)min((int64_t)nk, (int64_t)nk - nq + j + 1)) : nk;
  }
};

// Where a search for a query tile stands: at request `r0`, whose first tile is
// `base`; `top`, once a start out of order was met, is the
// largest valid start before it (below), else -1.
struct Walk {
  int r0 = 0, base = 0, top = -1;
};

struct __align__(8) Bars {
  uint64_t q_full, q_empty, full[kSlots], empty[kSlots], cut_full[4], s_full[2], p_full[2], o_done[2], drain;
  uint32_t tmem_base;
  int abort_flag;
  Unit unit;      // the softmax warps' unit
  Walk walk[kSoftWarps];  // where each softmax warp's search for a unit stands (MANY)
  int poison[2];  // by unit parity: the unit (from 1) with values that are not finite in a masked tile
};

// alignment slack, Q, ring, barriers, two floats a row
constexpr size_t kSmemBytes = 1024 + 4 * (size_t)kChunkBytes + kSlots * (size_t)kSlotBytes + 1024 + 2 * kTile * 4;
static_assert(sizeof(Bars) <= 1024, "barriers share one KB");
static_assert(kSmemBytes <= 232448, "227 KB a CTA");

// A request's rows, checked: invalid query bounds count as no queries, invalid
// key bounds as no keys.
struct Bounds {
  int64_t q0, nq, k0, nk;
  bool bad, ordered;  // ordered: the query bounds are valid
};
__device__ __forceinline__ Bounds bounds_of(const Args& a, int i) {
  Bounds b;
  b.q0 = a.q_starts[i];
  b.nq = (int64_t)a.q_starts[i + 1] - b.q0;
  b.k0 = a.k_starts[i];
  b.nk = (int64_t)a.k_starts[i + 1] - b.k0;
  b.ordered = b.q0 >= 0 && b.nq >= 0 && b.q0 + b.nq <= a.Tq;
  b.bad = !b.ordered;
  if (!b.ordered) b.nq = 0;
  if (b.k0 < 0 || b.nk < 0 || b.k0 + b.nk > a.Tk) {
    b.bad = true;
    b.k0 = b.nk = 0;
  }
  return b;
}

// Where query starts descend or leave the rows, the requests that keep their
// queries are those with bounds in order that begin at or behind every valid
// start before them: no two of them share a row.
__device__ __forceinline__ bool valid_start(const Args& a, int64_t v) { return v >= 0 && v <= a.Tq; }

// By a converged warp, 32 requests a step, `b` those of this lane (all 0 behind
// the last) and `top` the largest valid start before the step (the step's first
// start is as large where all before it is in order): whether this lane's request
// keeps its queries.
__device__ __forceinline__ bool keeps_queries(const Args& a, const Bounds& b, int& top) {
  const int lane = threadIdx.x & 31;
  int most = valid_start(a, b.q0) ? (int)b.q0 : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, most, o);
    if (lane >= o) most = max(most, y);
  }
  most = max(most, top);
  top = __shfl_sync(0xffffffffu, most, 31);
  return b.ordered && b.q0 >= most;
}

// Query tile `x` over all requests (in order; a request's last tile, which sees
// the most keys, first); by a converged warp.  False when there are fewer.  The
// next search goes on from `w` and must not look for an earlier tile.
template <int ROWS>
__device__ __forceinline__ bool find_tile(const Args& a, int x, Unit& u, Walk& w) {
  const int lane = threadIdx.x & 31;
  for (; w.r0 < a.B; w.r0 += 32) {
    Bounds b{};
    int n = 0;
    const bool real = w.r0 + lane < a.B;
    if (real) {
      b = bounds_of(a, w.r0 + lane);
      n = (int)((b.nq + ROWS - 1) / ROWS);
    }
    int top = w.top;
    if (top >= 0 || __any_sync(0xffffffffu, real && !b.ordered)) {
      top = max(top, 0);
      if (!keeps_queries(a, b, top)) n = 0;
    }
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    const int lo = w.base + s - n;
    const uint32_t mine = __ballot_sync(0xffffffffu, x >= lo && x < lo + n);
    if (mine) {
      const int src = __ffs(mine) - 1;
      u.q0 = __shfl_sync(0xffffffffu, (int)b.q0, src);
      u.nq = __shfl_sync(0xffffffffu, (int)b.nq, src);
      u.k0 = __shfl_sync(0xffffffffu, (int)b.k0, src);
      u.nk = __shfl_sync(0xffffffffu, (int)b.nk, src);
      u.first = __shfl_sync(0xffffffffu, (n - 1 - (x - lo)) * ROWS, src);
      return true;
    }
    w.base += __shfl_sync(0xffffffffu, s, 31);
    w.top = top;
  }
  return false;
}

// Infinities and NaN: the exponent bits are all ones.
template <typename E>
constexpr uint32_t kExponent = std::is_same<E, __half>::value ? 0x7C00u : 0x7F80u;
template <typename E>
__device__ __forceinline__ bool not_finite(uint32_t half) {
  return (half & kExponent<E>) == kExponent<E>;
}
// Bit 15 (31) is set when the lower (upper) half is not finite: adding the
// exponent's lowest bit to an exponent of ones carries into it.
template <typename E>
__device__ __forceinline__ uint32_t not_finite_bits(uint32_t w) {
  constexpr uint32_t both = kExponent<E> * 0x10001u, low = (kExponent<E> & (0u - kExponent<E>)) * 0x10001u;
  return ((w & both) + low) & 0x80008000u;
}

// Clears row `row` of a 64-value chunk of one key tile's values where it lies
// behind the last valid key, and its values that are not finite elsewhere;
// true when there were any of the latter.
template <typename E>
__device__ __forceinline__ bool clean_row(uint8_t* chunk, int row, int valid) {
  uint4* line = reinterpret_cast<uint4*>(chunk + row * 128);
  if (row >= valid) {
#pragma unroll
    for (int p = 0; p < 8; ++p) line[p ^ (row & 7)] = make_uint4(0, 0, 0, 0);
    return false;
  }
  uint4 w[8];
  uint32_t any = 0;
#pragma unroll
  for (int p = 0; p < 8; ++p) w[p] = line[p ^ (row & 7)];
#pragma unroll
  for (int p = 0; p < 8; ++p)
    any |= not_finite_bits<E>(w[p].x) | not_finite_bits<E>(w[p].y) | not_finite_bits<E>(w[p].z) |
           not_finite_bits<E>(w[p].w);
  if (!any) return false;
  auto clean = [](uint32_t x) {
    return (not_finite<E>(x) ? 0u : x & 0xFFFFu) | (not_finite<E>(x >> 16) ? 0u : x & 0xFFFF0000u);
  };
#pragma unroll
  for (int p = 0; p < 8; ++p)
    line[p ^ (row & 7)] = make_uint4(clean(w[p].x), clean(w[p].y), clean(w[p].z), clean(w[p].w));
  return true;
}

// Lane 4 k + e of a quad holds p[i]; afterwards p[i] is what lane 4 k + i held
// in p[e].
__device__ __forceinline__ uint4 shfl_xor4(uint4 v, int mask) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, mask), __shfl_xor_sync(0xffffffffu, v.y, mask),
                    __shfl_xor_sync(0xffffffffu, v.z, mask), __shfl_xor_sync(0xffffffffu, v.w, mask));
}
__device__ __forceinline__ void quad_transpose(uint4 (&p)[4], int lane) {
  const bool odd = lane & 1, high = lane & 2;
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const uint4 got = shfl_xor4(odd ? p[i] : p[i + 1], 1);
    p[i] = odd ? got : p[i];
    p[i + 1] = odd ? p[i + 1] : got;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const uint4 got = shfl_xor4(high ? p[i] : p[i + 2], 2);
    p[i] = high ? got : p[i];
    p[i + 2] = high ? p[i + 2] : got;
  }
}

template <typename E, bool PAIR, bool MANY>
__global__ void __launch_bounds__(kThreads, 1)
    expanded_kernel(const __grid_constant__ CUtensorMap qn_map, const __grid_constant__ CUtensorMap qr_map,
                    const __grid_constant__ CUtensorMap kn_map, const __grid_constant__ CUtensorMap kr_map,
                    const __grid_constant__ CUtensorMap v_map, Args a) {
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* q_smem = smem;
  uint8_t* ring = smem + 4 * kChunkBytes;
  Bars* bars = reinterpret_cast<Bars*>(ring + kSlots * kSlotBytes);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  constexpr int kCtas = PAIR ? 2 : 1, kUnit = kCtas * kTile;  // queries a CTA or pair takes
  const int rank = PAIR ? (int)cluster_rank() : 0;
  auto bar = [&](uint64_t* p) { return smem_addr(p); };

  if (tid == 0) {
    bars->abort_flag = 0;
    bars->poison[0] = bars->poison[1] = 0;
    mbar_init(bar(&bars->q_full), 1);
    mbar_init(bar(&bars->q_empty), 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar(&bars->full[s]), 1);
      mbar_init(bar(&bars->empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(&bars->cut_full[s]), 1);
      mbar_init(bar(&bars->cut_full[s + 2]), 1);
      mbar_init(bar(&bars->s_full[s]), 1);
      mbar_init(bar(&bars->p_full[s]), kCtas * (kSoftWarps + kCleanWarps));
      mbar_init(bar(&bars->o_done[s]), 1);
    }
    mbar_init(bar(&bars->drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    tmem_alloc_all<PAIR>(smem_addr(&bars->tmem_base));
  } else if (warp == 8 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qn_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qr_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kn_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kr_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
  }
  __syncwarp();

  // The CTA's units in order, by a converged warp: every role walks them itself.
  // Walking CTAs take all heads of one query tile before the next tile, so that
  // a round of the grid holds units of like length.
  auto next_unit = [&](int i, Unit& u, Walk& w) {
    if (a.persistent) {
      const int64_t at = blockIdx.x + (int64_t)i * gridDim.x;
      const int64_t x = at / a.H;
      u.head = (int)(at - x * a.H);
      return x < INT32_MAX && find_tile<kUnit>(a, (int)x, u, w);
    }
    u.head = blockIdx.y;
    return i == 0 && find_tile<kUnit>(a, blockIdx.x / kCtas, u, w);
  };
  tmem_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // the other CTA's barriers are set up
  tmem_fence_after();

  // A pair holds half the keys of a K tile (64 rows, four chunks a slot) and
  // half the values of a V tile in each CTA.
  constexpr int kKeyRows = kTile / kCtas, kKeyChunk = kKeyRows * 128, kKeyChunks = kSlotBytes / kKeyChunk;
  const int nch = (a.dn + a.dr) / 64, kslots = (nch + kKeyChunks - 1) / kKeyChunks;
  const int vch = a.dv / 64 / kCtas, vslots = (vch + 1) / 2;
  // key tiles of a unit, and the first of them that the mask cuts for some row
  auto tiles_of = [&](const Unit& u) {
    return (u.seen(a, (int)min((int64_t)u.nq, (int64_t)u.first + kUnit) - 1) + kTile - 1) / kTile;
  };
  auto cut_of = [&](const Unit& u) { return u.seen(a, u.first) / kTile; };

  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's
  volatile int* abort_flag = &bars->abort_flag;

  auto p_arrive = [&](uint32_t g) {
    if constexpr (PAIR)
      mbar_arrive_at_relaxed(bar(&bars->p_full[g & 1]), 0);
    else
      mbar_arrive(bar(&bars->p_full[g & 1]));
  };
  // Running over all units: g key tiles, seq ring slots, cut tiles that the mask
  // cuts.  Tile g's S, P and product use the barriers g & 1, phase (g >> 1) & 1.
  uint32_t g = 0;

  if (warp == 8) {
    // ---------------- TMA ----------------
    // full[s] counts the bytes of both CTAs of a pair, at rank 0.  The values of
    // a tile that the mask cuts are counted at cut_full of the CTA that holds
    // (and cleans) them; the product learns of them through p_full.  A pair's ring
    // can hold three such tiles before the first has landed (one slot a tile, no
    // K behind the last), and a barrier takes one tile at a time: four barriers.
    uint32_t seq = 0, queries = 0;
    int cut = 0;
    bool ok = true;
    Unit u;
    Walk w;
    for (int i = 0; next_unit(i, u, w); ++i) {
      const int tiles = tiles_of(u), cut0 = cut_of(u);
      if (lane == 0 && tiles > 0 && ok) {
        auto load = [&](uint32_t dst, const CUtensorMap* map, int x, int z, uint64_t* p) {
          if constexpr (PAIR)
            tma_load_3d_at(dst, map, x, u.head, z, bar(p), 0);
          else
            tma_load_3d(dst, map, x, u.head, z, bar(p));
        };
        if (queries) ok = mbar_wait_fast(bar(&bars->q_empty), (queries - 1) & 1u, abort_flag);
        if (ok) {
          ++queries;
          if (rank == 0) mbar_expect_tx(bar(&bars->q_full), kCtas * nch * kChunkBytes);
          for (int c = 0; c < nch; ++c) {
            const bool rope = c * 64 >= a.dn;
            load(smem_addr(q_smem + c * kChunkBytes), rope ? &qr_map : &qn_map, rope ? 0 : c * 64,
                 u.q0 + u.first + rank * kTile, &bars->q_full);
          }
        }
        auto slot = [&](bool value, int tile, int part) {
          const uint32_t s = seq % kSlots;
          if (seq >= kSlots) ok = mbar_wait_fast(bar(&bars->empty[s]), (seq / kSlots - 1) & 1u, abort_flag);
          if (!ok) return;
          const int per = value ? 2 : kKeyChunks, bytes = value ? kChunkBytes : kKeyChunk;
          const int n = min(per, (value ? vch : nch) - per * part);
          const bool masked = value && tile >= cut0;
          if (masked && part == 0) ++cut;
          uint64_t* local = &bars->cut_full[(cut - 1) & 3];
          if (masked) {
            if (part == 0) mbar_expect_tx(bar(local), vch * kChunkBytes);
            if (rank == 0) mbar_arrive(bar(&bars->full[s]));
          } else if (rank == 0) {
            mbar_expect_tx(bar(&bars->full[s]), kCtas * n * bytes);
          }
          for (int c = 0; c < n; ++c) {
            const uint32_t dst = smem_addr(ring + s * kSlotBytes + c * bytes);
            const int x = (per * part + c) * 64, z = u.k0 + tile * kTile;
            if (masked)
              tma_load_3d(dst, &v_map, rank * vch * 64 + x, u.head, z, bar(local));
            else if (value)
              load(dst, &v_map, rank * vch * 64 + x, z, &bars->full[s]);
            else if (x < a.dn)
              load(dst, &kn_map, x, z + rank * kKeyRows, &bars->full[s]);
            else if constexpr (PAIR)
              tma_load_2d_at(dst, &kr_map, 0, z + rank * kKeyRows, bar(&bars->full[s]), 0);
            else
              tma_load_2d(dst, &kr_map, 0, z, bar(&bars->full[s]));
          }
          ++seq;
        };
        for (int t = 0; t <= tiles && ok; ++t) {
          for (int p = 0; p < kslots && ok && t < tiles; ++p) slot(false, t, p);
          for (int p = 0; p < vslots && ok && t > 0; ++p) slot(true, t - 1, p);
        }
      }
      __syncwarp();
    }
    if (!ok) {
      // copies still in flight write this CTA's (this pair's) shared memory: wait
      // for them; a pair leaves together
      volatile int never = 0;
      for (uint32_t k = seq > kSlots ? seq - kSlots : 0; k < seq && rank == 0; ++k) {
        never = 0;
        mbar_wait(bar(&bars->full[k % kSlots]), (k / kSlots) & 1u, &never);
      }
      never = 0;
      if (rank == 0 && queries) mbar_wait(bar(&bars->q_full), (queries - 1) & 1u, &never);
      for (int k = max(0, cut - 4); k < cut; ++k) {
        never = 0;
        mbar_wait(bar(&bars->cut_full[k & 3]), (k >> 2) & 1u, &never);
      }
    }
    __syncwarp();
    if (blockIdx.y == 0)
      for (int64_t i = (int64_t)blockIdx.x * 32 + lane; i < a.B; i += (int64_t)gridDim.x * 32)
        if (bounds_of(a, (int)i).bad) report(a.status, a.status_host, kStatusBadGeometry);
  } else if (warp == 9) {
    // ---------------- MMA ----------------
    // All lanes walk the loops, so that descriptors stay in uniform registers;
    // one elected lane waits and issues the unrolled MMAs of a slot.
    constexpr bool bf16 = std::is_same<E, __nv_bfloat16>::value;
    constexpr uint32_t id_s = make_idesc_f16(kUnit, kTile, bf16, false, false);
    const bool leader = elect_one() && rank == 0;
    uint32_t seq = 0, queries = 0;
    bool ok = true;
    const uint64_t qd = make_sw128_desc(smem_addr(q_smem));
    const uint64_t kd0 = make_sw128_desc(smem_addr(ring)), vd0 = make_sw128_mn_desc(smem_addr(ring), kChunkBytes);
    auto commit = [&](uint64_t* p) {
      if constexpr (PAIR)
        mma_commit2(bar(p));
      else
        mma_commit(bar(p));
    };
    auto landed = [&](uint32_t s, uint32_t phase) {
      ok = ok && mbar_wait_fast(bar(&bars->full[s]), phase, abort_flag);
      tmem_fence_after();
      return ok;
    };
    Unit u;
    Walk w;
    for (int i = 0; next_unit(i, u, w); ++i) {
      const int tiles = tiles_of(u);
      if (tiles == 0) continue;
      if (leader) ok = ok && mbar_wait_fast(bar(&bars->q_full), queries & 1u, abort_flag);
      ++queries;
      for (int t = 0; t <= tiles; ++t) {
        if (t < tiles) {
          const uint32_t d = kSCol + ((g + t) & 1) * kTile;
          for (int p = 0; p < kslots; ++p, ++seq) {
            const uint32_t s = seq % kSlots, phase = (seq / kSlots) & 1u;
            const uint64_t ad = qd + (uint64_t)(p * (kKeyChunks * kChunkBytes >> 4));
            const uint64_t kd = kd0 + (uint64_t)(s * (kSlotBytes >> 4));
            const int n = min(kKeyChunks, nch - kKeyChunks * p);
            if (leader && landed(s, phase)) {
#pragma unroll
              for (int c = 0; c < kKeyChunks; ++c) {
                if (c < n) {
#pragma unroll
                  for (int k = 0; k < 4; ++k) {
                    const uint64_t x = ad + (c * kChunkBytes >> 4) + 2 * k, y = kd + (c * kKeyChunk >> 4) + 2 * k;
                    if constexpr (PAIR)
                      mma_f16_ss2(d, x, y, id_s, (p | c | k) != 0);
                    else
                      mma_f16_ss(d, x, y, id_s, (p | c | k) != 0);
                  }
                }
              }
              commit(&bars->empty[s]);
            }
          }
          if (leader && ok) {
            commit(&bars->s_full[(g + t) & 1]);
            if (t + 1 == tiles) commit(&bars->q_empty);
          }
        }
        if (t > 0) {
          const uint32_t v = g + t - 1;  // the tile whose values are multiplied
          const uint32_t pa = kSCol + (v & 1) * kTile;
          const int steps = (min(kTile, u.nk - (t - 1) * kTile) + 15) >> 4;
          const bool more = t > 1;  // adds to what is there
          if (leader) {
            if constexpr (PAIR)
              ok = ok && mbar_wait_peer(bar(&bars->p_full[v & 1]), (v >> 1) & 1u, abort_flag);
            else
              ok = ok && mbar_wait_fast(bar(&bars->p_full[v & 1]), (v >> 1) & 1u, abort_flag);
          }
          for (int p = 0; p < vslots; ++p, ++seq) {
            const uint32_t s = seq % kSlots, phase = (seq / kSlots) & 1u;
            // a pair's slot holds half of N = 256 or 128; a CTA's all of N = 128 or 64
            const bool two = 2 * p + 1 < vch;
            const uint32_t id_o = two ? make_idesc_f16(kUnit, kUnit, bf16, false, true)
                                      : make_idesc_f16(kUnit, kUnit / 2, bf16, false, true);
            const uint64_t vd = vd0 + (uint64_t)(s * (kSlotBytes >> 4));
            const uint32_t o = kOCol + p * 128;
            if (leader && landed(s, phase)) {
              auto step = [&](int k) {
                if constexpr (PAIR)
                  mma_f16_ts2(o, pa + 8 * k, vd + 128 * k, id_o, more || k);
                else
                  mma_f16_ts(o, pa + 8 * k, vd + 128 * k, id_o, more || k);
              };
              if (steps == 8) {
#pragma unroll
                for (int k = 0; k < 8; ++k) step(k);
              } else {
                for (int k = 0; k < steps; ++k) step(k);
              }
              commit(&bars->empty[s]);
            }
          }
          if (leader && ok) commit(&bars->o_done[v & 1]);
        }
      }
      g += tiles;
    }
    __syncwarp();
    // no MMA is in flight when TMEM is freed.  The lane that issued waits alone:
    // a lane that spins must not keep its warp from one with work.
    if (leader) {
      volatile int never = 0;
      commit(&bars->drain);
      if (!mbar_wait(bar(&bars->drain), 0, &never)) *abort_flag = 1;
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ---------------- values of the tiles that the mask cuts ----------------
    bool ok = true;
    uint32_t seq = 0;
    int cut = 0, units = 0;
    Unit u;
    Walk w;
    for (int i = 0; next_unit(i, u, w); ++i) {
      const int tiles = tiles_of(u), cut0 = cut_of(u);
      if (tiles == 0) continue;
      ++units;
      for (int t = 0; t < tiles; ++t) {
        const uint32_t v = g + t;
        ok = ok && __all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->s_full[v & 1]), (v >> 1) & 1u, abort_flag));
        if (t >= cut0 && ok) {
          // its values lie in the ring where the producer put them
          const uint32_t s0 = seq + kslots + t * (kslots + vslots) + (t + 1 < tiles ? kslots : 0);
          ok = __all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->cut_full[cut & 3]), (cut >> 2) & 1u, abort_flag));
          ++cut;
          const int valid = min(kTile, u.nk - t * kTile), end = (valid + 15) & ~15;  // the product stops at `end`
          bool found = false;
          for (int c = 0; c < vch && ok; ++c) {
            const uint32_t s = (s0 + (c >> 1)) % kSlots;
            for (int row = tid - 320; row < end && ok; row += 64)
              found |= clean_row<E>(ring + s * kSlotBytes + (c & 1) * kChunkBytes, row, valid);
          }
          if (found) {
            bars->poison[units & 1] = units;
            // the other CTA's rows meet these values too
            if constexpr (PAIR) store_at(smem_addr(&bars->poison[units & 1]), rank ^ 1, units);
          }
          fence_async_shared();
          __syncwarp();
          if (lane == 0) {
            if constexpr (PAIR)
              mbar_arrive_at(bar(&bars->p_full[v & 1]), 0);
            else
              p_arrive(v);
          }
        } else if (lane == 0) {
          p_arrive(v);
        }
        __syncwarp();
      }
      g += tiles;
      seq += tiles * (kslots + vslots);
    }
  } else {
    // ---------------- softmax, epilogue ----------------
    // When S of tile t is there, P V of tile t - 2 is done and that of t - 1
    // may not be: two barriers by tile parity keep the waits unambiguous.
    const int quarter = warp & 3, half = warp >> 2;
    const int r = quarter * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int ocols = a.dv >> 1, o0 = half * ocols;  // this thread's result columns
    float* xchg = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 1024);  // [2][128]
    bool stop = false;
    int units = 0;
    if constexpr (MANY) {
      if (lane == 0) bars->walk[warp] = Walk{};
      __syncwarp();
    }
    for (int i = 0; !stop; ++i) {
    int tiles, vis, vis0;
    {
      Unit u;
      Walk w;
      if constexpr (MANY) w = bars->walk[warp];
      if (!next_unit(i, u, w)) break;
      if constexpr (MANY) {
        __syncwarp();
        if (lane == 0) bars->walk[warp] = w;
        __syncwarp();
      }
      // kept in shared memory for the epilogue: registers are short in between
      if (tid == 0) bars->unit = u;
      const int j0 = u.first + rank * kTile;
      tiles = tiles_of(u);
      vis = j0 + r < u.nq ? u.seen(a, j0 + r) : 0;
      vis0 = u.seen(a, j0);
    }
    float m = -INFINITY, l = 0.f;  // m: the maximum in use less kWeightShift, from which weights are counted
    if (tiles > 0) ++units;
    for (int t = 0; t < tiles; ++t) {
      const uint32_t v_ = g + t, b = v_ & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->s_full[b]), (v_ >> 1) & 1u, abort_flag))) {
        stop = true;
      }
      float v[64];
      if (!stop) {
        tmem_fence_after();
        uint32_t w[32];
        const uint32_t src = tmem + lanes + kSCol + b * kTile + half * 64;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          tmem_ld32(src + 32 * h, w);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 32; ++i) v[32 * h + i] = __uint_as_float(w[i]);
        }
        if (a.negative) {
#pragma unroll
          for (int i = 0; i < 64; ++i) v[i] = -v[i];
        }
      }
      const int key0 = t * kTile + half * 64;
      const bool masked = (t + 1) * kTile > vis0;
      if (masked) {
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = key0 + i < vis ? v[i] : -INFINITY;
      }
      float top = v[0];
#pragma unroll
      for (int i = 1; i < 64; ++i) top = fmaxf(top, v[i]);
      // the largest exponent as it is formed below, whatever FP32 makes of m + slack;
      // also orders every read of S before the stores of P into its columns
      const bool grow = any_of(stop || fmaf(top, a.c, -m) > kMaxSlack + kWeightShift<E>, 1, kSoftThreads);
      if (grow) {
        stop = any_of(stop, 1, kSoftThreads);
        if (stop) break;
        xchg[half * kTile + r] = top * a.c;
        bar_sync(1, kSoftThreads);
        top = fmaxf(m, fmaxf(xchg[r], xchg[kTile + r]) - kWeightShift<E>);
        bar_sync(1, kSoftThreads);
        const float f = top == m ? 1.f : ex2(m - top);
        m = top;
        l *= f;
        if (t > 0) {
          // (a warp whose wait gives up goes on: all stop at the next tile)
          if (__all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->o_done[(v_ - 1) & 1]), ((v_ - 1) >> 1) & 1u, abort_flag))) {
            tmem_fence_after();
            for (int o = 0; o < ocols; o += 32) {
              uint32_t w[32];
              tmem_ld32(tmem + lanes + kOCol + o0 + o, w);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) w[i] = __float_as_uint(__uint_as_float(w[i]) * f);
              tmem_st32(tmem + lanes + kOCol + o0 + o, w);
            }
            tmem_wait_st();
          }
        }
      }
      const float sub = m == -INFINITY ? 0.f : m;
      uint32_t w[32];
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float p0 = ex2(fmaf(v[2 * i], a.c, -sub)), p1 = ex2(fmaf(v[2 * i + 1], a.c, -sub));
        sum += p0 + p1;
        w[i] = Elem<E>::pack(p0, p1);
      }
      // A tile's weights are added up before they meet the running sum: one by
      // one, small ones would be rounded against a large one thousands of times
      // (30,000 keys, all but one 17.5 nats below the first: 3.8e-4 off the log-sum).
      l += sum;
      tmem_st32(tmem + lanes + kSCol + b * kTile + half * 32, w);
      tmem_wait_st();
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) p_arrive(v_);
      __syncwarp();
    }
    g += tiles;
    if (!stop && tiles > 0)
      stop = !__all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->o_done[(g - 1) & 1]), ((g - 1) >> 1) & 1u, abort_flag));
    stop = any_of(stop, 1, kSoftThreads);
    if (!stop) {
      tmem_fence_after();
      xchg[half * kTile + r] = l;
      const Unit u = bars->unit;
      const int j0 = u.first + rank * kTile;
      bar_sync(1, kSoftThreads);
      l = xchg[r] + xchg[kTile + r];
      const bool poison = tiles > 0 && bars->poison[units & 1] == units;
      const float inv = inverse_sum(l);
      const bool mine = j0 + r < u.nq;
      const int64_t at = (int64_t)(u.q0 + j0 + r) * a.H + u.head;
      if (mine && a.lse && half == 0)
        a.lse[at] = vis > 0 ? ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2 : -INFINITY;
      for (int o = 0; o < ocols; o += 32) {
        uint32_t w[32];
        if (tiles > 0) {
          tmem_ld32(tmem + lanes + kOCol + o0 + o, w);
          tmem_wait_ld();
        }
        float f[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) f[i] = vis > 0 ? __uint_as_float(w[i]) * inv : 0.f;
        if (poison) {
          for (int k = cut_of(u) * kTile; k < vis; ++k) {
            const uint16_t* src = a.v + (int64_t)(u.k0 + k) * a.v_t + u.head * a.v_h + o0 + o;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (not_finite<E>(src[i])) f[i] += Elem<E>::to_float(src[i]);
          }
        }
        // four lanes exchange their rows' four pieces, so that a store of the quad
        // is 64 bytes of one row
        uint4 p[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          p[i] = make_uint4(Elem<E>::pack(f[8 * i], f[8 * i + 1]), Elem<E>::pack(f[8 * i + 2], f[8 * i + 3]),
                            Elem<E>::pack(f[8 * i + 4], f[8 * i + 5]), Elem<E>::pack(f[8 * i + 6], f[8 * i + 7]));
        quad_transpose(p, lane);
        const int row = r & ~3;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j0 + row + i < u.nq)
            *reinterpret_cast<uint4*>(a.out + ((int64_t)(u.q0 + j0 + row + i) * a.H + u.head) * a.dv + o0 + o +
                                      8 * (lane & 3)) = p[i];
      }
    }
    tmem_fence_before();
    }
  }
  // Rows outside every request: their log-sums, with fill_tail the results too.
  // The warps that are done early look whether all starts are in order.
  const int64_t cta = (int64_t)blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t ctas = min((int64_t)gridDim.x * gridDim.y, (int64_t)kFillCtas);
  const bool fills = (a.fill_tail || a.lse) && cta < ctas;
  bool unordered = false;
  if (fills && warp >= 10)
    for (int i = tid - 320; i < a.B; i += 64) unordered |= !bounds_of(a, i).ordered;
  const bool disorder = __syncthreads_or(unordered);
  if constexpr (PAIR) cluster_sync();  // neither CTA leaves while the other may reach its memory
  if (fills) {
    const int pieces = a.fill_tail ? a.dv >> 3 : 1;
    auto fill = [&](int64_t lo, int64_t hi) {
      const int64_t all = (hi - lo) * a.H * pieces;
      for (int64_t i = cta * kThreads + tid; i < all; i += ctas * kThreads) {
        const int64_t at = lo * a.H + i / pieces;
        const int piece = (int)(i % pieces);
        if (a.fill_tail) reinterpret_cast<uint4*>(a.out + at * a.dv)[piece] = make_uint4(0, 0, 0, 0);
        if (a.lse && piece == 0) a.lse[at] = -INFINITY;
      }
    };
    if (!disorder) {
      fill(0, a.B ? a.q_starts[0] : 0);
      fill(a.B ? a.q_starts[a.B] : 0, a.Tq);
    } else {
      // what lies between the requests that keep their queries
      int top = 0, done = 0;
      for (int r0 = 0; r0 < a.B; r0 += 32) {
        Bounds b{};
        if (r0 + lane < a.B) b = bounds_of(a, r0 + lane);
        const bool keeps = keeps_queries(a, b, top);
        for (uint32_t left = __ballot_sync(0xffffffffu, keeps); left; left &= left - 1) {
          const int src = __ffs(left) - 1;
          const int q0 = __shfl_sync(0xffffffffu, (int)b.q0, src), nq = __shfl_sync(0xffffffffu, (int)b.nq, src);
          fill(done, q0);
          done = q0 + nq;
        }
      }
      fill(done, a.Tq);
    }
  }
  if (tid == 0 && bars->abort_flag) report(a.status, a.status_host, kStatusWaitTimeout);
  if (warp == 9) {
    tmem_fence_after();
    tmem_free_all<PAIR>(bars->tmem_base);
  }
  if constexpr (PAIR) cluster_sync();
}

bool stride_ok(int64_t s, int64_t count) {
  return s % 8 == 0 && s < (int64_t)1 << 38 && (count > 1 ? s > 0 : s >= 0);
}

// [tokens][heads][dim] view (strides in elements), box 64 values x 1 head x box_rows tokens.
int make_rows_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t heads, int64_t stride_h,
                  int64_t tokens, int64_t stride_t, int box_rows) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("glm53_latent_expanded: cuTensorMapEncodeTiled is unavailable");
    return GLM53_ERR_CUDA;
  }
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)(stride_h ? stride_h : 8) * 2, (cuuint64_t)(stride_t ? stride_t : 8) * 2};
  cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows};
  cuuint32_t step[3] = {1, 1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(base),
         dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("glm53_latent_expanded: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return GLM53_ERR_CUDA;
  }
  return GLM53_OK;
}

int make_shared_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t tokens, int64_t stride_t, int box_rows) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("glm53_latent_expanded: cuTensorMapEncodeTiled is unavailable");
    return GLM53_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)tokens};
  cuuint64_t strides[1] = {(cuuint64_t)(stride_t ? stride_t : 8) * 2};
  cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
  cuuint32_t step[2] = {1, 1};
  const CUresult r =
      fn(map, bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2, const_cast<void*>(base),
         dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_last_error("glm53_latent_expanded: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return GLM53_ERR_CUDA;
  }
  return GLM53_OK;
}

template <typename E, bool PAIR, bool MANY = false>
int launch(const CUtensorMap& qn, const CUtensorMap& qr, const CUtensorMap& kn, const CUtensorMap& kr,
           const CUtensorMap& v, const Args& a, cudaStream_t st) {
  const auto kernel = expanded_kernel<E, PAIR, MANY>;
  const int rc = ensure_max_smem((const void*)kernel, kSmemBytes);
  if (rc) return rc;
  // Units at most: one more a request than whole units in all.
  constexpr int kCtas = PAIR ? 2 : 1, kUnit = kCtas * kTile;
  const int64_t units = (a.Tq + kUnit - 1) / kUnit + a.B;
  Args b = a;
  // A CTA an SM walks the units: the next one's queries and keys load, and its
  // first scores form, under the results of the last.  64 heads, walking / one
  // unit a CTA: 16 x 150 queries and keys of 256 + 256 values 136 / 164 us,
  // 4 x 512 92 / 111, 1 x 2,048 of 256 + 192 172 / 182.  All heads of a query
  // tile come before the next tile, so one request's keys and values of all
  // heads should stay in L2 (126 MB): over 8,192 keys of 256 + 192 values
  // (402 MB) 947 / 772, of 192 + 64 (201 MB) 615 / 543.  Many short requests, one
  // unit a CTA / walking: 300 of 100 queries and keys 2,230 / 1,051, 2,000 of 3 and
  // 20 19,960 / 5,720.  A pair's units are long and stay one each.  Lengths are on
  // the device: `held` and the rule for pairs go by averages, measured with equal
  // requests, and one long request among many short ones gets what those get.
  const double held = 2.0 * a.Tk / a.B * a.H * (a.dn + a.dv);
  b.persistent = !PAIR && held <= 126e6;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = b.persistent ? dim3((unsigned)std::min<int64_t>(sm_count(), units * a.H))
                             : dim3((unsigned)(units * kCtas), (unsigned)a.H);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kSmemBytes;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = kCtas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = PAIR ? 1 : 0;
  cudaLaunchKernelEx(&cfg, kernel, qn, qr, kn, kr, v, b);
  return check_launch("expanded_kernel");
}

}  // namespace
}  // namespace latent
}  // namespace glm53

using namespace glm53;
using namespace glm53::latent;

extern "C" int glm53_latent_expanded(const void* q_nope, int64_t qn_stride_t, int64_t qn_stride_h, const void* q_rope,
                                     int64_t qr_stride_t, int64_t qr_stride_h, const void* k_nope, int64_t kn_stride_t,
                                     int64_t kn_stride_h, const void* k_rope, int64_t kr_stride_t, const void* values,
                                     int64_t v_stride_t, int64_t v_stride_h, int64_t query_tokens, int64_t key_tokens,
                                     int64_t heads, int64_t nope_dim, int64_t rope_dim, int64_t value_dim, int dtype,
                                     const int32_t* query_starts, const int32_t* key_starts, int64_t requests,
                                     float scale, int causal, void* out, float* lse, int fill_tail, uint32_t* status,
                                     uint32_t* status_host, void* stream) {
  const char* fn = "glm53_latent_expanded";
  if (dtype != GLM53_DTYPE_BF16 && dtype != GLM53_DTYPE_FP16) {
    set_last_error("%s: unknown element type %d", fn, dtype);
    return GLM53_ERR_INVALID;
  }
  if (nope_dim <= 0 || nope_dim % 64 != 0 || (rope_dim != 0 && rope_dim != 64) || nope_dim + rope_dim > 256 ||
      value_dim <= 0 || value_dim % 64 != 0 || value_dim > 256) {
    set_last_error("%s: nope %lld, rotary %lld (0 or 64) and value %lld sizes are multiples of 64; queries and values "
                   "hold at most 256",
                   fn, (long long)nope_dim, (long long)rope_dim, (long long)value_dim);
    return GLM53_ERR_INVALID;
  }
  if (query_tokens < 0 || query_tokens > INT32_MAX || key_tokens < 0 || key_tokens > INT32_MAX || heads < 1 ||
      heads > 1024 || requests < 0 || requests > 65535 || !std::isfinite(scale)) {
    set_last_error("%s: %lld heads (1 to 1024), %lld requests (up to 65535), a finite scale", fn, (long long)heads,
                   (long long)requests);
    return GLM53_ERR_INVALID;
  }
  const int64_t Tq = query_tokens, Tk = key_tokens;
  if (!stride_ok(qn_stride_t, Tq) || !stride_ok(qn_stride_h, heads) || !stride_ok(kn_stride_t, Tk) ||
      !stride_ok(kn_stride_h, heads) || !stride_ok(v_stride_t, Tk) || !stride_ok(v_stride_h, heads) ||
      (rope_dim &&
       (!stride_ok(qr_stride_t, Tq) || !stride_ok(qr_stride_h, heads) || !stride_ok(kr_stride_t, Tk)))) {
    set_last_error("%s: strides must be positive multiples of 8", fn);
    return GLM53_ERR_INVALID;
  }
  if (query_tokens == 0) return GLM53_OK;
  if (!q_nope || !out || (rope_dim && !q_rope) || (key_tokens && (!k_nope || !values || (rope_dim && !k_rope))) ||
      !query_starts || !key_starts ||
      (((uintptr_t)q_nope | (uintptr_t)q_rope | (uintptr_t)k_nope | (uintptr_t)k_rope | (uintptr_t)values |
        (uintptr_t)out) & 15)) {
    set_last_error("%s: tensors must be non-NULL and 16-byte aligned", fn);
    return GLM53_ERR_INVALID;
  }
  const bool bf16 = dtype == GLM53_DTYPE_BF16;
  // Two CTAs take 256 queries as a pair, each reading and holding half of K and
  // V, where requests are long enough to pay for the pair's hand-shakes and for
  // units of 256 rows.  Measured, CTAs alone / pairs: 64 heads of 256 + 256
  // values, 1,024 queries and keys 72 / 83 us, 2,048 194 / 188, 512 queries over
  // 4,096 keys 140 / 122, 2,048 over 8,192 856 / 715; 16 heads of 192 + 128
  // values, 4 x 512 queries over 512 keys 24 / 33, over 2,512 72.5 / 72.3, 512
  // over 4,096 51 / 48.
  // With one query tile a request a pair's second half of rows is empty, but two
  // SMs read its keys: worth it for wide rows while there are SMs for all pairs.
  // Alone / pairs, 128 queries over 8,192 keys: 64 heads of 256 + 256 values
  // 137 / 118, 8 heads 119 / 95 (over 2,048 37 / 33), 64 heads of 256 + 128
  // values 97.5 / 98.8, 96 heads 104 / 212.
  const bool one_tile = Tq <= requests * kTile;
  const bool pair = value_dim % 128 == 0 &&
                    (one_tile ? nope_dim + rope_dim + value_dim > 448 && 2 * requests * heads <= sm_count() &&
                                    Tk >= requests * 2560
                              : Tk >= requests * 2048);
  const int key_rows = pair ? kTile / 2 : kTile;
  CUtensorMap qn, qr, kn, kr, v;
  int rc = make_rows_map(&qn, q_nope, bf16, nope_dim, heads, qn_stride_h, Tq, qn_stride_t, kTile);
  if (rc) return rc;
  qr = kn = kr = v = qn;  // maps that no load reads (no rotary part, no keys)
  if (rope_dim && (rc = make_rows_map(&qr, q_rope, bf16, rope_dim, heads, qr_stride_h, Tq, qr_stride_t, kTile)))
    return rc;
  if (Tk) {
    if ((rc = make_rows_map(&kn, k_nope, bf16, nope_dim, heads, kn_stride_h, Tk, kn_stride_t, key_rows))) return rc;
    if ((rc = make_rows_map(&v, values, bf16, value_dim, heads, v_stride_h, Tk, v_stride_t, kTile))) return rc;
    if (rope_dim && (rc = make_shared_map(&kr, k_rope, bf16, rope_dim, Tk, kr_stride_t, key_rows))) return rc;
  }
  // a masked score is -inf, which a factor of 0 would turn into NaN
  const float c = std::max(std::fabs(scale) * kLog2e, 1e-37f);
  Args a{Tq, Tk, (int)heads, (int)nope_dim, (int)rope_dim, (int)value_dim, query_starts, key_starts, (int)requests,
         c, scale < 0, causal, (const uint16_t*)values, v_stride_t, v_stride_h, (uint16_t*)out, lse, fill_tail, 0,
         status, status_host};
  const cudaStream_t st = (cudaStream_t)stream;
  if (pair)
    return bf16 ? launch<__nv_bfloat16, true>(qn, qr, kn, kr, v, a, st) : launch<__half, true>(qn, qr, kn, kr, v, a, st);
  // Softmax warps whose search for a unit goes on where it stood, for many
  // requests: 64 heads, from the start / so, 200 requests of 20 queries and 40
  // keys 682 / 640 us, 300 1,081 / 951, 2,000 of 3 and 20 17,050 / 5,720; but what
  // is kept in shared memory costs 8 requests of 512 156 / 161, five ragged ones
  // of 16 heads 31.1 / 31.6 (both spill: 164 / 176 bytes stored, 132 / 152 loaded).
  if (requests > 128)
    return bf16 ? launch<__nv_bfloat16, false, true>(qn, qr, kn, kr, v, a, st)
                : launch<__half, false, true>(qn, qr, kn, kr, v, a, st);
  return bf16 ? launch<__nv_bfloat16, false>(qn, qr, kn, kr, v, a, st) : launch<__half, false>(qn, qr, kn, kr, v, a, st);
}
