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
// Roles: warps 0-7 softmax (two threads a row, 64 keys each) and epilogue,
// warp 8 TMA, warp 9 MMA, warps 10 and 11 clean values (below).  Every mbarrier wait is bounded; a CTA that gives up
// sets GLM53_STATUS_WAIT_TIMEOUT, waits for its copies and MMAs, frees its
// TMEM and exits.
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
constexpr int kOCol = 0;     // TMEM: O at 0..255, S tiles at 256 and 384
constexpr int kSCol = 256;

struct Args {
  int64_t Tq, Tk;
  int H, dn, dr, dv;
  const int32_t *q_starts, *k_starts;
  int B;
  float c;  // scale log2(e)
  int causal;
  const uint16_t* v;
  int64_t v_t, v_h;
  uint16_t* out;
  float* lse;
  int fill_tail;
  uint32_t *status, *status_host;
};

struct __align__(8) Bars {
  uint64_t q_full, full[kSlots], empty[kSlots], s_full[2], p_full[2], o_done[2], drain;
  uint32_t tmem_base;
  int abort_flag;
  int poison;                       // a masked tile holds values that are not finite
  int found;                        // this CTA has a query tile
  int first;                        // its first query row in the request
  int64_t q0, k0, nq, nk;           // the request's rows
  int warp_sum[kThreads / 32];
};

// alignment slack, Q, ring, barriers, two floats a row
constexpr size_t kSmemBytes = 1024 + 4 * (size_t)kChunkBytes + kSlots * (size_t)kSlotBytes + 1024 + 2 * kTile * 4;
static_assert(sizeof(Bars) <= 1024, "barriers share one KB");
static_assert(kSmemBytes <= 232448, "227 KB a CTA");

// A request's rows, checked: invalid query bounds count as no queries, invalid
// key bounds as no keys.
struct Bounds {
  int64_t q0, nq, k0, nk;
  bool bad;
};
__device__ __forceinline__ Bounds bounds_of(const Args& a, int i) {
  Bounds b;
  b.q0 = a.q_starts[i];
  b.nq = (int64_t)a.q_starts[i + 1] - b.q0;
  b.k0 = a.k_starts[i];
  b.nk = (int64_t)a.k_starts[i + 1] - b.k0;
  b.bad = false;
  if (b.q0 < 0 || b.nq < 0 || b.q0 + b.nq > a.Tq) {
    b.bad = true;
    b.nq = 0;
  }
  if (b.k0 < 0 || b.nk < 0 || b.k0 + b.nk > a.Tk) {
    b.bad = true;
    b.k0 = b.nk = 0;
  }
  return b;
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

template <typename E>
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
  const int head = blockIdx.y;
  auto bar = [&](uint64_t* p) { return smem_addr(p); };

  if (tid == 0) {
    bars->found = 0;
    bars->abort_flag = 0;
    bars->poison = 0;
    mbar_init(bar(&bars->q_full), 1);
    for (int s = 0; s < kSlots; ++s) {
      mbar_init(bar(&bars->full[s]), 1);
      mbar_init(bar(&bars->empty[s]), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(&bars->s_full[s]), 1);
      mbar_init(bar(&bars->p_full[s]), kSoftWarps + kCleanWarps);
      mbar_init(bar(&bars->o_done[s]), 1);
    }
    mbar_init(bar(&bars->drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_addr(&bars->tmem_base)),
                 "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp == 8 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qn_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&qr_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kn_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&kr_map)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&v_map)) : "memory");
  }
  __syncwarp();

  // which request and query tile: count tiles over the requests, a block's
  // worth at a time
  int base = 0;
  for (int r0 = 0; r0 < a.B; r0 += kThreads) {
    int n = 0;
    Bounds b{};
    if (r0 + tid < a.B) {
      b = bounds_of(a, r0 + tid);
      n = (int)((b.nq + kTile - 1) / kTile);
      if (b.bad && blockIdx.x == 0 && head == 0) report(a.status, a.status_host, kStatusBadGeometry);
    }
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int x = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += x;
    }
    if (lane == 31) bars->warp_sum[warp] = s;
    __syncthreads();
    int before = base;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
      if (w < warp) before += bars->warp_sum[w];
      base += bars->warp_sum[w];
    }
    const int lo = before + s - n;
    if ((int)blockIdx.x >= lo && (int)blockIdx.x < lo + n) {
      bars->found = 1;
      // the later query tiles see more keys: they go first
      bars->first = (n - 1 - ((int)blockIdx.x - lo)) * kTile;
      bars->q0 = b.q0;
      bars->nq = b.nq;
      bars->k0 = b.k0;
      bars->nk = b.nk;
    }
    if (base > (int)blockIdx.x) break;
    __syncthreads();
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  if (!bars->found) {
    if (warp == 9)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(bars->tmem_base), "r"(512) : "memory");
    // surplus CTAs zero the rows outside every request
    if (a.fill_tail) {
      int64_t lo = a.B ? a.q_starts[a.B] : 0, hi = a.B ? a.q_starts[0] : 0;
      lo = lo < 0 ? 0 : lo;
      hi = hi < 0 ? 0 : (hi > a.Tq ? a.Tq : hi);
      const int64_t rows = hi + (a.Tq > lo ? a.Tq - lo : 0);
      const int pieces = a.dv >> 3;
      const int64_t step = (int64_t)(gridDim.x - base) * kThreads;
      for (int64_t i = (int64_t)(blockIdx.x - base) * kThreads + tid; i < rows * pieces; i += step) {
        const int64_t k = i / pieces, row = k < hi ? k : lo + (k - hi);
        const int64_t at = row * a.H + head;
        reinterpret_cast<uint4*>(a.out + at * a.dv)[i - k * pieces] = make_uint4(0, 0, 0, 0);
        if (a.lse && i == k * pieces) a.lse[at] = -INFINITY;
      }
    }
    return;
  }
  const Bounds bd{bars->q0, bars->nq, bars->k0, bars->nk, false};
  const int j0 = bars->first;
  const int rows = (int)(bd.nq - j0 < kTile ? bd.nq - j0 : kTile);
  const int nk = (int)bd.nk;
  const int vis0 = a.causal ? (int)max((int64_t)0, min(bd.nk, bd.nk - bd.nq + j0 + 1)) : nk;  // row 0's keys
  const int vis_last = a.causal ? (int)max((int64_t)0, min(bd.nk, bd.nk - bd.nq + j0 + rows)) : nk;
  const int tiles = (vis_last + kTile - 1) / kTile;
  const int nch = (a.dn + a.dr) / 64, kslots = (nch + 1) / 2, vch = a.dv / 64, vslots = (vch + 1) / 2;
  const int64_t q0 = bd.q0 + j0, k0 = bd.k0;

  constexpr uint32_t tmem = 0;  // all 512 columns are this CTA's
  volatile int* abort_flag = &bars->abort_flag;

  if (warp == 8) {
    // ---------------- TMA ----------------
    if (lane == 0 && tiles > 0) {
      mbar_expect_tx(bar(&bars->q_full), nch * kChunkBytes);
      for (int c = 0; c < nch; ++c) {
        const bool rope = c * 64 >= a.dn;
        tma_load_3d(smem_addr(q_smem + c * kChunkBytes), rope ? &qr_map : &qn_map, rope ? 0 : c * 64, head, (int)q0,
                    bar(&bars->q_full));
      }
      uint32_t seq = 0;
      bool ok = true;
      auto slot = [&](bool value, int tile, int part, int chunks) {
        const uint32_t s = seq % kSlots;
        if (seq >= kSlots) ok = mbar_wait(bar(&bars->empty[s]), (seq / kSlots - 1) & 1u, abort_flag);
        if (!ok) return;
        const int n = min(2, chunks - 2 * part);
        mbar_expect_tx(bar(&bars->full[s]), n * kChunkBytes);
        for (int c = 0; c < n; ++c) {
          const uint32_t dst = smem_addr(ring + s * kSlotBytes + c * kChunkBytes);
          const int x = (2 * part + c) * 64, z = (int)(k0 + (int64_t)tile * kTile);
          if (value)
            tma_load_3d(dst, &v_map, x, head, z, bar(&bars->full[s]));
          else if (x >= a.dn)
            tma_load_2d(dst, &kr_map, 0, z, bar(&bars->full[s]));
          else
            tma_load_3d(dst, &kn_map, x, head, z, bar(&bars->full[s]));
        }
        ++seq;
      };
      for (int t = 0; t <= tiles && ok; ++t) {
        for (int p = 0; p < kslots && ok && t < tiles; ++p) slot(false, t, p, nch);
        for (int p = 0; p < vslots && ok && t > 0; ++p) slot(true, t - 1, p, vch);
      }
      if (!ok) {
        // copies still in flight write this CTA's shared memory: wait for them
        volatile int never = 0;
        for (uint32_t k = seq > kSlots ? seq - kSlots : 0; k < seq; ++k)
          mbar_wait(bar(&bars->full[k % kSlots]), (k / kSlots) & 1u, &never);
        never = 0;
        mbar_wait(bar(&bars->q_full), 0, &never);
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA ----------------
    // All lanes walk the loops, so that descriptors stay in uniform registers;
    // one elected lane waits and issues, eight unrolled MMAs a slot.
    if (tiles > 0) {
      constexpr bool bf16 = std::is_same<E, __nv_bfloat16>::value;
      constexpr uint32_t id_s = make_idesc_f16(kTile, kTile, bf16, false, false);
      const bool leader = elect_one();
      uint32_t seq = 0;
      bool ok = true;
      const uint64_t qd = make_sw128_desc(smem_addr(q_smem));
      const uint64_t kd0 = make_sw128_desc(smem_addr(ring)), vd0 = make_sw128_mn_desc(smem_addr(ring), kChunkBytes);
      if (leader) ok = mbar_wait_fast(bar(&bars->q_full), 0, abort_flag);
      for (int t = 0; t <= tiles; ++t) {
        if (t < tiles) {
          const uint32_t d = kSCol + (t & 1) * kTile;
          for (int p = 0; p < kslots; ++p, ++seq) {
            const uint32_t s = seq % kSlots, phase = (seq / kSlots) & 1u;
            const uint64_t ad = qd + (uint64_t)(p * (kSlotBytes >> 4));
            const uint64_t kd = kd0 + (uint64_t)(s * (kSlotBytes >> 4));
            if (leader) {
              ok = ok && mbar_wait_fast(bar(&bars->full[s]), phase, abort_flag);
              tmem_fence_after();
              if (ok) {
#pragma unroll
                for (int k = 0; k < 4; ++k) mma_f16_ss(d, ad + 2 * k, kd + 2 * k, id_s, (p | k) != 0);
                if (2 * p + 1 < nch) {
#pragma unroll
                  for (int k = 0; k < 4; ++k)
                    mma_f16_ss(d, ad + (kChunkBytes >> 4) + 2 * k, kd + (kChunkBytes >> 4) + 2 * k, id_s, 1);
                }
                mma_commit(bar(&bars->empty[s]));
              }
            }
          }
          if (leader && ok) mma_commit(bar(&bars->s_full[t & 1]));
        }
        if (t > 0) {
          const int u = t - 1;
          const uint32_t pa = kSCol + (u & 1) * kTile;
          const int steps = (min(kTile, nk - u * kTile) + 15) >> 4;
          if (leader) ok = ok && mbar_wait_fast(bar(&bars->p_full[u & 1]), (u >> 1) & 1u, abort_flag);
          for (int p = 0; p < vslots; ++p, ++seq) {
            const uint32_t s = seq % kSlots, phase = (seq / kSlots) & 1u;
            const uint32_t id_o = 2 * p + 1 < vch ? make_idesc_f16(kTile, 128, bf16, false, true)
                                                  : make_idesc_f16(kTile, 64, bf16, false, true);
            const uint64_t vd = vd0 + (uint64_t)(s * (kSlotBytes >> 4));
            const uint32_t o = kOCol + p * 128;
            if (leader) {
              ok = ok && mbar_wait_fast(bar(&bars->full[s]), phase, abort_flag);
              tmem_fence_after();
              if (ok) {
                if (steps == 8) {
#pragma unroll
                  for (int k = 0; k < 8; ++k) mma_f16_ts(o, pa + 8 * k, vd + 128 * k, id_o, (u | k) != 0);
                } else {
                  for (int k = 0; k < steps; ++k) mma_f16_ts(o, pa + 8 * k, vd + 128 * k, id_o, (u | k) != 0);
                }
                mma_commit(bar(&bars->empty[s]));
              }
            }
          }
          if (leader && ok) mma_commit(bar(&bars->o_done[u & 1]));
        }
      }
      // no MMA is in flight when TMEM is freed.  The lane that issued waits
      // alone: a lane that spins must not keep its warp from one with work.
      if (leader) {
        volatile int never = 0;
        mma_commit(bar(&bars->drain));
        if (!mbar_wait(bar(&bars->drain), 0, &never)) *abort_flag = 1;
      }
    }
    __syncwarp();
  } else if (warp >= 10) {
    // ---------------- values of the tiles that the mask cuts ----------------
    bool ok = true;
    for (int t = 0; t < tiles; ++t) {
      ok = ok && __all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->s_full[t & 1]), (t >> 1) & 1u, abort_flag));
      if ((t + 1) * kTile > vis0 && ok) {
        // value slots of tile t in the order the producer fills the ring; once
        // tile t - 1 is multiplied, each slot's previous use is over and its
        // barrier's parity means this one
        if (t > 0)
          ok = __all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->o_done[(t - 1) & 1]), ((t - 1) >> 1) & 1u, abort_flag));
        const uint32_t s0 = kslots + t * (kslots + vslots) + (t + 1 < tiles ? kslots : 0);
        const int valid = min(kTile, nk - t * kTile), end = (valid + 15) & ~15;  // the product stops at `end`
        bool found = false;
        for (int c = 0; c < vch && ok; ++c) {
          const uint32_t q = s0 + (c >> 1), s = q % kSlots;
          if (!(c & 1))
            ok = __all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->full[s]), (q / kSlots) & 1u, abort_flag));
          for (int row = tid - 320; row < end && ok; row += 64)
            found |= clean_row<E>(ring + s * kSlotBytes + (c & 1) * kChunkBytes, row, valid);
        }
        if (found) bars->poison = 1;
        fence_async_shared();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&bars->p_full[t & 1]));
      __syncwarp();
    }
  } else {
    // ---------------- softmax, epilogue ----------------
    // When S of tile t is there, P V of tile t - 2 is done and that of t - 1
    // may not be: two barriers by tile parity keep the waits unambiguous.
    const int quarter = warp & 3, half = warp >> 2;
    const int r = quarter * 32 + lane;  // row of the tile = TMEM lane
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const int vis = r < rows ? (a.causal ? (int)max((int64_t)0, min(bd.nk, bd.nk - bd.nq + j0 + r + 1)) : nk) : 0;
    const int ocols = a.dv >> 1, o0 = half * ocols;  // this thread's result columns
    float m = -INFINITY, l = 0.f;
    bool stop = false;
    float* xchg = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(bars) + 1024);  // [2][128]
    for (int t = 0; t < tiles; ++t) {
      const int b = t & 1;
      if (!__all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->s_full[b]), (t >> 1) & 1u, abort_flag))) {
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
          for (int i = 0; i < 32; ++i) v[32 * h + i] = __uint_as_float(w[i]) * a.c;
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
      // also orders every read of S before the stores of P into its columns
      const bool grow = any_of(stop || top > m + kMaxSlack, 1, kSoftThreads);
      if (grow) {
        stop = any_of(stop, 1, kSoftThreads);
        if (stop) break;
        xchg[half * kTile + r] = top;
        bar_sync(1, kSoftThreads);
        top = fmaxf(m, fmaxf(xchg[r], xchg[kTile + r]));
        bar_sync(1, kSoftThreads);
        const float f = top == m ? 1.f : ex2(m - top);
        m = top;
        l *= f;
        if (t > 0) {
          // (a warp whose wait gives up goes on: all stop at the next tile)
          if (__all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->o_done[(t - 1) & 1]), ((t - 1) >> 1) & 1u, abort_flag))) {
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
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float p0 = ex2(v[2 * i] - sub), p1 = ex2(v[2 * i + 1] - sub);
        l += p0 + p1;
        w[i] = Elem<E>::pack(p0, p1);
      }
      tmem_st32(tmem + lanes + kSCol + b * kTile + half * 32, w);
      tmem_wait_st();
      tmem_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(&bars->p_full[b]));
      __syncwarp();
    }
    if (!stop && tiles > 0)
      stop = !__all_sync(0xffffffffu, mbar_wait_fast(bar(&bars->o_done[(tiles - 1) & 1]), ((tiles - 1) >> 1) & 1u, abort_flag));
    stop = any_of(stop, 1, kSoftThreads);
    if (!stop) {
      tmem_fence_after();
      xchg[half * kTile + r] = l;
      bar_sync(1, kSoftThreads);
      l = xchg[r] + xchg[kTile + r];
      const bool poison = bars->poison != 0;
      const float inv = 1.f / l;
      const int64_t at = (q0 + r) * a.H + head;
      if (r < rows && a.lse && half == 0)
        a.lse[at] = vis > 0 ? ((m == -INFINITY ? 0.f : m) + log2f(l)) * kLn2 : -INFINITY;
      // 16-bit rows into the Q buffer (every S is done), pieces of 16 bytes
      // swizzled by row, then whole rows to memory
      const int row_bytes = a.dv * 2;
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
          for (int k = vis0 / kTile * kTile; k < vis; ++k) {
            const uint16_t* src = a.v + (k0 + k) * a.v_t + head * a.v_h + o0 + o;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (not_finite<E>(src[i])) f[i] += Elem<E>::to_float(src[i]);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<uint4*>(q_smem + r * row_bytes + 16 * (((o0 + o) / 8 + i) ^ (r & 7))) =
              make_uint4(Elem<E>::pack(f[8 * i], f[8 * i + 1]), Elem<E>::pack(f[8 * i + 2], f[8 * i + 3]),
                         Elem<E>::pack(f[8 * i + 4], f[8 * i + 5]), Elem<E>::pack(f[8 * i + 6], f[8 * i + 7]));
      }
      bar_sync(1, kSoftThreads);
      const int pieces = a.dv >> 3;
      uint4* out = reinterpret_cast<uint4*>(a.out + (q0 * a.H + head) * a.dv);
      if (lane < pieces) {
#pragma unroll 4
        for (int row = warp; row < rows; row += kSoftWarps)
          out[(int64_t)row * a.H * pieces + lane] =
              *reinterpret_cast<const uint4*>(q_smem + row * row_bytes + 16 * (lane ^ (row & 7)));
      }
    }
    tmem_fence_before();
  }
  __syncthreads();
  if (tid == 0 && bars->abort_flag) report(a.status, a.status_host, kStatusWaitTimeout);
  if (warp == 9) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(bars->tmem_base), "r"(512) : "memory");
  }
}

bool stride_ok(int64_t s, int64_t count) {
  return s % 8 == 0 && s < (int64_t)1 << 38 && (count > 1 ? s > 0 : s >= 0);
}

// [tokens][heads][dim] view (strides in elements), box 64 values x 1 head x 128 tokens.
int make_rows_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t heads, int64_t stride_h,
                  int64_t tokens, int64_t stride_t) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("glm53_latent_expanded: cuTensorMapEncodeTiled is unavailable");
    return GLM53_ERR_CUDA;
  }
  cuuint64_t dims[3] = {(cuuint64_t)dim, (cuuint64_t)heads, (cuuint64_t)tokens};
  cuuint64_t strides[2] = {(cuuint64_t)(stride_h ? stride_h : 8) * 2, (cuuint64_t)(stride_t ? stride_t : 8) * 2};
  cuuint32_t box[3] = {64, 1, kTile};
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

int make_shared_map(CUtensorMap* map, const void* base, bool bf16, int64_t dim, int64_t tokens, int64_t stride_t) {
  auto fn = encode_fn();
  if (!fn) {
    set_last_error("glm53_latent_expanded: cuTensorMapEncodeTiled is unavailable");
    return GLM53_ERR_CUDA;
  }
  cuuint64_t dims[2] = {(cuuint64_t)dim, (cuuint64_t)tokens};
  cuuint64_t strides[1] = {(cuuint64_t)(stride_t ? stride_t : 8) * 2};
  cuuint32_t box[2] = {64, kTile};
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
  CUtensorMap qn, qr, kn, kr, v;
  int rc = make_rows_map(&qn, q_nope, bf16, nope_dim, heads, qn_stride_h, Tq, qn_stride_t);
  if (rc) return rc;
  qr = kn = kr = v = qn;  // maps that no load reads (no rotary part, no keys)
  if (rope_dim && (rc = make_rows_map(&qr, q_rope, bf16, rope_dim, heads, qr_stride_h, Tq, qr_stride_t))) return rc;
  if (Tk) {
    if ((rc = make_rows_map(&kn, k_nope, bf16, nope_dim, heads, kn_stride_h, Tk, kn_stride_t))) return rc;
    if ((rc = make_rows_map(&v, values, bf16, value_dim, heads, v_stride_h, Tk, v_stride_t))) return rc;
    if (rope_dim && (rc = make_shared_map(&kr, k_rope, bf16, rope_dim, Tk, kr_stride_t))) return rc;
  }
  Args a{Tq, Tk, (int)heads, (int)nope_dim, (int)rope_dim, (int)value_dim, query_starts, key_starts, (int)requests,
         scale * kLog2e, causal, (const uint16_t*)values, v_stride_t, v_stride_h, (uint16_t*)out, lse, fill_tail,
         status, status_host};
  // a tile more a request than whole tiles in all: where rows lie outside every
  // request, at least one CTA a head has no tile and zeroes them
  const dim3 grid((unsigned)((Tq + kTile - 1) / kTile + requests), (unsigned)heads);
  const auto kernel = bf16 ? expanded_kernel<__nv_bfloat16> : expanded_kernel<__half>;
  if ((rc = ensure_max_smem((const void*)kernel, kSmemBytes))) return rc;
  kernel<<<grid, kThreads, kSmemBytes, (cudaStream_t)stream>>>(qn, qr, kn, kr, v, a);
  return check_launch(fn);
}
