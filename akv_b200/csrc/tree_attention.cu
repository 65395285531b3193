// Attention of drafted token trees over the paged cache, with learned sinks.
//
// Request b has L cached keys (slots kv_indices[..], all visible to every
// drafted token) followed by its n drafted tokens (slots draft_slots[..],
// whose K/V the caller has stored).  Drafted token i sees drafted token j
// when bit j of tree_mask[i] is set, and with a window a key only when
// q_pos - k_pos <= window:
//   out_i = sum_j e^{s_ij} v_j / (sum_j e^{s_ij} + e^{sink}),  s_ij = scale q_i . k_j
// The reference verifies drafts through its native backends with a dense
// boolean mask (akv/system/sglang.patch:2170-2183 for the decode call that
// this stands beside); here one 64-bit word per token is the whole mask.
//
// Work: the rows of a KV head are (drafted token, query head of the group),
// row = token * group + head, 128 rows to a tile.  A work item is a run of
// 128-key tiles of one request for one or two (head, row tile) units; the
// host cuts the flat list of all key tiles into equal runs, one per CTA, and
// a second kernel joins the pieces of units that were cut.
//
// Bound.  A key costs Hkv D 4 bytes and 4 Hq D flops per drafted token: HBM up to
// about 16 tokens per request at a group of 8, the softmax and the tensor
// cores above.  Measured (device time): 64 requests of 16 tokens over 4K-12K
// keys at random slots, 64 / 8 heads of 64 (1.11 GB): 260-310 us over calls in a
// row (the SM clock falls under load; 260 us the fastest, 4.2 TB/s, 0.65 of the
// copy rate, 533 TFLOP/s); with its softmax taken out 208 us (the gather), with
// its loads taken out 253 us (scores -> P -> P.V per tile; a unit's 128 keys take
// about 3,900 cycles, of which 2,200 are exponentials at two warps per
// scheduler).  Trees of 33-64 tokens over 16K-32K keys of head_dim 128: 575-600 us in
// a row, 585 TFLOP/s (510-530 us alone); a head's K/V are gathered once per two row
// tiles, 437 us alone.  Short items are a chain of latencies: 128 requests of 8
// tokens and 100-140 keys in a window 45-54 us, of which at most five items of
// about 10,000 cycles in a row explain 26; what the rest is was not found.

// The pieces that decide the time: 128-key tiles with one CTA per SM (64-key
// tiles with two CTAs 342 us on the first case, 80 registers a thread spill);
// producers that issue a copy in four instructions (29 with a 64-bit
// product and a swizzle each: 299 us); masks applied to the scores in tensor
// memory, so that the ordinary path has none; a quarter of the exponentials as
// polynomials on the FMA pipes (none 287 us, three eighths 279); registers (the
// same loop at 96 instead of 128 a thread, by spills, 10 % slower).  No gain: units
// half a tile apart, scores loaded behind the work on the last ones, one pass
// over the scores with a running base, 16 softmax warps.

#include <climits>
#include <type_traits>

#include "tcgen05.cuh"

namespace akv {
namespace {

constexpr int kTreeRows = 128;
constexpr int kTreeKeys = 128;
constexpr int kTreeUnits = 2;
constexpr uint32_t kPoly = 0x1111;  // pairs of sixteen whose exponentials are polynomials

struct TreeItem {   // 12 int32
  int q0, n;        // first drafted token of the request, and their number
  int kv0, prefix;  // first cached key, and their number
  int lo, hi;       // keys [lo, hi) of prefix ++ drafted
  int head0, tile0; // unit u: head head0 + u * head_step, row tile tile0 + u * tile_step
  int head_step, tile_step;
  int units;        // 2: a pair; 1: both units share its keys
  int partial;      // first partial result (kTreeUnits per item), or -1
};

struct TreeParams {
  const void* q;
  long long q_st, q_sh;
  const void* k;
  const void* v;
  long long k_ss, k_sh, v_ss, v_sh;
  long long num_slots;
  long long tokens, keys;  // entries of the token and key vectors
  const int* kv_indices;
  const int* draft_slots;
  const unsigned long long* tree_mask;
  const int* q_positions;
  const int* kv_positions;
  long long window;  // < 0: none
  const float* sinks;
  float scale_log2;
  int group, num_q_heads;
  const TreeItem* items;
  const int* cta_items;
  float* part_acc;  // [partials][D / 4][kTreeRows][4]: a warp's rows side by side
  float* part_ml;   // [partials][kTreeRows][2]: maximum in base 2, sum
  void* out;
  long long o_st, o_sh;
  float* lse;
  int* error_flag;
};

// A pair of fp32 values as T, the lower address first.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) {
  return pack_bf16(lo, hi);
}
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

// Slot of key j of an item; -1: a padding token, read as zeros.
__device__ __forceinline__ long long key_slot(const TreeParams& p, const TreeItem& w, int j) {
  const bool cached = j < w.prefix;
  long long slot = cached ? __ldg(p.kv_indices + w.kv0 + j)
                          : __ldg(p.draft_slots + w.q0 + (j - w.prefix));
  if (slot >= p.num_slots || (cached && slot < 0)) {  // never touch memory outside the pools
    if (p.error_flag) atomicOr(p.error_flag, 1);
    slot = 0;
  }
  return slot < 0 ? -1 : slot;
}

// Visible drafted tokens of a token at `pos`: its mask m, without those the
// window hides.
__device__ __forceinline__ unsigned long long row_mask(const TreeParams& p, const TreeItem& w,
                                                       unsigned long long m, long long pos) {
  if (w.n < 64) m &= (1ull << w.n) - 1;
  if (p.window >= 0) {
    for (unsigned long long left = m; left; left &= left - 1) {
      const int j = __ffsll((long long)left) - 1;
      if (pos - p.q_positions[w.q0 + j] > p.window) m &= ~(1ull << j);
    }
  }
  return m;
}

// Joins the sink (-inf: none) to a row's maximum m (base 2) and sum l: `scale` is the
// factor of the accumulator in the output, lse the natural logarithm.  The
// maximum takes the sink in, so neither a sink far above every score nor one
// of a row without keys overflows.
struct RowEnd {
  float scale, lse;
};
__device__ __forceinline__ RowEnd row_end(float sink, float m, float l) {
  sink *= kLog2e;
  const float top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
  const float f = fast_exp2(m - base);
  const float den = l * f + fast_exp2(sink - base);
  RowEnd e;
  e.scale = den == 0.f ? 0.f : f / den;  // NaN stays NaN
  e.lse = den == 0.f ? -INFINITY : (base + log2f(den)) * kLn2;
  return e;
}

__device__ __forceinline__ void cp_async16_full(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src));
}

// The largest of three, NaN if one is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// 2^x for a pair on the FMA pipes, so that they share the exponentials with
// the special-function unit: x = i + f with i the nearest integer (the low
// bits of x + 1.5 * 2^23), 2^f on [-1/2, 1/2] by a polynomial of degree 5 with
// constant term 1, fitted to 2^f (relative error at most 1.1e-7 as a real
// polynomial, 1.7e-7 evaluated here in fp32: under 2 ulp), and i added to
// the exponent field.  At x <= -127 the result is exactly 0.  A NaN is lost
// (the caller's maximum sees it).
__device__ __forceinline__ void exp2_pair(f32x2 x, float& e0, float& e1) {
  float x0, x1;
  f2_unpack(x, x0, x1);
  x = f2_pack(fmaxf(x0, -127.f), fmaxf(x1, -127.f));
  const f32x2 magic = f2_pack(12582912.f, 12582912.f);
  const f32x2 t = f2_add(x, magic);
  const f32x2 f = f2_sub(x, f2_sub(t, magic));
  f32x2 y = f2_pack(0x1.5bba14p-10f, 0x1.5bba14p-10f);
  y = f2_fma(y, f, f2_pack(0x1.3cea88p-7f, 0x1.3cea88p-7f));
  y = f2_fma(y, f, f2_pack(0x1.c6b752p-5f, 0x1.c6b752p-5f));
  y = f2_fma(y, f, f2_pack(0x1.ebf9bcp-3f, 0x1.ebf9bcp-3f));
  y = f2_fma(y, f, f2_pack(0x1.62e42ap-1f, 0x1.62e42ap-1f));
  y = f2_fma(y, f, f2_pack(1.f, 1.f));
  float t0, t1, y0, y1;
  f2_unpack(t, t0, t1);
  f2_unpack(y, y0, y1);
  e0 = __int_as_float(__float_as_int(y0) + (__float_as_int(t0) << 23));
  e1 = __int_as_float(__float_as_int(y1) + (__float_as_int(t1) << 23));
}

// The thread's copies so far, once landed, arrive on an mbarrier.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// Zeroes the infinities and NaN of eight elements; true if there were any.
template <int HALF>
__device__ __forceinline__ bool scrub(uint4& x) {
  constexpr uint32_t kExp = HALF ? 0x7c00u : 0x7f80u;
  uint32_t e[4] = {x.x, x.y, x.z, x.w};
  bool hit = false;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if ((e[k] & kExp) == kExp) { e[k] &= 0xffff0000u; hit = true; }
    if ((e[k] >> 16 & kExp) == kExp) { e[k] &= 0xffffu; hit = true; }
  }
  x = make_uint4(e[0], e[1], e[2], e[3]);
  return hit;
}

// ws_wait by a whole warp, which then takes one way.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, ws_wait(bar, parity, abort));
}

// Tiles per bit of an item's hit word.
__device__ __forceinline__ int tiles_per_hit(int n_tiles) { return (n_tiles + 63) / 64; }

// One CTA per SM with two units, each with 256 tensor-memory columns: scores
// of 128 keys, the accumulator of D and, at head_dim 64, P beside them (at 128
// P overwrites the second half of its scores).  K and V tiles of 128 keys alternate in a ring of
// 32 KiB slots, one or two heads' rows each.  256-byte pieces gathered by
// cp.async are what reaches the copy rate on random slots (a bare gather: 6.9
// TB/s with 256-byte pieces and 16 warps per SM, 5.8 with 8, 4.9 with 128-byte
// pieces; TMA row gathers stop at 4.9, L2 prefetches cost more than they
// bring), so at head_dim 64 two heads share a CTA.
template <int D>
struct TreeCfg {
  static constexpr int kSoftmax = 8, kProducers = 4;  // warps
  static constexpr int kThreads = 32 * (kSoftmax + kProducers + 2);  // and two issuers
  static constexpr int kHeadBytes = kTreeKeys * D * 2;  // one head's rows of a tile
  static constexpr int kSlotBytes = 32768;
  static constexpr int kSlots = D == 64 ? 6 : 5;
  static constexpr int kQBytes = kTreeRows * D * 2;
  static constexpr int kRingOff = 2 * kQBytes;
  static constexpr int kRowOff = kRingOff + kSlots * kSlotBytes;  // [2][128] (maximum, sum)
  static constexpr int kBarOff = kRowOff + 2 * kTreeRows * 8;
  // Tiles of V that infinities or NaN were taken out of: a word per producer
  // warp and item, for eight items.  The producers are at most four items
  // ahead (an item has two slots at least), so a word is read before its place
  // serves another item.
  static constexpr int kHitOff = kBarOff + 256, kHitItems = 8;
  static constexpr int kSmem = kHitOff + 8 * kProducers * kHitItems;
  static constexpr int kColP = D == 64 ? 128 : 64, kColO = 256 - D;
  static_assert(kSmem <= 232448, "shared memory of one CTA");
};

// A position in the slot ring.
template <int SLOTS>
struct RingPos {
  uint32_t slot = 0, phase = 0;
  __device__ __forceinline__ void advance(uint32_t n) {  // n <= SLOTS
    slot += n;
    if (slot >= SLOTS) {
      slot -= SLOTS;
      phase ^= 1;
    }
  }
};

// Visible keys among the 64 from j0 on, as bits, of this lane's row of token i
// (position pos).  Every lane of the warp calls it; tokens rise with the lane.
__device__ __forceinline__ unsigned long long seen64(const TreeParams& p, const TreeItem& w,
                                                     unsigned long long mask, int i, int pos,
                                                     int j0, int lane) {
  if (j0 >= w.hi) return 0;
  const int cached = min(max(w.prefix - j0, 0), 64);
  unsigned long long seen;
  if (cached == 0) {
    seen = mask >> (j0 - w.prefix);  // j0 < hi <= prefix + 64
  } else {
    seen = cached < 64 ? mask << cached : 0;
    if (p.window < 0) {
      seen |= cached < 64 ? (1ull << cached) - 1 : ~0ull;
    } else {
      // Each lane tests two keys, for one of the warp's tokens after another.
      const int* kp = p.kv_positions + w.kv0 + j0;
      const bool in0 = lane < cached, in1 = lane + 32 < cached;
      const long long p0 = in0 ? kp[lane] : 0, p1 = in1 ? kp[lane + 32] : 0;
      for (unsigned left = 0xffffffffu; left;) {
        const int src = __ffs(left) - 1;
        const int token = __shfl_sync(0xffffffffu, i, src);
        const long long at = __shfl_sync(0xffffffffu, pos, src);
        const unsigned lo = __ballot_sync(0xffffffffu, in0 && at - p0 <= p.window);
        const unsigned hi = __ballot_sync(0xffffffffu, in1 && at - p1 <= p.window);
        if (i == token) seen |= (unsigned long long)hi << 32 | lo;
        left = __ballot_sync(0xffffffffu, i > token);
      }
    }
  }
  if (w.hi - j0 < 64) seen &= (1ull << (w.hi - j0)) - 1;
  return seen;
}

// Infinities and NaN were taken out of tiles of V of an item (hits: bit b for
// its tiles [b per, (b + 1) per)): adds those that a row sees to columns [d0,
// d1) of its result (out, or the partial acc).  By a whole warp, rows `live` or
// not: a lane searches a key's row and the warp then takes the keys that have
// any, as bits of their columns, one after another.  The other roles wait for
// it, 100 ms at most: measured, a tile of 128 keys with one NaN takes about 8 us,
// one of nothing but NaN 33 us (head_dim 64) or 72 us (128), so an item of
// 170,000 such keys still ends in time.
template <typename T, int D>
__device__ __noinline__ void restore(const TreeParams& p, int item, unsigned long long hits,
                                     int per, unsigned long long mask, long long pos, int head,
                                     bool live, T* out, float* acc, int d0, int d1) {
  constexpr int kWords = D / 32;
  constexpr uint32_t kExp = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
  const TreeItem w = p.items[item];
  const int lane = threadIdx.x & 31;
  uint32_t up[kWords] = {}, down[kWords] = {};  // columns with +inf, with -inf; both: NaN
  for (; hits; hits &= hits - 1) {
    const int first = w.lo + (__ffsll((long long)hits) - 1) * per * kTreeKeys;
    const int n = min(w.hi - first, per * kTreeKeys);
    for (int k0 = 0; k0 < n; k0 += 32) {
      uint32_t key_up[kWords] = {}, key_down[kWords] = {}, any = 0;
      const int j = first + k0 + lane;
      const long long slot = k0 + lane < n ? key_slot(p, w, j) : -1;
      // The key's position; without a window one that is never hidden.
      const long long at = p.window >= 0 && k0 + lane < n && j < w.prefix
                               ? p.kv_positions[w.kv0 + j] : LLONG_MAX >> 1;
      if (slot >= 0) {
        const T* row = static_cast<const T*>(p.v) + slot * p.v_ss + head * p.v_sh;
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          if (32 * k < d0 || 32 * k >= d1) continue;
          uint4 v[4];  // 32 columns, requested together
#pragma unroll
          for (int c = 0; c < 4; ++c) v[c] = *reinterpret_cast<const uint4*>(row + 32 * k + 8 * c);
#pragma unroll
          for (int e = 0; e < 32; ++e) {
            const uint32_t x = (&v[e / 8].x)[e / 2 % 4] >> 16 * (e & 1) & 0xffffu;
            if ((x & kExp) != kExp) continue;
            const bool nan = (x & 0x7fffu) != kExp;
            if (nan || !(x & 0x8000u)) key_up[k] |= 1u << e;
            if (nan || (x & 0x8000u)) key_down[k] |= 1u << e;
          }
          any |= key_up[k] | key_down[k];
        }
      }
      for (unsigned left = __ballot_sync(0xffffffffu, any); left; left &= left - 1) {
        const int src = __ffs(left) - 1;
        const int drafted = first + k0 + src - w.prefix;
        const long long key_at = __shfl_sync(0xffffffffu, at, src);
        const bool seen = live && (drafted >= 0 ? mask >> drafted & 1 : pos - key_at <= p.window);
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          const uint32_t u = __shfl_sync(0xffffffffu, key_up[k], src);
          const uint32_t d = __shfl_sync(0xffffffffu, key_down[k], src);
          if (seen) {
            up[k] |= u;
            down[k] |= d;
          }
        }
      }
    }
  }
  if (!live) return;
#pragma unroll
  for (int k = 0; k < kWords; ++k)
    for (uint32_t left = up[k] | down[k]; left; left &= left - 1) {
      const int bit = __ffs(left) - 1, d = 32 * k + bit;
      const float x = !(down[k] >> bit & 1) ? INFINITY : !(up[k] >> bit & 1) ? -INFINITY : NAN;
      if (out) out[d] = Elem<T>::from_f32(Elem<T>::to_f32(out[d]) + x);
      else acc[(d >> 2) * 4 * kTreeRows + (d & 3)] += x;
    }
}

// Warps 0-3 and 4-7 are the softmax of units 0 and 1 (warp w: rows 32 (w % 4)
// .., one row per thread), 8-11 the producers, 12 and 13 the MMA issuers, one
// per unit so that units never wait for one another.  A pair item gives the
// units different heads or row tiles over the same keys; a single one gives both
// the same rows and alternate key tiles, and its accumulators are joined out of
// tensor memory at the end.
// Barriers.  Per slot: full (every producer thread's copies have landed),
// empty (the products of both units that read it are done; the unit that
// reads a single item's slot signals twice).  Per unit: q (its Q tile is
// stored), s (scores done), f (head_dim 64: the scores are read, so the
// next product may overwrite them while P is made), p (P stored), o (P.V
// done), d (all of it done, at the end).  x: the units meet around the join.  A
// waiter is never two phases behind: S(c + 1) needs f(c) or o(c), P(c + 1) is
// stored after o(c), and Q of an item is sent after the last o before it.  Waits
// are bounded; once one runs out the CTA's abort flag ends every role's loop and
// *error_flag gets bit 2.
template <typename T, int D, bool WIN>
__global__ void __launch_bounds__(TreeCfg<D>::kThreads, 1)
tree_attention_kernel(const __grid_constant__ TreeParams p) {
  using C = TreeCfg<D>;
  using Pos = RingPos<C::kSlots>;
  constexpr int kHalf = std::is_same<T, __half>::value;  // fp16 operands
  constexpr bool kFree = D == 64;                        // P has columns of its own
  // fp16's weights are taken 2^7 times as large, which still leaves room for
  // the 2^8 that scores may pass the base by: a weight keeps 11 bits down to
  // 2^-21 of the row's largest (2^-14 without) and counts down to 2^-32.
  constexpr float kLift = kHalf ? 7.f : 0.f;
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t bars = base + C::kBarOff;
  auto bar_full = [&](uint32_t s) { return bars + 8u * s; };
  auto bar_empty = [&](uint32_t s) { return bars + 8u * (C::kSlots + s); };
  auto unit_bar = [&](int u, int i) { return bars + 8u * (2 * C::kSlots + 5 * u + i); };
  auto bar_q = [&](int u) { return unit_bar(u, 0); };
  auto bar_s = [&](int u) { return unit_bar(u, 1); };
  auto bar_f = [&](int u) { return unit_bar(u, 2); };
  auto bar_p = [&](int u) { return unit_bar(u, 3); };
  auto bar_o = [&](int u) { return unit_bar(u, 4); };
  const uint32_t bar_x = unit_bar(2, 0);
  auto bar_d = [&](int u) { return bars + 8u * (2 * C::kSlots + 11 + u); };
  static_assert(8 * (2 * C::kSlots + 13) <= 240, "barriers and flags");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBarOff + 240);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + C::kBarOff + 244);
  volatile int* scrubbed = reinterpret_cast<volatile int*>(smem + C::kBarOff + 248);
  volatile unsigned long long* hits =
      reinterpret_cast<volatile unsigned long long*>(smem + C::kHitOff);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 32) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(bar_full(s), 32 * C::kProducers);
      mbar_init(bar_empty(s), 2);
    }
    for (int u = 0; u < 2; ++u) {
      mbar_init(bar_q(u), kTreeRows);
      mbar_init(bar_s(u), 1);
      mbar_init(bar_f(u), 4);
      mbar_init(bar_p(u), 4);
      mbar_init(bar_o(u), 1);
      mbar_init(bar_d(u), 1);
    }
    mbar_init(bar_x, C::kSoftmax);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *scrubbed = 0;  // 1: some tile of the CTA's items was a hit
    *abort = base & 1023 ? 1 : 0;  // the swizzled tiles need a 1024-byte aligned base
  }
  // A CTA with an item that reaches past the call's vectors, as one of a plan
  // made after the call was captured may, does nothing.
  const int it0 = p.cta_items[blockIdx.x], items_end = p.cta_items[blockIdx.x + 1];
  bool past = false;
  for (int it = it0 + tid; it < items_end; it += C::kThreads) {
    const TreeItem w = p.items[it];
    past |= (long long)w.q0 + w.n > p.tokens || (long long)w.kv0 + w.prefix > p.keys;
  }
  tc_fence_before();
  past = __syncthreads_or(past);
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int it1 = past ? it0 : items_end;
  if (past && tid == 0 && p.error_flag) atomicOr(p.error_flag, 4);

  if (warp >= C::kSoftmax + C::kProducers) {
    // ---- MMA issuers: one thread per unit ----
    const int u = warp - C::kSoftmax - C::kProducers;
    if (lane == 0) {
      const uint32_t tu = tmem + 256 * u;
      const uint64_t qd = sw128_desc(base + u * C::kQBytes);
      Pos at;  // the item's first K slot
      uint32_t cnt = 0, n_q = 0;
      bool ok = true;
      for (int it = it0; it < it1 && ok; ++it) {
        const TreeItem w = p.items[it];
        const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
        const bool pair = w.units == 2;
        const int step = pair ? 1 : 2;
        const int n = pair ? n_tiles : (n_tiles - u + 1) / 2;  // this unit's tiles
        const uint32_t ring = base + C::kRingOff + (w.head_step ? u * C::kHeadBytes : 0);
        auto release = [&](uint32_t slot) {
          umma_commit(bar_empty(slot));
          if (!pair) umma_commit(bar_empty(slot));
        };
        // The copies are writes of the generic proxy that the full barrier
        // has made visible to this thread; the fence orders them before the
        // products that it issues.
        auto scores = [&](uint32_t c, const Pos& k) {  // S(c) = Q K^T
          ok = ok && ws_wait(bar_full(k.slot), k.phase, abort);
          if (c > 0) ok = ok && ws_wait(kFree ? bar_f(u) : bar_o(u), c - 1 & 1, abort);
          if (!ok) return;
          fence_async_smem();
          tc_fence_after();
          const uint64_t kd = sw128_desc(ring + k.slot * C::kSlotBytes);
#pragma unroll
          for (int i = 0; i < D / 16; ++i) {  // 16 dims a step: 32 bytes of a 64-dim atom
            const uint32_t off = ((i >> 2) * kTreeKeys * 128 + 32 * (i & 3)) >> 4;
            mma_ss(tu, qd + off, kd + off, f16_idesc(kTreeKeys, 0, kHalf), i > 0);
          }
          umma_commit(bar_s(u));
          release(k.slot);
        };
        auto values = [&](uint32_t c, const Pos& v, bool first) {  // O += P(c) V
          ok = ok && ws_wait(bar_full(v.slot), v.phase, abort) &&
               ws_wait(bar_p(u), c & 1, abort);
          if (!ok) return;
          fence_async_smem();
          tc_fence_after();
          const uint32_t vb = ring + v.slot * C::kSlotBytes;
          const uint64_t vd = D == 64 ? sw128_desc(vb) : sw128_desc_mn(vb, kTreeKeys * 128);
#pragma unroll
          for (int i = 0; i < kTreeKeys / 16; ++i)  // 16 keys: 8 P columns, 2 KiB of V
            mma_ts(tu + C::kColO, tu + C::kColP + 8 * i, vd + (2048 * i >> 4),
                   f16_idesc(D, 1, kHalf), !first || i > 0);
          umma_commit(bar_o(u));
          release(v.slot);
        };
        if (n > 0) {
          ok = ws_wait(bar_q(u), n_q++ & 1, abort);
          Pos k = at;
          if (!pair && u) k.advance(2);
          if (kFree) scores(cnt, k);
          for (int i = 0; i < n && ok; ++i) {
            Pos v = k, next = k;
            v.advance(1);
            next.advance(2 * step);
            // With P in columns of its own the next scores are made during
            // this tile's softmax; otherwise once its P.V is done.
            if (!kFree) scores(cnt + i, k);
            else if (i + 1 < n) scores(cnt + i + 1, next);
            values(cnt + i, v, i == 0);
            k = next;
          }
          cnt += n;
        }
        const uint32_t end = at.slot + 2 * n_tiles;
        at.phase ^= end / C::kSlots & 1;
        at.slot = end % C::kSlots;
      }
      if (n_q > 0) {
        // Every product and every commit has arrived before the CTA gives its
        // memories back: the last slot's release outlives the roles' waits, and
        // after a failed wait so may products.
        volatile int late = 0;
        umma_commit(bar_d(u));
        if (!ws_wait(bar_d(u), 0, &late)) *abort = 1;
      }
    }
    __syncwarp();
  } else if (warp >= C::kSoftmax) {
    // ---- producers: warp pw gathers keys 32 pw .. of every tile ----
    constexpr int kKpw = kTreeKeys / C::kProducers;
    const int pw = warp - C::kSoftmax;
    Pos at;
    bool ok = true;
    for (int it = it0; it < it1 && ok; ++it) {
      const TreeItem w = p.items[it];
      const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
      const int heads = w.head_step ? 2 : 1;
      int last = INT_MIN;  // the request's last position
      if (WIN) {
        for (int i = lane; i < w.n; i += 32) last = max(last, p.q_positions[w.q0 + i]);
        last = __reduce_max_sync(0xffffffffu, last);
      }
      volatile unsigned long long* hit_word = hits + pw * C::kHitItems + (it - it0) % C::kHitItems;
      if (lane == 0) *hit_word = 0;
      bool hidden = false;  // this lane's next key, by the window, from some token
      auto fetch = [&](int t) {
        const int j = w.lo + t * kTreeKeys + kKpw * pw + lane % kKpw;
        if (t >= n_tiles || j >= w.hi) return -1;
        hidden = WIN && j < w.prefix &&
                 (long long)last - p.kv_positions[w.kv0 + j] > p.window;
        return (int)key_slot(p, w, j);
      };
      int next = fetch(0);
      // chunks: 16-byte pieces per key, consecutive lanes on one key.
      auto tile = [&](int t, auto chunks) {
        constexpr int kCpk = decltype(chunks)::value, kPer = 32 / kCpk, kRounds = kKpw / kPer;
        const int c = lane % kCpk, hh = c / (D / 8), cc = c % (D / 8), sub = lane / kCpk;
        const int slot = next;
        // An infinity or NaN of a V row that only some rows see would reach
        // the others as 0 * V: the warp's keys of this tile are searched for them
        // before they are handed on if one may be hidden (by the tree, if the
        // tile has drafted tokens, or the window).
        const bool guarded =
            w.lo + (t + 1) * kTreeKeys > w.prefix || (WIN && __any_sync(0xffffffffu, hidden));
        next = fetch(t + 1);
        const bool whole = __all_sync(0xffffffffu, slot >= 0);
        // The slots of the keys that this lane copies a piece of, all before
        // the first copy: between the copies each would wait for its shuffle.
        int sl[kRounds];
#pragma unroll
        for (int i = 0; i < kRounds; ++i) sl[i] = __shfl_sync(0xffffffffu, slot, i * kPer + sub);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
          ok = warp_wait(bar_empty(at.slot), at.phase ^ 1, abort);
          if (!ok) return;
          const char* src = static_cast<const char*>(kv ? p.v : p.k) +
                            2 * ((w.head0 + hh) * (kv ? p.v_sh : p.k_sh) + cc * 8);
          const uint32_t stride = (uint32_t)(2 * (kv ? p.v_ss : p.k_ss));
          // The swizzle moves piece cc of key k to cc ^ (k & 7); the keys of
          // a lane differ in a constant, so one XOR each gives its address.
          const uint32_t off = C::kRingOff + at.slot * C::kSlotBytes + hh * C::kHeadBytes +
                               sw_chunk(kTreeKeys, kKpw * pw + sub, cc);
          auto place = [&](int i) { return (off ^ (i * kPer & 7) << 4) + i * kPer * 128; };
          if (whole) {
#pragma unroll
            for (int i = 0; i < kRounds; ++i)
              cp_async16_full(base + place(i), src + (unsigned long long)(uint32_t)sl[i] * stride);
          } else {  // some keys past the end or padding: zeros
#pragma unroll
            for (int i = 0; i < kRounds; ++i)
              cp_async16(base + place(i),
                         src + (unsigned long long)(uint32_t)max(sl[i], 0) * stride,
                         sl[i] < 0 ? 0 : 16);
          }
          if (kv == 1 && guarded) {
            cp_async_commit();
            cp_async_wait<0>();
            bool hit = false;
            for (int i = 0; i < kRounds; ++i) {  // the pieces that this thread copied
              uint4* v = reinterpret_cast<uint4*>(smem + place(i));
              uint4 x = *v;
              if (scrub<kHalf>(x)) {
                *v = x;
                hit = true;
              }
            }
            if (__any_sync(0xffffffffu, hit) && lane == 0) {
              *hit_word |= 1ull << t / tiles_per_hit(n_tiles);
              *scrubbed = 1;
            }
            fence_async_smem();
            mbar_arrive(bar_full(at.slot));
          } else {
            cp_async_arrive(bar_full(at.slot));
          }
          at.advance(1);
        }
      };
      for (int t = 0; t < n_tiles && ok; ++t) {
        if (heads * (D / 8) == 16) tile(t, std::integral_constant<int, 16>());
        else tile(t, std::integral_constant<int, 8>());
      }
    }
    cp_async_commit();
    cp_async_wait<0>();
  } else {
    // ---- softmax ----
    const int u = warp >> 2, r = tid & (kTreeRows - 1);
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's TMEM lanes
    const uint32_t tu = tmem + 256 * u + lanes;
    float2* rows = reinterpret_cast<float2*>(smem + C::kRowOff);
    uint32_t cnt = 0, n_x = 0;
    // Copies this thread's row of an item's Q: for the first item here, for
    // the next one once the last scores of the one before are made.
    auto load_q = [&](int it) {
      if (it < it1) {
        const TreeItem w = p.items[it];
        const int row = (w.tile0 + u * w.tile_step) * kTreeRows + r;
        const int i = row / p.group, h = (w.head0 + u * w.head_step) * p.group + row - i * p.group;
        if (i < w.n) {
          const T* src = static_cast<const T*>(p.q) + (long long)(w.q0 + i) * p.q_st +
                         (long long)h * p.q_sh;
#pragma unroll
          for (int c = 0; c < D / 8; ++c)
            cp_async16_full(base + u * C::kQBytes + sw_chunk(kTreeRows, r, c), src + 8 * c);
        }
      }
      cp_async_commit();
    };
    // Hands it on: before the epilogue of the item before, which the first
    // scores then run beside.
    auto send_q = [&](int it) {
      if (it >= it1) return;
      const TreeItem w = p.items[it];
      const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
      cp_async_wait<0>();
      if (w.units == 2 || n_tiles > u) {
        fence_async_smem();
        mbar_arrive(bar_q(u));
      }
    };
    load_q(it0);
    send_q(it0);
    for (int it = it0; it < it1; ++it) {
      float m = -INFINITY, l = 0.f;
      bool ok = true, warp_live;
      int n;  // this unit's tiles
      {
        const TreeItem w = p.items[it];
        const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
        const bool pair = w.units == 2;
        n = pair ? n_tiles : (n_tiles - u + 1) / 2;
        const int row0 = (w.tile0 + u * w.tile_step) * kTreeRows, i = (row0 + r) / p.group;
        warp_live = row0 + (warp & 3) * 32 < w.n * p.group;
        const int pos = i < w.n && p.window >= 0 ? p.q_positions[w.q0 + i] : 0;
        const unsigned long long word = i < w.n ? row_mask(p, w, p.tree_mask[w.q0 + i], pos) : 0;
        if (n == 0) load_q(it + 1);
        const int last = WIN ? __reduce_max_sync(0xffffffffu, pos) : 0;
        for (int v = 0; v < n && ok; ++v) {
          const uint32_t c = cnt + v;
          const int j0 = w.lo + (pair ? v : 2 * v + u) * kTreeKeys;
          bool old = false;  // the window hides a key of the tile from a row of the warp
          if (WIN && j0 + kTreeKeys <= w.prefix) {
            const int* kp = p.kv_positions + w.kv0 + j0 + lane;
            const int oldest = min(min(kp[0], kp[32]), min(kp[64], kp[96]));
            old = __any_sync(0xffffffffu, (long long)last - oldest > p.window);
          }
          ok = warp_wait(bar_s(u), c & 1, abort);
          if (!ok) break;
          if (v == n - 1) load_q(it + 1);
          if (warp_live) {
            tc_fence_after();
            // (The kernel without windows keeps the run-time tests of one, here and
            // in the helpers: compiled without them its loop is 2 to 4 % slower.)
            const bool tail = j0 + kTreeKeys > w.prefix;
            if (WIN ? tail || old : tail || p.window >= 0) {
              // Hidden keys get a score of -inf in tensor memory, so that the
              // ordinary path below has no mask (and no registers for one).
#pragma unroll 1
              for (int b = 0; b < kTreeKeys; b += 64) {
                const unsigned long long seen = seen64(p, w, word, i, pos, j0 + b, lane);
                if (__all_sync(0xffffffffu, seen == ~0ull)) continue;
#pragma unroll 1
                for (int q = 0; q < 64; q += 32) {
                  const uint32_t bits = (uint32_t)(seen >> q);
                  float x[32];
                  tmem_ld32_sync(tu + b + q, x);
                  uint32_t y[2][16];
#pragma unroll
                  for (int k = 0; k < 32; ++k)
                    y[k / 16][k % 16] = __float_as_uint(bits >> k & 1 ? x[k] : -INFINITY);
                  tmem_st16_async(tu + b + q, y[0]);
                  tmem_st16_async(tu + b + q + 16, y[1]);
                }
              }
              tmem_st_wait();
            }
          }
          if (warp_live) {
            // The scores are read twice, for the maximum and for P: more than
            // 64 of them in registers cost spills.
            float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int b = 0; b < kTreeKeys; b += 64) {
              float s[64];
              tmem_ld64_sync(tu + b, s);
#pragma unroll
              for (int k = 0; k < 64; k += 2)
                m4[k >> 1 & 3] = max3_nan(m4[k >> 1 & 3], s[k], s[k + 1]);
            }
            const float bm =
                max3_nan(max3_nan(m4[0], m4[1], m4[2]), m4[3], -INFINITY) * p.scale_log2;
            // The base only moves when the tile exceeds it by 2^8; then l and
            // O are rescaled.
            float alpha = 1.f;
            bool rescale = false;
            if (bm > m + kStaleMax || (m == -INFINITY && bm != -INFINITY)) {
              rescale = m != -INFINITY;
              alpha = rescale ? fast_exp2(m - bm) : 0.f;
              m = bm;
            }
            const float nb = m == -INFINITY ? 0.f : kLift - m;
            const f32x2 scale2 = f2_pack(p.scale_log2, p.scale_log2), nb2 = f2_pack(nb, nb);
            f32x2 sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
            // The last columns come first: P overwrites the second half of its
            // scores at head_dim 128, each piece of it columns that are read.
#pragma unroll
            for (int b = kTreeKeys - 32; b >= 0; b -= 32) {
              float s[32];
              tmem_ld32_sync(tu + b, s);
              if (kFree && b == 0) {  // every score of the tile is read
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar_f(u));
              }
              uint32_t pk[16];
#pragma unroll
              for (int k = 0; k < 32; k += 2) {
                float x0, x1;
                const f32x2 x = f2_fma(f2_pack(s[k], s[k + 1]), scale2, nb2);
                if (kPoly >> (k / 2) & 1) {
                  exp2_pair(x, x0, x1);
                } else {
                  f2_unpack(x, x0, x1);
                  x0 = fast_exp2(x0);
                  x1 = fast_exp2(x1);
                }
                sum[k >> 1 & 1] = f2_add(sum[k >> 1 & 1], f2_pack(x0, x1));
                pk[k / 2] = pack2<T>(x0, x1);
              }
              // P's columns, and O's, are free once the product before is done
              // (with P over the scores S(c) came after it).
              if (b == kTreeKeys - 32 && kFree && c > 0) ok = warp_wait(bar_o(u), c - 1 & 1, abort);
              tmem_st16_async(tu + C::kColP + b / 2, pk);
            }
            tmem_st_wait();
            float l0, l1;
            f2_unpack(f2_add(sum[0], sum[1]), l0, l1);
            l = l * alpha + (l0 + l1);
            if (!(bm < INFINITY)) l = NAN;  // an infinite or NaN score: the row is NaN
            if (__any_sync(0xffffffffu, rescale)) {
              tc_fence_after();
#pragma unroll
              for (int d = 0; d < D; d += 32) {
                float o[32];
                tmem_ld32_sync(tu + C::kColO + d, o);
                uint32_t z[32];
#pragma unroll
                for (int k = 0; k < 32; ++k) z[k] = __float_as_uint(o[k] * alpha);
                tmem_st32_sync(tu + C::kColO + d, z);
              }
            }
            tc_fence_before();
          } else if (kFree) {
            // A warp without rows keeps the others' pace: with S(c + 1) made
            // early it would otherwise arrive on p twice before they do once.
            if (lane == 0) mbar_arrive(bar_f(u));
            if (c > 0) ok = warp_wait(bar_o(u), c - 1 & 1, abort);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar_p(u));
        }
      }
      if (!ok) break;
      m -= kLift;  // the base that P, l and O are in
      // The item is read, and the row worked out, again: over the tiles they
      // would only hold registers.
      const TreeItem w = p.items[it];
      const bool pair = w.units == 2;
      const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
      const int row = (w.tile0 + u * w.tile_step) * kTreeRows + r, i = row / p.group;
      const int head = w.head0 + u * w.head_step, h = head * p.group + row - i * p.group;
      const bool live = i < w.n;
      const float sink = live && p.sinks ? p.sinks[h] : -INFINITY;  // on its way over the wait
      cnt += n;
      if (n > 0 && !warp_wait(bar_o(u), cnt - 1 & 1, abort)) break;
      send_q(it + 1);
      tc_fence_after();
      float f[2] = {1.f, 0.f};
      if (!pair) {  // the two units' rows meet
        rows[u * kTreeRows + r] = make_float2(m, l);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_x);
        if (!warp_wait(bar_x, n_x++ & 1, abort)) break;
        tc_fence_after();
        const float2 a = rows[r], b = rows[kTreeRows + r];
        m = fmaxf(a.x, b.x);
        const float top = m == -INFINITY ? 0.f : m;
        f[0] = fast_exp2(a.x - top);
        f[1] = fast_exp2(b.x - top);
        l = a.y * f[0] + b.y * f[1];
      }
      if (warp_live) {
        const bool direct = w.partial < 0;
        const long long part = (long long)w.partial + (pair ? u : 0);
        float* acc = p.part_acc + part * D * kTreeRows + 4 * r;
        RowEnd e = {0.f, 0.f};
        if (direct) e = row_end(sink, m, l);
        T* dst = static_cast<T*>(p.out) + (long long)(w.q0 + i) * p.o_st + (long long)h * p.o_sh;
        // A pair's units write all their columns, a single item's half each.
        const int d0 = pair ? 0 : u * (D / 2), d1 = pair ? D : d0 + D / 2;
        for (int d = d0; d < d1; d += 32) {
          float o[32];
          __syncwarp();
          tmem_ld32_sync(tmem + lanes + (pair ? 256 * u : 0) + C::kColO + d, o);
          if (!pair) {
            float o1[32];
            if (n_tiles > 1) tmem_ld32_sync(tmem + lanes + 256 + C::kColO + d, o1);
#pragma unroll
            for (int k = 0; k < 32; ++k) o[k] = o[k] * f[0] + (n_tiles > 1 ? o1[k] * f[1] : 0.f);
          }
          if (!live) continue;
          if (direct) {
#pragma unroll
            for (int k = 0; k < 32; k += 8) {
              uint4 x;
              x.x = pack2<T>(o[k] * e.scale, o[k + 1] * e.scale);
              x.y = pack2<T>(o[k + 2] * e.scale, o[k + 3] * e.scale);
              x.z = pack2<T>(o[k + 4] * e.scale, o[k + 5] * e.scale);
              x.w = pack2<T>(o[k + 6] * e.scale, o[k + 7] * e.scale);
              *reinterpret_cast<uint4*>(dst + d + k) = x;
            }
          } else {
#pragma unroll
            for (int k = 0; k < 32; k += 4)
              *reinterpret_cast<float4*>(acc + (d + k) * kTreeRows) =
                  make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
          }
        }
        unsigned long long hit = 0;  // of all producers
        if (*scrubbed)
          for (int k = 0; k < C::kProducers; ++k)
            hit |= hits[k * C::kHitItems + (it - it0) % C::kHitItems];
        if (hit) {
          const long long at = live && p.window >= 0 ? p.q_positions[w.q0 + i] : 0;
          restore<T, D>(p, it, hit, tiles_per_hit(n_tiles),
                        live ? row_mask(p, w, p.tree_mask[w.q0 + i], at) : 0, at, head, live,
                        direct ? dst : nullptr, direct ? nullptr : acc, d0, d1);
        }
        if (live && (pair || u == 0)) {
          if (!direct) {
            reinterpret_cast<float2*>(p.part_ml)[part * kTreeRows + r] = make_float2(m, l);
          } else if (p.lse) {
            p.lse[(long long)(w.q0 + i) * p.num_q_heads + h] = e.lse;
          }
        }
      }
      tc_fence_before();  // O's reads before the next item's products
      if (!pair) {        // of either unit
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_x);
        if (!warp_wait(bar_x, n_x++ & 1, abort)) break;
      }
    }
    cp_async_wait<0>();  // a next item's Q, if a failed wait ended the loop
  }
  tc_fence_before();
  __syncthreads();
  pdl_launch_dependents();
  if (tid == 0 && *abort && p.error_flag) atomicOr(p.error_flag, 2);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

struct TreeMerge {  // 8 int32
  int q0, n, head0, tile0, steps;  // steps: head_step | tile_step << 1 | units << 2
  int first, count, unused;
};

// Joins the pieces of units that were cut.  A block takes kRows rows of one
// unit, a thread four columns of a row; neighbouring threads have
// neighbouring rows, as the partial results lie.
constexpr int kMergeThreads = 256;
template <int D>
constexpr int merge_rows() { return kMergeThreads / (D / 4); }

template <typename T, int D>
__global__ void __launch_bounds__(kMergeThreads)
tree_merge_kernel(const TreeParams p, const TreeMerge* merges) {
  constexpr int kRows = merge_rows<D>();
  const TreeMerge g = merges[blockIdx.x];
  // Before any return: once every block has left, the stream goes on, and the
  // pieces' kernel has to be done by then.
  pdl_wait();
  const int u = blockIdx.y / (kTreeRows / kRows);
  const int r = blockIdx.y % (kTreeRows / kRows) * kRows + threadIdx.x % kRows;
  const int d = threadIdx.x / kRows * 4;
  if (u >= g.steps >> 2) return;
  const int head = g.head0 + u * (g.steps & 1);
  const int row = (g.tile0 + u * (g.steps >> 1 & 1)) * kTreeRows + r;
  const int i = row / p.group, h = head * p.group + row % p.group;
  if (i >= g.n || g.q0 + g.n > p.tokens) return;
  const float2* ml = reinterpret_cast<const float2*>(p.part_ml) +
                     ((long long)g.first + u) * kTreeRows + r;
  const float* acc = p.part_acc + (((long long)g.first + u) * D + d) * kTreeRows + 4 * r;
  float m = -INFINITY;
#pragma unroll 4
  for (int s = 0; s < g.count; ++s) m = fmaxf(m, ml[s * kTreeUnits * kTreeRows].x);
  const float base = m == -INFINITY ? 0.f : m;
  float den = 0.f, num[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < g.count; ++s) {
    const float2 x = ml[s * kTreeUnits * kTreeRows];
    const float4 a =
        *reinterpret_cast<const float4*>(acc + (long long)s * kTreeUnits * D * kTreeRows);
    const float f = fast_exp2(x.x - base);
    den += x.y * f;
    num[0] += a.x * f;
    num[1] += a.y * f;
    num[2] += a.z * f;
    num[3] += a.w * f;
  }
  const RowEnd e = row_end(p.sinks ? p.sinks[h] : -INFINITY, m, den);
  T* o = static_cast<T*>(p.out) + (long long)(g.q0 + i) * p.o_st + (long long)h * p.o_sh + d;
  *reinterpret_cast<uint2*>(o) = make_uint2(pack2<T>(num[0] * e.scale, num[1] * e.scale),
                                            pack2<T>(num[2] * e.scale, num[3] * e.scale));
  if (p.lse && d == 0) p.lse[(long long)(g.q0 + i) * p.num_q_heads + h] = e.lse;
}

template <typename T, int D, bool WIN>
int launch_items(const TreeParams& p, int n_ctas, cudaStream_t s) {
  using C = TreeCfg<D>;
  if (cudaFuncSetAttribute(tree_attention_kernel<T, D, WIN>,
                           cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess)
    return AKV_ERR_CUDA;
  tree_attention_kernel<T, D, WIN><<<n_ctas, C::kThreads, C::kSmem, s>>>(p);
  return AKV_OK;
}

template <typename T, int D>
int launch_tree(const TreeParams& p, int n_ctas, const TreeMerge* merges, int n_merges,
                cudaStream_t s) {
  // With a window, tiles that no row loses a key of take the ordinary way: 128
  // requests of 2,040 keys and 8 tokens 160 us (all tiles searched and masked: 255,
  // without a window 144).  In one kernel that costs the others 4 to 9 %.
  const int status = p.window >= 0 ? launch_items<T, D, true>(p, n_ctas, s)
                                   : launch_items<T, D, false>(p, n_ctas, s);
  if (status != AKV_OK) return status;
  if (n_merges > 0 &&
      launch_pdl(tree_merge_kernel<T, D>, dim3(n_merges, kTreeUnits * kTreeRows / merge_rows<D>()),
                 dim3(kMergeThreads), 0, s, p, merges) != cudaSuccess)
    return AKV_ERR_CUDA;
  return launch_status();
}

}  // namespace
}  // namespace akv

extern "C" int32_t akv_tree_attention_units(void) { return akv::kTreeUnits; }

extern "C" int64_t akv_tree_attention_args_bytes(void) { return sizeof(akv_tree_attention_args); }

extern "C" int akv_tree_attention(const akv_tree_attention_args* args, void* stream) {
  AKV_NVTX_RANGE("akv_tree_attention");
  using namespace akv;
  if (args == nullptr) return AKV_ERR_INVALID;
  const akv_tree_attention_args& x = *args;
  if (x.num_kv_heads <= 0 || x.num_q_heads <= 0 || x.num_q_heads > INT32_MAX / 64 ||
      x.num_q_heads % x.num_kv_heads || x.n_ctas < 0 || x.n_ctas > INT32_MAX || x.n_merges < 0 ||
      x.n_merges > INT32_MAX || x.tokens < 0 || x.keys < 0 || !((float)x.sm_scale > 0.f) ||
      !((float)x.sm_scale * kLog2e < INFINITY) ||  // a hidden score of -inf stays -inf
      x.num_slots <= 0 || x.num_slots > INT32_MAX || (x.dtype != AKV_F16 && x.dtype != AKV_BF16))
    return AKV_ERR_INVALID;
  if (x.head_dim != 64 && x.head_dim != 128) return AKV_ERR_UNSUPPORTED;
  if (x.n_ctas == 0) return AKV_OK;
  if (!x.q || !x.k_pool || !x.v_pool || !x.draft_slots || !x.tree_mask || !x.items ||
      !x.cta_items || !x.out || !x.kv_indices ||
      (x.n_merges > 0 && (!x.merges || !x.partial_acc || !x.partial_ml)) ||
      (x.window >= 0 && (!x.q_positions || !x.kv_positions)))
    return AKV_ERR_INVALID;
  const void* bases[] = {x.q, x.k_pool, x.v_pool, x.out};
  for (const void* b : bases)
    if (reinterpret_cast<uintptr_t>(b) & 15) return AKV_ERR_INVALID;
  if (x.k_stride_slot < 0 || x.v_stride_slot < 0 || x.k_stride_slot >= (1ll << 31) ||
      x.v_stride_slot >= (1ll << 31))
    return AKV_ERR_INVALID;  // bytes between slots in 32 bits
  const int64_t strides[] = {x.q_stride_token, x.q_stride_head,    x.k_stride_slot,
                             x.k_stride_head,  x.v_stride_slot,    x.v_stride_head,
                             x.out_stride_token, x.out_stride_head};
  for (int64_t s : strides)
    if (s % 8) return AKV_ERR_INVALID;  // 16-byte rows
  TreeParams p{x.q, x.q_stride_token, x.q_stride_head, x.k_pool, x.v_pool, x.k_stride_slot,
               x.k_stride_head, x.v_stride_slot, x.v_stride_head, x.num_slots, x.tokens, x.keys,
               x.kv_indices,
               x.draft_slots, reinterpret_cast<const unsigned long long*>(x.tree_mask),
               x.q_positions, x.kv_positions, x.window, x.sinks, (float)x.sm_scale * kLog2e,
               (int)(x.num_q_heads / x.num_kv_heads), (int)x.num_q_heads,
               reinterpret_cast<const TreeItem*>(x.items), x.cta_items, x.partial_acc,
               x.partial_ml, x.out, x.out_stride_token, x.out_stride_head, x.lse, x.error_flag};
  const TreeMerge* m = reinterpret_cast<const TreeMerge*>(x.merges);
  const int n = (int)x.n_ctas, nm = (int)x.n_merges;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (x.dtype == AKV_BF16)
    return x.head_dim == 64 ? launch_tree<__nv_bfloat16, 64>(p, n, m, nm, s)
                            : launch_tree<__nv_bfloat16, 128>(p, n, m, nm, s);
  return x.head_dim == 64 ? launch_tree<__half, 64>(p, n, m, nm, s)
                          : launch_tree<__half, 128>(p, n, m, nm, s);
}
