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
// 64-key tiles of one request for up to `units` (head, row tile) pairs; the
// host cuts the flat list of all key tiles into equal runs, one per CTA, and
// a second kernel joins the pieces of requests that were cut.

#include <type_traits>

#include "tcgen05.cuh"

namespace akv {
namespace {

constexpr int kTreeRows = 128;
constexpr int kTreeKeys = 64;

struct TreeItem {   // 12 int32
  int q0, n;        // first drafted token of the request, and their number
  int kv0, prefix;  // first cached key, and their number
  int lo, hi;       // keys [lo, hi) of prefix ++ drafted
  int head0, tile0; // unit u: head head0 + u * head_step, row tile tile0 + u * tile_step
  int head_step, tile_step;
  int units;
  int partial;      // first partial result (one per unit of the CTA), or -1
};

struct TreeParams {
  const void* q;
  long long q_st, q_sh;
  const void* k;
  const void* v;
  long long k_ss, k_sh, v_ss, v_sh;
  long long num_slots;
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
  float* part_acc;  // [partials][kTreeRows][D]
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

// Visible drafted tokens of token i: its mask, without those the window hides.
__device__ __forceinline__ unsigned long long row_mask(const TreeParams& p, const TreeItem& w,
                                                       int i) {
  unsigned long long m = p.tree_mask[w.q0 + i];
  if (w.n < 64) m &= (1ull << w.n) - 1;
  if (p.window >= 0) {
    const long long pos = p.q_positions[w.q0 + i];
    for (unsigned long long left = m; left; left &= left - 1) {
      const int j = __ffsll((long long)left) - 1;
      if (pos - p.q_positions[w.q0 + j] > p.window) m &= ~(1ull << j);
    }
  }
  return m;
}

// Joins the sink to a row's maximum m (base 2) and sum l: `scale` is the
// factor of the accumulator in the output, lse the natural logarithm.  The
// maximum takes the sink in, so neither a sink far above every score nor one
// of a row without keys overflows.
struct RowEnd {
  float scale, lse;
};
__device__ __forceinline__ RowEnd row_end(const float* sinks, int h, float m, float l) {
  const float sink = sinks ? sinks[h] * kLog2e : -INFINITY;
  const float top = fmaxf(m, sink), base = top == -INFINITY ? 0.f : top;
  const float f = fast_exp2(m - base);
  const float den = l * f + fast_exp2(sink - base);
  RowEnd e;
  e.scale = den > 0.f ? f / den : 0.f;
  e.lse = den > 0.f ? (base + log2f(den)) * kLn2 : -INFINITY;
  return e;
}

// ws_wait by a whole warp, which then takes one way.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort) {
  return __all_sync(0xffffffffu, ws_wait(bar, parity, abort));
}

// Key j visible to a row: its token's mask word and position.
__device__ __forceinline__ bool key_seen(const TreeParams& p, const TreeItem& w,
                                         unsigned long long mask, long long pos, int j) {
  if (j >= w.prefix) return mask >> (j - w.prefix) & 1;
  return p.window < 0 || pos - p.kv_positions[w.kv0 + j] <= p.window;
}

constexpr int tree_units(int head_dim) { return head_dim == 64 ? 2 : 1; }

// Two CTAs per SM, each with 256 tensor-memory columns: per unit, SB score
// buffers of 64 columns and the accumulator of D (P overwrites its scores).
// K and V tiles of 64 keys alternate in a ring of 16 KiB slots: at head_dim 64
// two heads' rows (256 contiguous bytes a key in the usual pools), at 128 one.
// 256-byte pieces gathered by cp.async from several CTAs per SM reach the
// copy rate on random slots (6.9 TB/s in a bare gather, against 4.9 for
// 128-byte pieces and 4.9 for TMA row gathers, whose issue is the limit).
template <int D>
struct TreeCfg {
  static constexpr int kUnits = tree_units(D);
  static constexpr int kBuffers = D == 64 ? 1 : 2;   // score buffers per unit
  static constexpr int kSoftmax = 4 * kUnits;        // warps
  static constexpr int kProducers = 2;               // warps
  static constexpr int kThreads = 32 * (kSoftmax + kProducers + kUnits);
  static constexpr int kHeadBytes = kTreeKeys * D * 2;  // one head's rows of a tile
  static constexpr int kSlotBytes = 16384;
  static constexpr int kSlots = 5;
  static constexpr int kAhead = 3;                   // slots requested before the oldest is awaited
  static constexpr int kQBytes = kTreeRows * D * 2;
  static constexpr int kRingOff = kUnits * kQBytes;
  static constexpr int kBarOff = kRingOff + kSlots * kSlotBytes;
  static constexpr int kSmem = kBarOff + 256;
  static constexpr int kUnitCols = 256 / kUnits;
  static constexpr int kColO = kUnitCols - D;
  static_assert(kHeadBytes * kUnits == kSlotBytes || kUnits == 1, "slot holds every unit's head");
  static_assert(kAhead <= kSlots - 2, "a slot is signalled before its successors wait for room");
};

// Warps: 4 per unit run its softmax (warp w: rows 32 (w % 4) ..), then two
// producers, then one MMA issuer per unit, so that units never wait for one
// another.  Per slot: full (every producer thread's copies have landed), empty
// (each unit's MMAs that read it are done).  Per unit: q (its Q tile is
// stored), s[b] (scores done), p[b] (P stored), o (every P.V), done (the last
// P.V of an item).  Waits are bounded; once one runs out the CTA's abort
// flag ends every role's loop and *error_flag gets bit 2.
template <typename T, int D>
__global__ void __launch_bounds__(TreeCfg<D>::kThreads, 2)
tree_attention_kernel(const TreeParams p) {
  using C = TreeCfg<D>;
  constexpr int U = C::kUnits, SB = C::kBuffers;
  constexpr int kHalf = std::is_same<T, __half>::value;  // fp16 operands
  extern __shared__ __align__(1024) unsigned char smem[];
  const uint32_t base = smem_u32(smem);
  const uint32_t bars = base + C::kBarOff;
  auto bar_full = [&](uint32_t s) { return bars + 8u * s; };
  auto bar_empty = [&](uint32_t s) { return bars + 8u * (C::kSlots + s); };
  constexpr int kUnitBars = 3 + 2 * SB;
  auto unit_bar = [&](int u, int i) { return bars + 8u * (2 * C::kSlots + u * kUnitBars + i); };
  auto bar_q = [&](int u) { return unit_bar(u, 0); };
  auto bar_o = [&](int u) { return unit_bar(u, 1); };
  auto bar_done = [&](int u) { return unit_bar(u, 2); };
  auto bar_s = [&](int u, uint32_t b) { return unit_bar(u, 3 + b); };
  auto bar_p = [&](int u, uint32_t b) { return unit_bar(u, 3 + SB + b); };
  static_assert(8 * (2 * C::kSlots + U * kUnitBars) + 16 <= 256, "barriers and flags");
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::kBarOff + 240);
  volatile int* abort = reinterpret_cast<volatile int*>(smem + C::kBarOff + 244);
  volatile int* scrubbed = reinterpret_cast<volatile int*>(smem + C::kBarOff + 248);

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(tmem_slot)),
                 "r"(256));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (tid == 32) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(bar_full(s), 32 * C::kProducers);
      mbar_init(bar_empty(s), U);
    }
    for (int u = 0; u < U; ++u) {
      mbar_init(bar_q(u), kTreeRows);
      mbar_init(bar_o(u), 1);
      mbar_init(bar_done(u), 1);
      for (int b = 0; b < SB; ++b) {
        mbar_init(bar_s(u, b), 1);
        mbar_init(bar_p(u, b), 4);
      }
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    *abort = base & 1023 ? 1 : 0;  // the swizzled tiles need a 1024-byte aligned base
    *scrubbed = 0;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  const int it0 = p.cta_items[blockIdx.x], it1 = p.cta_items[blockIdx.x + 1];

  if (warp >= C::kSoftmax + C::kProducers) {
    // ---- one MMA issuer per unit ----
    if (lane == 0) {
      const int u = warp - C::kSoftmax - C::kProducers;
      const uint32_t tu = tmem + u * C::kUnitCols;
      const uint32_t sq = base + u * C::kQBytes;
      uint32_t seq = 0, cnt = 0, items = 0;  // slots; this unit's tiles and items so far
      for (int it = it0; it < it1; ++it) {
        const TreeItem w = p.items[it];
        const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
        if (u >= w.units) {  // idle: give the slots back
          bool ok = true;
          for (int t = 0; t < 2 * n_tiles && ok; ++t, ++seq) {
            ok = ws_wait(bar_full(seq % C::kSlots), seq / C::kSlots & 1, abort);
            if (ok) mbar_arrive(bar_empty(seq % C::kSlots));
          }
          if (!ok) break;
          continue;
        }
        if (!ws_wait(bar_q(u), items & 1, abort)) break;
        const uint32_t head = w.head_step ? u * C::kHeadBytes : 0;
        auto scores = [&](uint32_t c, uint32_t sk) {  // S(c) = Q K^T
          tc_fence_after();
          const uint32_t kb = base + C::kRingOff + sk % C::kSlots * C::kSlotBytes + head;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t off = 32u * (k & 3);
            mma_ss(tu + c % SB * kTreeKeys,
                   sw128_desc(sq + (k >> 2) * kTreeRows * 128 + off),
                   sw128_desc(kb + (k >> 2) * kTreeKeys * 128 + off),
                   f16_idesc(kTreeKeys, 0, kHalf), k > 0);
          }
          umma_commit(bar_s(u, c % SB));
          umma_commit(bar_empty(sk % C::kSlots));
        };
        auto values = [&](uint32_t c, uint32_t sv, bool first, bool last) {  // O += P(c) V
          tc_fence_after();
          const uint32_t vb = base + C::kRingOff + sv % C::kSlots * C::kSlotBytes + head;
#pragma unroll
          for (int k = 0; k < kTreeKeys / 16; ++k) {  // 16 keys: 8 P columns, 2 KiB of V
            const uint64_t vd = D == 64 ? sw128_desc(vb + 2048 * k)
                                        : sw128_desc_mn(vb + 2048 * k, kTreeKeys * 128);
            mma_ts(tu + C::kColO, tu + c % SB * kTreeKeys + 8 * k, vd, f16_idesc(D, 1, kHalf),
                   !first || k > 0);
          }
          umma_commit(bar_o(u));
          umma_commit(bar_empty(sv % C::kSlots));
          if (last) umma_commit(bar_done(u));
        };
        bool ok = true;
        // With two score buffers S(t) is issued before P(t-1).V(t-1), so the
        // softmax never waits for a product; with one, after it is done.
        for (int t = 0; t < n_tiles + SB - 1 && ok; ++t) {
          if (t < n_tiles) {
            const uint32_t sk = seq + 2 * t;
            ok = ws_wait(bar_full(sk % C::kSlots), sk / C::kSlots & 1, abort);
            // The buffer's last product is done: of SB tiles before or, as an
            // item begins, the last one of the item before (all were issued).
            if (ok && t >= SB) ok = ws_wait(bar_o(u), cnt + t - SB & 1, abort);
            if (ok && t == 0 && cnt > 0) ok = ws_wait(bar_o(u), cnt - 1 & 1, abort);
            if (!ok) break;
            scores(cnt + t, sk);
          }
          const int v = t - (SB - 1);
          if (v >= 0) {
            const uint32_t c = cnt + v, sv = seq + 2 * v + 1;
            ok = ws_wait(bar_full(sv % C::kSlots), sv / C::kSlots & 1, abort) &&
                 ws_wait(bar_p(u, c % SB), c / SB & 1, abort);
            if (!ok) break;
            values(c, sv, v == 0, v == n_tiles - 1);
          }
        }
        if (!ok) break;
        seq += 2 * n_tiles;
        cnt += n_tiles;
        ++items;
      }
    }
    __syncwarp();
  } else if (warp >= C::kSoftmax) {
    // ---- producers: warp pw gathers keys 32 pw .. of every tile ----
    const int pw = warp - C::kSoftmax;
    static_assert(kTreeKeys == 32 * C::kProducers, "one key per producer lane");
    uint32_t seq = 0;
    // Signals slot `s` (its copies have landed); a V slot of a guarded tile
    // is first searched for infinities and NaN, which P = 0 would not mask.
    uint32_t guard = 0;  // bit a: the slot requested a slots ago is a guarded V tile
    int cpk = 0;         // 16-byte chunks per key of the current item, and of guarded slots
    auto signal = [&](uint32_t s, bool guarded, int chunks) {
      if (guarded) {
        unsigned char* tile = smem + C::kRingOff + s % C::kSlots * C::kSlotBytes;
        const int per = 32 / chunks;
        for (int i = 0; i < 32 / per; ++i) {
          const int key = 32 * pw + i * per + lane / chunks, c = lane % chunks;
          uint4* at = reinterpret_cast<uint4*>(tile + c / (D / 8) * C::kHeadBytes +
                                               sw_chunk(kTreeKeys, key, c % (D / 8)));
          uint4 x = *at;
          uint32_t* e = reinterpret_cast<uint32_t*>(&x);
          bool hit = false;
          constexpr uint32_t kExp = kHalf ? 0x7c00u : 0x7f80u;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if ((e[k] & kExp) == kExp) { e[k] &= 0xffff0000u; hit = true; }
            if ((e[k] >> 16 & kExp) == kExp) { e[k] &= 0xffffu; hit = true; }
          }
          if (hit) {
            *at = x;
            *scrubbed = 1;
          }
        }
      }
      fence_async_smem();
      mbar_arrive(bar_full(s % C::kSlots));
    };
    int old_cpk = 0;
    bool ok = true;
    for (int it = it0; it < it1; ++it) {
      const TreeItem w = p.items[it];
      const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
      cpk = (w.head_step ? w.units : 1) * (D / 8);
      auto fetch = [&](int t) {
        const int j = w.lo + t * kTreeKeys + 32 * pw + lane;
        return t < n_tiles && j < w.hi ? (int)key_slot(p, w, j) : -1;
      };
      int next = fetch(0);
      for (int t = 0; t < n_tiles; ++t) {
        const int slot = next;
        next = fetch(t + 1);
        const bool guarded = p.window >= 0 || w.lo + (t + 1) * kTreeKeys > w.prefix;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv, ++seq) {
          if (!warp_wait(bar_empty(seq % C::kSlots), (seq / C::kSlots & 1) ^ 1, abort)) {
            ok = false;
            break;
          }
          const uint32_t dst = base + C::kRingOff + seq % C::kSlots * C::kSlotBytes;
          const T* pool = static_cast<const T*>(kv ? p.v : p.k) +
                          w.head0 * (kv ? p.v_sh : p.k_sh);
          const long long ss = kv ? p.v_ss : p.k_ss, sh = kv ? p.v_sh : p.k_sh;
          auto copy = [&](auto chunks) {
            constexpr int kCpk = decltype(chunks)::value, kPer = 32 / kCpk;
            const int c = lane % kCpk, hh = c / (D / 8), cc = c % (D / 8);
            const T* src = pool + hh * sh + cc * 8;
#pragma unroll
            for (int i = 0; i < 32 / kPer; ++i) {
              const int kk = i * kPer + lane / kCpk, key = 32 * pw + kk;
              const int sl = __shfl_sync(0xffffffffu, slot, kk);
              cp_async16(dst + hh * C::kHeadBytes + sw_chunk(kTreeKeys, key, cc),
                         src + (sl < 0 ? 0 : sl) * ss, sl < 0 ? 0 : 16);
            }
          };
          if (cpk == 16) copy(std::integral_constant<int, 16>());
          else copy(std::integral_constant<int, 8>());
          cp_async_commit();
          guard = guard << 1 | (uint32_t)(kv && guarded);
          if (seq >= C::kAhead - 1) {
            cp_async_wait<C::kAhead - 1>();
            const uint32_t ago = C::kAhead - 1;
            // The slot of `ago` requests before: of this item, or of the one before it.
            signal(seq - ago, guard >> ago & 1, 2 * t + kv >= (int)ago ? cpk : old_cpk);
          }
        }
        if (!ok) break;
      }
      if (!ok) break;
      // An item has at least one tile (two slots), so the slots still to be
      // signalled are of the current item and, for one of them, the last.
      old_cpk = cpk;
    }
    if (ok) {
      cp_async_wait<0>();
#pragma unroll
      for (int ago = C::kAhead - 2; ago >= 0; --ago)
        if (seq >= (uint32_t)ago + 1) signal(seq - 1 - ago, guard >> ago & 1, cpk);
    }
    cp_async_wait<0>();
  } else {
    // ---- softmax: warp w serves unit w / 4 and its rows 32 (w % 4) .. ----
    const int u = warp >> 2, r = tid & (kTreeRows - 1);
    const uint32_t tu = tmem + u * C::kUnitCols + ((uint32_t)(warp & 3) << 21);
    uint32_t cnt = 0, items = 0;
    for (int it = it0; it < it1; ++it) {
      const TreeItem w = p.items[it];
      if (u >= w.units) continue;
      const int n_tiles = (w.hi - w.lo + kTreeKeys - 1) / kTreeKeys;
      const int head = w.head0 + u * w.head_step;
      const int row0 = (w.tile0 + u * w.tile_step) * kTreeRows;
      const int i = (row0 + r) / p.group, h = head * p.group + (row0 + r) - i * p.group;
      const bool live = i < w.n;
      const bool warp_live = row0 + (warp & 3) * 32 < w.n * p.group;
      if (live) {
        const uint4* src = reinterpret_cast<const uint4*>(
            static_cast<const T*>(p.q) + (long long)(w.q0 + i) * p.q_st + (long long)h * p.q_sh);
        unsigned char* dst = smem + u * C::kQBytes;
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
          *reinterpret_cast<uint4*>(dst + sw_chunk(kTreeRows, r, c)) = src[c];
      }
      fence_async_smem();
      mbar_arrive(bar_q(u));
      const unsigned long long mask = live ? row_mask(p, w, i) : 0;
      const long long pos = live && p.window >= 0 ? p.q_positions[w.q0 + i] : 0;
      float m = -INFINITY, l = 0.f;
      bool ok = true;
      for (int t = 0; t < n_tiles; ++t) {
        const uint32_t c = cnt + t, b = c % SB;
        ok = warp_wait(bar_s(u, b), c / SB & 1, abort);
        if (!ok) break;
        if (warp_live) {
          tc_fence_after();
          const uint32_t ts = tu + b * kTreeKeys;
          const int j0 = w.lo + t * kTreeKeys;
          unsigned long long seen = ~0ull;
          if (p.window >= 0 || j0 + kTreeKeys > w.prefix) {
            const int cached = min(max(w.prefix - j0, 0), kTreeKeys);
            seen = cached == 0          ? mask >> (j0 - w.prefix)
                   : cached < kTreeKeys ? mask << cached
                                        : 0;
            if (p.window < 0) {
              seen |= cached == kTreeKeys ? ~0ull : (1ull << cached) - 1;
            } else {
              const int* kp = p.kv_positions + w.kv0 + j0;
              const int p0 = lane < cached ? kp[lane] : 0;
              const int p1 = lane + 32 < cached ? kp[lane + 32] : 0;
              for (int k = 0; k < cached; ++k) {
                const int kpos = __shfl_sync(0xffffffffu, k < 32 ? p0 : p1, k & 31);
                if (pos - kpos <= p.window) seen |= 1ull << k;
              }
            }
            if (j0 + kTreeKeys > w.hi) seen &= (1ull << (w.hi - j0)) - 1;
          }
          const bool masked = __any_sync(0xffffffffu, seen != ~0ull);
          // The scores stay in tensor memory and are read twice, 32 columns
          // at a time (for the maximum, for P): 64 of them in registers
          // spill at the 80 that two CTAs leave a thread.
          auto scores32 = [&](int half, float(&s)[32]) {
            tmem_ld32_sync(ts + 32 * half, s);
            if (masked) {
              const uint32_t bits = (uint32_t)(seen >> 32 * half);
#pragma unroll
              for (int k = 0; k < 32; ++k) s[k] = bits >> k & 1 ? s[k] : -INFINITY;
            }
          };
          float bm;
          {
            float s[32], m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              scores32(half, s);
#pragma unroll
              for (int k = 0; k < 32; ++k) m4[k & 3] = fmaxf(m4[k & 3], s[k]);
            }
            bm = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * p.scale_log2;
          }
          // The base only moves when the tile exceeds it by 2^8; then l and
          // O are rescaled.
          float alpha = 1.f;
          bool rescale = false;
          if (bm > m + kStaleMax || (m == -INFINITY && bm != -INFINITY)) {
            rescale = m != -INFINITY;
            alpha = rescale ? fast_exp2(m - bm) : 0.f;
            m = bm;
          }
          const float nb = m == -INFINITY ? 0.f : -m;
          const f32x2 scale2 = f2_pack(p.scale_log2, p.scale_log2), nb2 = f2_pack(nb, nb);
          f32x2 sum0 = f2_pack(0.f, 0.f), sum1 = sum0;
          // P in two halves, each stored over the first columns of its
          // scores, which this warp has read.
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            uint32_t pk[16];
            float s[32];
            scores32(half, s);
#pragma unroll
            for (int k = 0; k < 32; k += 2) {
              float x0, x1;
              f2_unpack(f2_fma(f2_pack(s[k], s[k + 1]), scale2, nb2), x0, x1);
              x0 = fast_exp2(x0);
              x1 = fast_exp2(x1);
              if (k & 2) sum1 = f2_add(sum1, f2_pack(x0, x1));
              else sum0 = f2_add(sum0, f2_pack(x0, x1));
              pk[k / 2] = pack2<T>(x0, x1);
            }
            tmem_st16_sync(ts + 16 * half, pk);
          }
          float l0, l1;
          f2_unpack(f2_add(sum0, sum1), l0, l1);
          l = l * alpha + (l0 + l1);
          if (__any_sync(0xffffffffu, rescale)) {
            // With one score buffer S(t) came after P(t-1).V(t-1).
            if (SB > 1) ok = warp_wait(bar_o(u), c - 1 & 1, abort);
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
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_p(u, b));
      }
      if (!ok) break;
      cnt += n_tiles;
      if (!warp_wait(bar_done(u), items & 1, abort)) break;
      ++items;
      if (!warp_live) continue;
      tc_fence_after();
      const bool direct = w.partial < 0;
      const long long at = ((long long)w.partial + u) * kTreeRows + r;
      const RowEnd e = row_end(p.sinks, live ? h : 0, m, l);
      T* dst = static_cast<T*>(p.out) + (long long)(w.q0 + i) * p.o_st + (long long)h * p.o_sh;
#pragma unroll
      for (int d = 0; d < D; d += 32) {
        float o[32];
        __syncwarp();
        tmem_ld32_sync(tu + C::kColO + d, o);
        if (!live) continue;
        if (*scrubbed) {
          // Infinities and NaN were taken out of guarded V tiles: the rows
          // that see them get them here.
          for (int j = p.window >= 0 ? w.lo : max(w.lo, w.prefix & ~(kTreeKeys - 1)); j < w.hi;
               ++j) {
            if (!key_seen(p, w, mask, pos, j)) continue;
            const long long slot = key_slot(p, w, j);
            if (slot < 0) continue;
            const T* v = static_cast<const T*>(p.v) + slot * p.v_ss + head * p.v_sh + d;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float x = Elem<T>::to_f32(v[k]);
              if (!isfinite(x)) o[k] += x;
            }
          }
        }
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
          float4* acc = reinterpret_cast<float4*>(p.part_acc + at * D + d);
#pragma unroll
          for (int k = 0; k < 32; k += 4) acc[k / 4] = make_float4(o[k], o[k + 1], o[k + 2], o[k + 3]);
        }
      }
      if (live && !direct) {
        p.part_ml[2 * at] = m;
        p.part_ml[2 * at + 1] = l;
      } else if (live && p.lse) {
        p.lse[(long long)(w.q0 + i) * p.num_q_heads + h] = e.lse;
      }
      tc_fence_before();  // O's reads before the next item's products
    }
  }
  tc_fence_before();
  __syncthreads();
  pdl_launch_dependents();
  if (tid == 0 && *abort && p.error_flag) atomicOr(p.error_flag, 2);
  if (warp == 0) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(256));
  }
}

struct TreeMerge {  // 8 int32
  int q0, n, head0, tile0, steps;  // steps: head_step | tile_step << 1 | units << 2
  int first, count, unused;
};

// Joins the pieces of one unit: one warp per row.
constexpr int kMergeWarps = 8;

template <typename T, int D>
__global__ void __launch_bounds__(32 * kMergeWarps)
tree_merge_kernel(const TreeParams p, const TreeMerge* merges, int units) {
  const TreeMerge g = merges[blockIdx.x];
  const int lane = threadIdx.x & 31;
  const int u = blockIdx.y / (kTreeRows / kMergeWarps);
  const int r = blockIdx.y % (kTreeRows / kMergeWarps) * kMergeWarps + (threadIdx.x >> 5);
  if (u >= g.steps >> 2) return;
  const int head = g.head0 + u * (g.steps & 1);
  const int row = (g.tile0 + u * (g.steps >> 1 & 1)) * kTreeRows + r;
  const int i = row / p.group, h = head * p.group + row % p.group;
  if (i >= g.n) return;
  pdl_wait();
  const long long step = (long long)units * kTreeRows;  // rows between two pieces
  const long long at = ((long long)g.first + u) * kTreeRows + r;
  float m = -INFINITY;
  for (int s = lane; s < g.count; s += 32) m = fmaxf(m, p.part_ml[2 * (at + s * step)]);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, x));
  const float base = m == -INFINITY ? 0.f : m;
  float den = 0.f, num[D / 32];
#pragma unroll
  for (int d = 0; d < D / 32; ++d) num[d] = 0.f;
  for (int s = 0; s < g.count; ++s) {
    const long long a = at + s * step;
    const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + 2 * a);
    const float f = fast_exp2(ml.x - base);
    den += ml.y * f;
#pragma unroll
    for (int d = 0; d < D / 32; ++d) num[d] += p.part_acc[a * D + lane + 32 * d] * f;
  }
  const RowEnd e = row_end(p.sinks, h, m, den);
  T* o = static_cast<T*>(p.out) + (long long)(g.q0 + i) * p.o_st + (long long)h * p.o_sh + lane;
#pragma unroll
  for (int d = 0; d < D / 32; ++d) o[32 * d] = Elem<T>::from_f32(num[d] * e.scale);
  if (p.lse && lane == 0) p.lse[(long long)(g.q0 + i) * p.num_q_heads + h] = e.lse;
}

template <typename T, int D>
int launch_tree(const TreeParams& p, int n_ctas, const TreeMerge* merges, int n_merges,
                cudaStream_t s) {
  using C = TreeCfg<D>;
  if (cudaFuncSetAttribute(tree_attention_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                           C::kSmem) != cudaSuccess)
    return AKV_ERR_CUDA;
  tree_attention_kernel<T, D><<<n_ctas, C::kThreads, C::kSmem, s>>>(p);
  if (n_merges > 0 &&
      launch_pdl(tree_merge_kernel<T, D>, dim3(n_merges, C::kUnits * (kTreeRows / kMergeWarps)),
                 dim3(32 * kMergeWarps), 0, s, p, merges, (int)C::kUnits) != cudaSuccess)
    return AKV_ERR_CUDA;
  return launch_status();
}

}  // namespace
}  // namespace akv

extern "C" int32_t akv_tree_attention_units(int32_t head_dim) {
  return head_dim == 64 || head_dim == 128 ? akv::tree_units(head_dim) : -AKV_ERR_UNSUPPORTED;
}

extern "C" int akv_tree_attention(
    const void* q, int64_t q_stride_token, int64_t q_stride_head, const void* k_pool,
    const void* v_pool, int64_t k_stride_slot, int64_t k_stride_head, int64_t v_stride_slot,
    int64_t v_stride_head, int64_t num_slots, int32_t dtype, const int32_t* kv_indices,
    const int32_t* draft_slots, const int64_t* tree_mask, const int32_t* q_positions,
    const int32_t* kv_positions, int64_t window, const float* sinks, float sm_scale,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, const int32_t* items,
    const int32_t* cta_items, int32_t n_ctas, const int32_t* merges, int32_t n_merges,
    float* partial_acc, float* partial_ml, void* out, int64_t out_stride_token,
    int64_t out_stride_head, float* lse, int32_t* error_flag, void* stream) {
  AKV_NVTX_RANGE("akv_tree_attention");
  using namespace akv;
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads || n_ctas < 0 ||
      n_merges < 0 || !(sm_scale > 0.f) || num_slots <= 0 || (dtype != AKV_F16 && dtype != AKV_BF16))
    return AKV_ERR_INVALID;
  if (head_dim != 64 && head_dim != 128) return AKV_ERR_UNSUPPORTED;
  if (n_ctas == 0) return AKV_OK;
  if (!q || !k_pool || !v_pool || !draft_slots || !tree_mask || !items || !cta_items || !out ||
      !kv_indices || (n_merges > 0 && (!merges || !partial_acc || !partial_ml)) ||
      (window >= 0 && (!q_positions || !kv_positions)))
    return AKV_ERR_INVALID;
  const void* bases[] = {q, k_pool, v_pool, out};
  for (const void* b : bases)
    if (reinterpret_cast<uintptr_t>(b) & 15) return AKV_ERR_INVALID;
  const int64_t strides[] = {q_stride_token, q_stride_head,    k_stride_slot,  k_stride_head,
                             v_stride_slot,  v_stride_head,    out_stride_token, out_stride_head};
  for (int64_t s : strides)
    if (s % 8) return AKV_ERR_INVALID;  // 16-byte rows
  TreeParams p{q, q_stride_token, q_stride_head, k_pool, v_pool, k_stride_slot, k_stride_head,
               v_stride_slot, v_stride_head, num_slots, kv_indices, draft_slots,
               reinterpret_cast<const unsigned long long*>(tree_mask), q_positions, kv_positions,
               window, sinks, sm_scale * kLog2e, num_q_heads / num_kv_heads, num_q_heads,
               reinterpret_cast<const TreeItem*>(items), cta_items, partial_acc, partial_ml, out,
               out_stride_token, out_stride_head, lse, error_flag};
  const TreeMerge* m = reinterpret_cast<const TreeMerge*>(merges);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == AKV_BF16)
    return head_dim == 64 ? launch_tree<__nv_bfloat16, 64>(p, n_ctas, m, n_merges, s)
                          : launch_tree<__nv_bfloat16, 128>(p, n_ctas, m, n_merges, s);
  return head_dim == 64 ? launch_tree<__half, 64>(p, n_ctas, m, n_merges, s)
                        : launch_tree<__half, 128>(p, n_ctas, m, n_merges, s);
}
