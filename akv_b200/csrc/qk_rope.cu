// Per-head RMS norms of Q and K, the position rotation and the store of K and
// V into the paged cache, in one pass over a layer's projections.
//
// For every token and head row x of D elements (fp32 arithmetic, one rounding
// to the tensors' type at the end):
//   y = x * rsqrt(mean(x^2) + eps) * w              (skipped without weights)
//   rotation of y's first R elements by the token's table row (cos | sin):
//     halves (NEOX):      (y_i, y_{i+R/2}) -> (y_i c - y_{i+R/2} s, y_{i+R/2} c + y_i s)
//     adjacent pairs:     the same with (y_{2i}, y_{2i+1})
//   Q rows go to q_out, K rows to k_out and / or k_pool[slot], V rows are
//   copied to v_pool[slot].  The reference runs its model's q_norm / k_norm,
//   rotary module and set_kv_buffer one after the other (native SGLang
//   modules around akv/system/sglang.patch:2437-2445).
//
// Bound: HBM.  Each element is read and written once.  A row is shared by
// D / 16 lanes, each with two 8-element pieces: with halves the two that
// rotate into one another ([8j, 8j + 8) and [R/2 + 8j, ..)), with pairs j and
// j + D/16, which rotate within themselves.  So the rotation needs no exchange,
// the lanes of an access are neighbours, and the norm's sum is log2(D/16)
// shuffles.  A lane keeps its 8 cos, 8 sin and 16 weights in registers for the
// four rows (two in fp32) that it requests before it uses the first; the
// arithmetic is packed (f32x2), two elements an instruction, since with scalar
// instructions their issue was the limit (142 us at best on the first case
// below).  Measured, bf16 (calls one after another in a graph, other inputs each):
// 16,411 tokens of 64 + 8 + 8 heads of 128 (681 MB) 124 us, 5.5 TB/s, 0.84 of the
// copy rate, at 12 blocks of 64 threads per SM (80 registers); two rows per lane 132
// us, eight 138 us, four at 16 warps per SM 141 us and at 28 146 us (more spills:
// at 80 registers every instantiation keeps 48 to 148 bytes of a thread in local
// memory, 116 in this one).  fp32, 8,205 tokens of the same heads (676 MB) 105 us,
// 6.4 TB/s.  2,048 tokens of head_dim 64 (42.5 MB) 12 us; one token 3.8 us.  With
// only a part of D turning (fp16, pairs, 64 of 128, 76.6 MB) 17.5-18.1 us, 4.3
// TB/s: 2.6 waves of blocks, and the masks of what does not turn (16.5 without;
// two rows per lane 18.8).

#include <type_traits>

#include "attention_common.cuh"

namespace akv {
namespace {

constexpr int kRopeThreads = 64;

struct RopeArgs {
  const void* q;
  long long q_st, q_sh;
  const void* k;
  long long k_st, k_sh;
  const void* v;
  long long v_st, v_sh;
  void* q_out;
  long long qo_st, qo_sh;
  void* k_out;
  long long ko_st, ko_sh;
  void* k_pool;
  long long kp_ss, kp_sh;
  void* v_pool;
  long long vp_ss, vp_sh;
  const void* q_weight;
  const void* k_weight;
  int weight_f32;
  float eps, inv_dim;
  const void* positions;
  int positions_is64;
  const void* slots;
  int slots_is64;
  const void* table;
  int table_dtype;
  long long table_stride, max_position, num_slots;
  long long tokens;
  int hq, hkv, dim, rotary;
  int q_units, k_units, units;  // units of kRows rows: Q's, K's (and V's), all
  int* error_flag;
};

// Eight consecutive elements, as fp32.
template <typename T>
struct Eight {
  Vec16<T> v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = ld16(p + i * Vec16<T>::N);
  }
  __device__ __forceinline__ void store(T* p) const {
#pragma unroll
    for (int i = 0; i < (int)sizeof(T) / 2; ++i) st16(p + i * Vec16<T>::N, v[i]);
  }
  __device__ __forceinline__ float get(int i) const {
    return Elem<T>::to_f32(v[i / Vec16<T>::N].e[i % Vec16<T>::N]);
  }
  __device__ __forceinline__ void set2(int i, float x, float y) {  // elements i, i + 1
    T* e = &v[i / Vec16<T>::N].e[i % Vec16<T>::N];
    if constexpr (std::is_same<T, __nv_bfloat16>::value) {
      *reinterpret_cast<__nv_bfloat162*>(e) = __floats2bfloat162_rn(x, y);
    } else if constexpr (std::is_same<T, __half>::value) {
      *reinterpret_cast<__half2*>(e) = __floats2half2_rn(x, y);
    } else {
      e[0] = x;
      e[1] = y;
    }
  }
};

// The two elements of each of a lane's eight turning pairs, in packed fp32
// pairs of neighbours: x turns into x c - y s, y into y c + x s.
struct Turn {
  f32x2 x[4], y[4];
};
// From values (or weights) of the lane's two runs.
template <bool NEOX>
__device__ __forceinline__ Turn turn_of(const float (&a)[8], const float (&b)[8]) {
  Turn t;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float* e = k < 2 ? a : b;  // adjacent pairs: 0-3 in the first run, 4-7 in the second
    const int i = 4 * (k & 1);
    t.x[k] = NEOX ? f2_pack(a[2 * k], a[2 * k + 1]) : f2_pack(e[i], e[i + 2]);
    t.y[k] = NEOX ? f2_pack(b[2 * k], b[2 * k + 1]) : f2_pack(e[i + 1], e[i + 3]);
  }
  return t;
}

template <typename T>
__device__ __forceinline__ void load8(const void* base, long long at, float (&out)[8]) {
  Eight<T> e;
  e.load(static_cast<const T*>(base) + at);
#pragma unroll
  for (int i = 0; i < 8; ++i) out[i] = e.get(i);
}

// Four consecutive elements (8 or 16 bytes), as fp32.
template <typename T>
__device__ __forceinline__ void load4(const void* base, long long at, float* out) {
  struct alignas(4 * sizeof(T)) Four { T e[4]; };
  const Four f = *reinterpret_cast<const Four*>(static_cast<const T*>(base) + at);
#pragma unroll
  for (int i = 0; i < 4; ++i) out[i] = Elem<T>::to_f32(f.e[i]);
}

// The eight cosines (or sines) of a lane's two runs: at a one run of eight
// (halves), or four at a and, if `both`, four at b (pairs).
template <typename T, bool NEOX>
__device__ __forceinline__ void load_turn(const void* base, long long a, long long b, bool both,
                                          float (&out)[8]) {
  if (NEOX) {
    load8<T>(base, a, out);
  } else {
    load4<T>(base, a, out);
    if (both) load4<T>(base, b, out + 4);
  }
}

// T: element type; LANES: lanes per row (D / 16 rounded up to a power of
// two); NEOX: halves or adjacent pairs; FULL: D is 16 LANES, so that every lane
// has two runs; TURN: all of D turns; ROWS: rows per lane group.
template <typename T, int LANES, bool NEOX, bool FULL, bool TURN, int ROWS>
__global__ void __launch_bounds__(kRopeThreads, 12) qk_norm_rope_kernel(const RopeArgs a) {
  const uint32_t group = blockIdx.x * (kRopeThreads / LANES) + threadIdx.x / LANES;
  const int j = threadIdx.x % LANES;
  const uint32_t token32 = group / (uint32_t)a.units;
  const int unit = (int)(group - token32 * a.units);
  const long long token = token32;
  if (token >= a.tokens) return;  // whole lane groups leave together
  // Shuffles stay inside the lane group, whose lanes all take the same path.
  const unsigned lanes =
      LANES == 32 ? 0xffffffffu
                  : ((1u << (LANES & 31)) - 1u) << ((threadIdx.x & 31) / LANES * LANES);
  const int kind = unit < a.q_units ? 0 : unit < a.q_units + a.k_units ? 1 : 2;
  const int first =
      (kind == 0 ? unit : kind == 1 ? unit - a.q_units : unit - a.q_units - a.k_units) * ROWS;
  const int heads = kind == 0 ? a.hq : a.hkv;
  // This lane's two runs of eight elements.  Halves: [8j, 8j + 8) of the
  // first half and of the second, and past the rotation the same of the rest.
  // Pairs: pieces j and j + LANES of the row, each turning within itself.
  const int half = a.rotary / 2, t = j - a.rotary / 16;
  const bool turned = NEOX ? t < 0 : 8 * j < a.rotary;
  const bool turned1 = NEOX ? turned : 8 * (j + LANES) < a.rotary;
  const int e0 = NEOX && t >= 0 ? a.rotary + 8 * t : 8 * j;
  const int e1 = !NEOX ? 8 * (j + LANES) : t >= 0 ? (a.rotary + a.dim) / 2 + 8 * t : half + 8 * j;
  const bool live = FULL || (NEOX ? 16 * j < a.dim : 8 * j < a.dim);
  const bool live1 = FULL || (NEOX ? live : e1 < a.dim);

  const T* src = static_cast<const T*>(kind == 0 ? a.q : kind == 1 ? a.k : a.v);
  const long long st = kind == 0 ? a.q_st : kind == 1 ? a.k_st : a.v_st;
  const long long sh = kind == 0 ? a.q_sh : kind == 1 ? a.k_sh : a.v_sh;
  src += token * st + first * sh;
  Eight<T> x0[ROWS], x1[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    if (first + r < heads) {
      if (live) x0[r].load(src + r * sh + e0);
      if (live1) x1[r].load(src + r * sh + e1);
    }

  long long slot = -1;
  if (kind != 0 && a.slots != nullptr) {
    slot = ld_index(a.slots, token, a.slots_is64);
    if (slot >= a.num_slots) {  // never touch memory outside the pools
      if (a.error_flag) *a.error_flag = 1;
      slot = -1;
    }
  }
  long long pos = ld_index(a.positions, token, a.positions_is64);
  if (pos < 0 || pos >= a.max_position) {
    if (a.error_flag) *a.error_flag = 1;
    pos = 0;
    slot = -1;
  }
  if (kind == 2) {
    if (slot < 0) return;
    T* dst = static_cast<T*>(a.v_pool) + slot * a.vp_ss + first * a.vp_sh;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
      if (first + r < heads) {
        if (live) x0[r].store(dst + r * a.vp_sh + e0);
        if (live1) x1[r].store(dst + r * a.vp_sh + e1);
      }
    return;
  }

  float c[8], s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    c[i] = 1.f;
    s[i] = 0.f;
  }
  if (turned) {
    const long long at = pos * a.table_stride + (NEOX ? 8 : 4) * j, at1 = at + 4 * LANES;
    if (a.table_dtype == AKV_F32) {
      load_turn<float, NEOX>(a.table, at, at1, turned1, c);
      load_turn<float, NEOX>(a.table, at + half, at1 + half, turned1, s);
    } else if (a.table_dtype == AKV_BF16) {
      load_turn<__nv_bfloat16, NEOX>(a.table, at, at1, turned1, c);
      load_turn<__nv_bfloat16, NEOX>(a.table, at + half, at1 + half, turned1, s);
    } else {
      load_turn<__half, NEOX>(a.table, at, at1, turned1, c);
      load_turn<__half, NEOX>(a.table, at + half, at1 + half, turned1, s);
    }
  }
  const void* weight = kind == 0 ? a.q_weight : a.k_weight;
  f32x2 c2[4], s2[4], n2[4];  // cos, sin, -sin
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    c2[k] = f2_pack(c[2 * k], c[2 * k + 1]);
    s2[k] = f2_pack(s[2 * k], s[2 * k + 1]);
    n2[k] = f2_pack(-s[2 * k], -s[2 * k + 1]);
  }
  const f32x2 keep = turned ? ~0ull : 0, keep1 = turned1 ? ~0ull : 0;
  Turn w;
  if (weight != nullptr) {
    float w0[8] = {}, w1[8] = {};
    if (a.weight_f32) {
      if (live) load8<float>(weight, e0, w0);
      if (live1) load8<float>(weight, e1, w1);
    } else {
      if (live) load8<T>(weight, e0, w0);
      if (live1) load8<T>(weight, e1, w1);
    }
    w = turn_of<NEOX>(w0, w1);
  }

  T* out = static_cast<T*>(kind == 0 ? a.q_out : a.k_out);
  if (out != nullptr)
    out += kind == 0 ? token * a.qo_st + first * a.qo_sh : token * a.ko_st + first * a.ko_sh;
  const long long oh = kind == 0 ? a.qo_sh : a.ko_sh;
  T* pool = kind == 1 && slot >= 0 && a.k_pool != nullptr
                ? static_cast<T*>(a.k_pool) + slot * a.kp_ss + first * a.kp_sh
                : nullptr;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    if (first + r >= heads) break;
    float y0[8], y1[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      y0[i] = live ? x0[r].get(i) : 0.f;
      y1[i] = live1 ? x1[r].get(i) : 0.f;
    }
    Turn v = turn_of<NEOX>(y0, y1);
    if (weight != nullptr) {
      f32x2 sx = f2_pack(0.f, 0.f), sy = sx;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        sx = f2_fma(v.x[k], v.x[k], sx);
        sy = f2_fma(v.y[k], v.y[k], sy);
      }
      float a0, a1;
      f2_unpack(f2_add(sx, sy), a0, a1);
      float ss = a0 + a1;
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(lanes, ss, d);
      const float inv = rsqrtf(ss * a.inv_dim + a.eps);
      const f32x2 inv2 = f2_pack(inv, inv);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        v.x[k] = f2_mul(v.x[k], f2_mul(w.x[k], inv2));
        v.y[k] = f2_mul(v.y[k], f2_mul(w.y[k], inv2));
      }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      f32x2 xs = f2_mul(v.x[k], s2[k]), ys;
      if (TURN) {
        ys = f2_mul(v.y[k], n2[k]);
      } else {
        // Past the rotation the turn is by cos 1 and sin 0, and the products
        // are masked to 0: an infinity times sin 0 would be NaN.  The sign is
        // set here too, since n2's registers would spill as well.
        const f32x2 on = NEOX || k < 2 ? keep : keep1;
        xs &= on;
        ys = (f2_mul(v.y[k], s2[k]) & on) ^ 0x8000000080000000ull;
      }
      float p0, p1, q0, q1;
      f2_unpack(f2_fma(v.x[k], c2[k], ys), p0, p1);
      f2_unpack(f2_fma(v.y[k], c2[k], xs), q0, q1);
      if (NEOX) {
        x0[r].set2(2 * k, p0, p1);
        x1[r].set2(2 * k, q0, q1);
      } else {
        Eight<T>& run = k < 2 ? x0[r] : x1[r];
        run.set2(4 * (k & 1), p0, q0);
        run.set2(4 * (k & 1) + 2, p1, q1);
      }
    }
    if (out != nullptr) {
      if (live) x0[r].store(out + r * oh + e0);
      if (live1) x1[r].store(out + r * oh + e1);
    }
    if (pool != nullptr) {
      if (live) x0[r].store(pool + r * a.kp_sh + e0);
      if (live1) x1[r].store(pool + r * a.kp_sh + e1);
    }
  }
}

template <typename T, int LANES, bool NEOX, bool FULL, bool TURN>
int launch_rope(RopeArgs& a, cudaStream_t stream) {
  constexpr int ROWS = sizeof(T) == 4 ? 2 : 4;
  a.q_units = (a.hq + ROWS - 1) / ROWS;
  a.k_units = (a.hkv + ROWS - 1) / ROWS;
  a.units = a.q_units + a.k_units * (a.v != nullptr ? 2 : 1);
  const long long groups = a.tokens * a.units, per = kRopeThreads / LANES;
  const long long blocks = (groups + per - 1) / per;
  if (groups + per > UINT32_MAX) return AKV_ERR_INVALID;  // 32-bit group numbers
  qk_norm_rope_kernel<T, LANES, NEOX, FULL, TURN, ROWS>
      <<<(unsigned)blocks, kRopeThreads, 0, stream>>>(a);
  return launch_status();
}

template <typename T, int LANES, bool NEOX>
int launch_rope_turn(RopeArgs& a, cudaStream_t stream) {
  if (a.dim != 16 * LANES) return launch_rope<T, LANES, NEOX, false, false>(a, stream);
  return a.rotary == a.dim ? launch_rope<T, LANES, NEOX, true, true>(a, stream)
                           : launch_rope<T, LANES, NEOX, true, false>(a, stream);
}

template <typename T, int LANES>
int launch_rope_style(RopeArgs& a, int neox, cudaStream_t stream) {
  return neox ? launch_rope_turn<T, LANES, true>(a, stream)
              : launch_rope_turn<T, LANES, false>(a, stream);
}

template <typename T>
int launch_rope_lanes(RopeArgs& a, int neox, cudaStream_t stream) {
  if (a.dim <= 32) return launch_rope_style<T, 2>(a, neox, stream);
  if (a.dim <= 64) return launch_rope_style<T, 4>(a, neox, stream);
  if (a.dim <= 128) return launch_rope_style<T, 8>(a, neox, stream);
  if (a.dim <= 256) return launch_rope_style<T, 16>(a, neox, stream);
  return launch_rope_style<T, 32>(a, neox, stream);
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace
}  // namespace akv

extern "C" int64_t akv_qk_norm_rope_args_bytes(void) { return sizeof(akv_qk_norm_rope_args); }

extern "C" int akv_qk_norm_rope(const akv_qk_norm_rope_args* args, void* stream) {
  AKV_NVTX_RANGE("akv_qk_norm_rope");
  using namespace akv;
  if (args == nullptr) return AKV_ERR_INVALID;
  const akv_qk_norm_rope_args& x = *args;
  if (x.tokens < 0 || x.num_q_heads <= 0 || x.num_kv_heads <= 0 || x.num_q_heads > INT32_MAX / 2 ||
      x.num_kv_heads > INT32_MAX / 2 || x.head_dim < 16 || x.head_dim > 512 || x.head_dim % 16 ||
      x.rotary_dim <= 0 || x.rotary_dim > x.head_dim || x.rotary_dim % 16 || x.dtype < AKV_F16 ||
      x.dtype > AKV_F32 || x.cache_dtype < AKV_F16 || x.cache_dtype > AKV_F32 ||
      ((x.q_weight || x.k_weight) && x.weight_dtype != x.dtype && x.weight_dtype != AKV_F32))
    return AKV_ERR_INVALID;
  if (x.tokens == 0) return AKV_OK;
  if (!x.q || !x.k || !x.q_out || !x.positions || !x.cos_sin_cache || x.max_position <= 0 ||
      (!x.k_out && !x.k_pool) ||
      (x.k_pool && (!x.v || !x.v_pool || !x.slots || x.num_slots <= 0)) || (x.v && !x.k_pool))
    return AKV_ERR_INVALID;
  const int64_t vec = x.dtype == AKV_F32 ? 4 : 8;  // elements of a 16-byte access
  const int64_t cache_vec = x.cache_dtype == AKV_F32 ? 4 : 8;
  const int64_t strides[] = {
      x.q_stride_token,     x.q_stride_head,      x.k_stride_token,     x.k_stride_head,
      x.v_stride_token,     x.v_stride_head,      x.q_out_stride_token, x.q_out_stride_head,
      x.k_out_stride_token, x.k_out_stride_head,  x.k_pool_stride_slot, x.k_pool_stride_head,
      x.v_pool_stride_slot, x.v_pool_stride_head};
  for (int64_t s : strides)
    if (s % vec) return AKV_ERR_INVALID;
  const void* bases[] = {x.q,      x.k,      x.v,        x.q_out,    x.k_out,
                         x.k_pool, x.v_pool, x.q_weight, x.k_weight, x.cos_sin_cache};
  for (const void* p : bases)
    if (!aligned16(p)) return AKV_ERR_INVALID;
  if (x.cache_stride % cache_vec) return AKV_ERR_INVALID;
  RopeArgs a{x.q, x.q_stride_token, x.q_stride_head, x.k, x.k_stride_token, x.k_stride_head, x.v,
             x.v_stride_token, x.v_stride_head, x.q_out, x.q_out_stride_token,
             x.q_out_stride_head, x.k_out, x.k_out_stride_token, x.k_out_stride_head, x.k_pool,
             x.k_pool_stride_slot, x.k_pool_stride_head, x.v_pool, x.v_pool_stride_slot,
             x.v_pool_stride_head, x.q_weight, x.k_weight, x.weight_dtype == AKV_F32,
             (float)x.eps, 1.f / (float)x.head_dim, x.positions, x.positions_is64 != 0, x.slots,
             x.slots_is64 != 0, x.cos_sin_cache, (int)x.cache_dtype, x.cache_stride, x.max_position,
             x.num_slots, x.tokens, (int)x.num_q_heads, (int)x.num_kv_heads, (int)x.head_dim,
             (int)x.rotary_dim, 0, 0, 0, x.error_flag};
  const int neox = x.is_neox_style != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (x.dtype) {
    case AKV_F16: return launch_rope_lanes<__half>(a, neox, s);
    case AKV_BF16: return launch_rope_lanes<__nv_bfloat16>(a, neox, s);
    default: return launch_rope_lanes<float>(a, neox, s);
  }
}
