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
// two rows (one in fp32) that it requests before it uses the first.  Measured on
// 16,411 tokens of 64 + 8 + 8 heads of 128, bf16 (681 MB): 142 us, 4.8 TB/s,
// 0.73 of the copy rate, at 8 blocks of 128 threads per SM; four rows per lane
// (102 registers, 5 blocks) 156-179 us, one row 177 us, two rows at a time
// in a loop that keeps the table row 160 us (spills): residency counts most.

#include "common.cuh"

namespace akv {
namespace {

constexpr int kRopeThreads = 128;

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
  float eps;
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
  __device__ __forceinline__ void set(int i, float x) {
    v[i / Vec16<T>::N].e[i % Vec16<T>::N] = Elem<T>::from_f32(x);
  }
};

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
// two); NEOX: halves or adjacent pairs; ROWS: rows per lane group.
template <typename T, int LANES, bool NEOX, int ROWS>
__global__ void __launch_bounds__(kRopeThreads, 8) qk_norm_rope_kernel(const RopeArgs a) {
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
  const bool live = NEOX ? 16 * j < a.dim : 8 * j < a.dim, live1 = NEOX ? live : e1 < a.dim;

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
  float w0[8], w1[8];
  if (weight != nullptr) {
    if (a.weight_f32) {
      if (live) load8<float>(weight, e0, w0);
      if (live1) load8<float>(weight, e1, w1);
    } else {
      if (live) load8<T>(weight, e0, w0);
      if (live1) load8<T>(weight, e1, w1);
    }
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
    if (weight != nullptr) {
      float ss = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) ss += y0[i] * y0[i] + y1[i] * y1[i];
#pragma unroll
      for (int d = LANES / 2; d > 0; d >>= 1) ss += __shfl_xor_sync(lanes, ss, d);
      const float inv = rsqrtf(ss / (float)a.dim + a.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (live) y0[i] *= inv * w0[i];
        if (live1) y1[i] *= inv * w1[i];
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (NEOX) {
        x0[r].set(i, y0[i] * c[i] - y1[i] * s[i]);
        x1[r].set(i, y1[i] * c[i] + y0[i] * s[i]);
      } else if (i < 4) {
        x0[r].set(2 * i, y0[2 * i] * c[i] - y0[2 * i + 1] * s[i]);
        x0[r].set(2 * i + 1, y0[2 * i + 1] * c[i] + y0[2 * i] * s[i]);
        x1[r].set(2 * i, y1[2 * i] * c[4 + i] - y1[2 * i + 1] * s[4 + i]);
        x1[r].set(2 * i + 1, y1[2 * i + 1] * c[4 + i] + y1[2 * i] * s[4 + i]);
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

template <typename T, int LANES, bool NEOX>
int launch_rope(RopeArgs& a, cudaStream_t stream) {
  constexpr int ROWS = sizeof(T) == 4 ? 1 : 2;
  a.q_units = (a.hq + ROWS - 1) / ROWS;
  a.k_units = (a.hkv + ROWS - 1) / ROWS;
  a.units = a.q_units + a.k_units * (a.v != nullptr ? 2 : 1);
  const long long groups = a.tokens * a.units, per = kRopeThreads / LANES;
  const long long blocks = (groups + per - 1) / per;
  if (groups + per > UINT32_MAX) return AKV_ERR_INVALID;  // 32-bit group numbers
  qk_norm_rope_kernel<T, LANES, NEOX, ROWS><<<(unsigned)blocks, kRopeThreads, 0, stream>>>(a);
  return launch_status();
}

template <typename T, int LANES>
int launch_rope_style(RopeArgs& a, int neox, cudaStream_t stream) {
  return neox ? launch_rope<T, LANES, true>(a, stream) : launch_rope<T, LANES, false>(a, stream);
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
             (float)x.eps, x.positions, x.positions_is64 != 0, x.slots, x.slots_is64 != 0,
             x.cos_sin_cache, (int)x.cache_dtype, x.cache_stride, x.max_position, x.num_slots,
             x.tokens, (int)x.num_q_heads, (int)x.num_kv_heads, (int)x.head_dim,
             (int)x.rotary_dim, 0, 0, 0, x.error_flag};
  const int neox = x.is_neox_style != 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  switch (x.dtype) {
    case AKV_F16: return launch_rope_lanes<__half>(a, neox, s);
    case AKV_BF16: return launch_rope_lanes<__nv_bfloat16>(a, neox, s);
    default: return launch_rope_lanes<float>(a, neox, s);
  }
}
