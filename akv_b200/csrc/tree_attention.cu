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

#include <algorithm>

#include "attention_common.cuh"

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

// One thread per row, keys one after another.
template <typename T, int D>
__global__ void __launch_bounds__(kTreeRows) tree_attention_kernel(const TreeParams p, int units) {
  __shared__ float ks[16][D], vs[16][D];
  __shared__ long long slots[16];
  const int r = threadIdx.x;
  for (int it = p.cta_items[blockIdx.x]; it < p.cta_items[blockIdx.x + 1]; ++it) {
    const TreeItem w = p.items[it];
    for (int u = 0; u < w.units; ++u) {
      const int head = w.head0 + u * w.head_step;
      const int row = (w.tile0 + u * w.tile_step) * kTreeRows + r;
      const int i = row / p.group, h = head * p.group + row % p.group;
      const bool live = i < w.n;
      const T* q = static_cast<const T*>(p.q) + (long long)(w.q0 + (live ? i : 0)) * p.q_st +
                   (long long)(live ? h : 0) * p.q_sh;
      const unsigned long long mask = live ? row_mask(p, w, i) : 0;
      const long long pos = live && p.window >= 0 ? p.q_positions[w.q0 + i] : 0;
      float acc[D], m = -INFINITY, l = 0.f;
      for (int d = 0; d < D; ++d) acc[d] = 0.f;
      for (int j0 = w.lo; j0 < w.hi; j0 += 16) {
        __syncthreads();
        if (r < 16) slots[r] = j0 + r < w.hi ? key_slot(p, w, j0 + r) : -1;
        __syncthreads();
        for (int e = r; e < 16 * D; e += kTreeRows) {
          const long long s = slots[e / D];
          const T* kp = static_cast<const T*>(p.k) + s * p.k_ss + head * p.k_sh;
          const T* vp = static_cast<const T*>(p.v) + s * p.v_ss + head * p.v_sh;
          ks[e / D][e % D] = s < 0 ? 0.f : Elem<T>::to_f32(kp[e % D]);
          vs[e / D][e % D] = s < 0 ? 0.f : Elem<T>::to_f32(vp[e % D]);
        }
        __syncthreads();
        for (int c = 0; c < 16 && j0 + c < w.hi; ++c) {
          const int j = j0 + c;
          bool seen = live && (j < w.prefix || (mask >> (j - w.prefix) & 1));
          if (seen && j < w.prefix && p.window >= 0)
            seen = pos - p.kv_positions[w.kv0 + j] <= p.window;
          if (!seen) continue;
          float s = 0.f;
          for (int d = 0; d < D; ++d) s += Elem<T>::to_f32(q[d]) * ks[c][d];
          s *= p.scale_log2;
          const float mn = fmaxf(m, s), base = mn == -INFINITY ? 0.f : mn;
          const float alpha = fast_exp2(m - base), e = fast_exp2(s - base);
          m = mn;
          l = l * alpha + e;
          for (int d = 0; d < D; ++d) acc[d] = acc[d] * alpha + e * vs[c][d];
        }
      }
      if (!live) continue;
      if (w.partial >= 0) {
        const long long at = (long long)(w.partial + u) * kTreeRows + r;
        for (int d = 0; d < D; ++d) p.part_acc[at * D + d] = acc[d];
        p.part_ml[2 * at] = m;
        p.part_ml[2 * at + 1] = l;
        continue;
      }
      const RowEnd e = row_end(p.sinks, h, m, l);
      T* o = static_cast<T*>(p.out) + (long long)(w.q0 + i) * p.o_st + (long long)h * p.o_sh;
      for (int d = 0; d < D; ++d) o[d] = Elem<T>::from_f32(acc[d] * e.scale);
      if (p.lse) p.lse[(long long)(w.q0 + i) * p.num_q_heads + h] = e.lse;
    }
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

constexpr int tree_units(int head_dim) { return head_dim == 64 ? 2 : 1; }

template <typename T, int D>
int launch_tree(const TreeParams& p, int n_ctas, const TreeMerge* merges, int n_merges,
                cudaStream_t s) {
  constexpr int U = tree_units(D);
  if (n_ctas > 0) tree_attention_kernel<T, D><<<n_ctas, kTreeRows, 0, s>>>(p, U);
  if (n_merges > 0)
    tree_merge_kernel<T, D><<<dim3(n_merges, U * (kTreeRows / kMergeWarps)), 32 * kMergeWarps, 0,
                              s>>>(p, merges, U);
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
      n_merges < 0 || num_slots <= 0 || (dtype != AKV_F16 && dtype != AKV_BF16))
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
