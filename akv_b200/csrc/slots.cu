// Slot maps, positions, draft-tree masks and block tables of a batch's new
// tokens, built on the device from the requests' lengths.
//
// Request b has L = raw_lens[b] tokens in columns [0, L) of its row of
// req_to_token and receives n = new_lens[b] more.  With pages of p = 2^k
// token slots (token t of a request at offset t % p of its page),
//
//   need_b = ceil((L + n) / p) - ceil(L / p)       pages the new tokens open
//   base_b = sum of need over the requests before b
//   new token t in [L, L + n):
//     page = row[L - 1] / p                        if t / p < ceil(L / p)
//            ring[(head + base_b + t / p - ceil(L / p)) % capacity]  otherwise
//     slot = page * p + t % p,  row[t] = slot
//   position = next_position[b] + depth of the node (with a draft tree)
//                               + t - L              (without)
//   mask     = own bit | mask of the parent (64 nodes at most per request)
//
// The reference builds these on the host (the scheduler allocates slots and
// writes req_to_token from Python, akv/system/sglang.patch:3133-3180); the
// reading side's metadata is page_table.cu.
//
// Bound: latency.  The kernel moves about 12-24 bytes per token and 8 per
// table entry, so one launch with two dependent load rounds is the floor.
// Every block therefore sums the whole batch's lengths itself (a batch is a
// few hundred loads from L2) instead of waiting for a scan kernel.  Measured
// (device time, calls one after another in a graph): one request 4.2 us; 64
// requests over 16-slot pages with block tables 5.7-6.1 us; 512 requests of 0-64
// drafted tokens with block tables of 4.2M entries (33.8 MB) 14.7-15.2 us, of
// which the tables about 8 (20.8 us with 4-byte copies; eight 16-byte loads in
// flight instead of four, or blocks of 512 threads, 20 us: then not all blocks
// are resident).  The loads of a table's old part wait for the sums only because
// a refused call must leave the table alone.  More blocks per request cost more
// sums than they save (4-byte copies: 15.5 us at one block, 19.9 at two, 28 at
// four).

#include <algorithm>

#include "common.cuh"

namespace akv {
namespace {

constexpr int kSlotThreads = 256;
constexpr int kTreeNodes = 64;

struct SlotArgs {
  int32_t* req_to_token;
  int64_t row_stride, rows, columns;
  const void* row_ids;
  int row_ids_is64;
  const void* raw_lens;
  int raw_lens_is64;
  const void* new_lens;
  int new_lens_is64;
  int batch;
  int shift;  // log2(page size)
  int32_t* ring;
  long long* ring_state;
  int64_t ring_capacity;
  const void* next_positions;  // null: the row length
  int next_is64;
  const int32_t* parents;      // null: no tree
  int64_t capacity;            // new tokens the outputs hold
  int32_t* new_offsets;
  int32_t* slots;
  int32_t* positions;
  int64_t* tree_mask;
  int32_t* block_table;
  int64_t table_stride, table_columns;
  int32_t* totals;             // {new tokens, pages}
  int32_t* status;
  unsigned* arrivals;
  int commit;
  int keep;  // a bad request keeps its entries of the outputs
};

struct Request {
  long long len, fresh, row, need;
  bool bad, unsized;  // unsized: bad, and its length leaves no room to keep
};

__device__ __forceinline__ Request load_request(const SlotArgs& a, int b) {
  Request r;
  r.row = ld_index(a.row_ids, b, a.row_ids_is64);
  r.len = ld_index(a.raw_lens, b, a.raw_lens_is64);
  r.fresh = ld_index(a.new_lens, b, a.new_lens_is64);
  const long long end = r.len + r.fresh;
  r.unsized = r.fresh < 0 || r.fresh > a.columns || (a.parents != nullptr && r.fresh > kTreeNodes);
  r.bad = r.unsized || r.row < 0 || r.row >= a.rows || r.len < 0 || r.len > a.columns ||
          end > a.columns ||
          (a.block_table != nullptr && ((end - 1) >> a.shift) >= a.table_columns);
  // A bad request takes part as one without new tokens, or (keep) as one whose
  // tokens take no page.
  if (r.bad && (r.unsized || !a.keep)) r.fresh = 0;
  const long long up = (1ll << a.shift) - 1;
  r.need = r.bad ? 0 : ((end + up) >> a.shift) - ((r.len + up) >> a.shift);
  return r;
}

// A row ends inside a page whose last slot is not at its offset: it cannot go on.
__device__ __forceinline__ bool off_page(int last, long long len, int p_mask) {
  return last < 0 || (last & p_mask) != ((len - 1) & p_mask);
}

// Pages counted for requests that off_page stopped, which no row holds: moves
// them in the ring behind those that were given out, entries [head, head +
// taken), where they are the first free ones once the head has passed the
// others.  Returns their number.  One warp, after every block has read its
// pages.  From the last to the first, so that an entry is read before one of a
// later request, which never lies before it, takes its place.
__device__ long long return_pages(const SlotArgs& a, long long head, long long taken, int lane) {
  const int p_mask = (1 << a.shift) - 1;
  auto entry = [&](long long at) { return a.ring + (head + at) % a.ring_capacity; };
  long long end = taken, to = taken;  // pages before which request's; next free place
  for (int i0 = (a.batch - 1) / 32 * 32; i0 >= 0; i0 -= 32) {
    long long need = 0;
    bool lost = false;
    if (i0 + lane < a.batch) {
      const Request r = load_request(a, i0 + lane);
      need = r.need;
      lost = need > 0 && (r.len & p_mask) != 0 &&
             off_page(a.req_to_token[r.row * a.row_stride + r.len - 1], r.len, p_mask);
    }
    const long long upto = warp_inclusive_scan(need);
    const long long all = __shfl_sync(0xffffffffu, upto, 31);
    for (unsigned left = __ballot_sync(0xffffffffu, lost); left;) {
      const int src = 31 - __clz(left);
      left ^= 1u << src;
      const long long n = __shfl_sync(0xffffffffu, need, src);
      const long long from = end - all + __shfl_sync(0xffffffffu, upto, src) - n;
      for (long long k = n; k > 0; k -= 32) {  // 32 entries, the last ones first
        const long long at = k - 1 - lane;
        const int page = at >= 0 ? *entry(from + at) : 0;
        __syncwarp();
        if (at >= 0) *entry(to - n + at) = page;
        __syncwarp();
      }
      to -= n;
    }
    end -= all;
  }
  return taken - to;
}

// Sums of one block over the batch, valid in every thread afterwards.
struct Sums {
  unsigned long long need, fresh, all_need, all_fresh;
};

__global__ void __launch_bounds__(kSlotThreads) map_slots_kernel(const SlotArgs a) {
  __shared__ unsigned long long s_sum[4][kSlotThreads / 32];
  __shared__ long long s_ring[3];
  const int b = blockIdx.y;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const Request me = load_request(a, b);
  int32_t* row = a.req_to_token + (me.bad ? 0 : me.row) * a.row_stride;
  const int p_mask = (1 << a.shift) - 1;
  const long long old_pages = (me.len + p_mask) >> a.shift;
  // The page the row ends in, if it ends inside one.
  const bool partial = !me.bad && (me.len & p_mask) != 0;
  const int last = partial ? row[me.len - 1] : 0;
  if (tid == 0) {
    s_ring[0] = a.ring_state[0];
    s_ring[1] = a.ring_state[1];
    s_ring[2] = s_ring[0] % a.ring_capacity;
  }
  Sums s = {0, 0, 0, 0};
  bool unsized = false;
  for (int i = tid; i < a.batch; i += kSlotThreads) {
    const Request r = load_request(a, i);
    s.all_need += r.need;
    s.all_fresh += r.fresh;
    if (i < b) {
      s.need += r.need;
      s.fresh += r.fresh;
    }
    unsized |= r.unsized;
  }
  s.need = warp_sum(s.need);
  s.fresh = warp_sum(s.fresh);
  s.all_need = warp_sum(s.all_need);
  s.all_fresh = warp_sum(s.all_fresh);
  if (lane == 0) {
    s_sum[0][warp] = s.need;
    s_sum[1][warp] = s.fresh;
    s_sum[2][warp] = s.all_need;
    s_sum[3][warp] = s.all_fresh;
  }
  unsized = __syncthreads_or(unsized) && a.keep;
  s = Sums{0, 0, 0, 0};
#pragma unroll
  for (int w = 0; w < kSlotThreads / 32; ++w) {
    s.need += s_sum[0][w];
    s.fresh += s_sum[1][w];
    s.all_need += s_sum[2][w];
    s.all_fresh += s_sum[3][w];
  }
  const long long head = s_ring[0];
  const bool short_ring = (long long)s.all_need > s_ring[1] - head;
  const bool over = (long long)s.all_fresh > a.capacity;
  const bool none = over || unsized;            // the outputs list no token
  const bool refused = short_ring || none;  // of the whole call: no slot is given out
  // A row whose last slot does not sit at its offset of a page cannot go on.
  const bool bad_page = partial && off_page(last, me.len, p_mask);
  const bool give = !refused && !bad_page && !me.bad;
  int st = 0;
  if (me.bad) st |= AKV_SLOTS_BAD_REQUEST;
  if (bad_page) st |= AKV_SLOTS_BAD_PAGE;

  // Pages given out are free ones, fewer than the ring holds: the index wraps
  // at most once.
  const long long first = s_ring[2] + (long long)s.need;
  auto fresh_page = [&](long long k) {
    const long long at = first + k;
    return a.ring[at < a.ring_capacity ? at : at - a.ring_capacity];
  };
  const int start = blockIdx.x * kSlotThreads + tid, step = gridDim.x * kSlotThreads;
  const long long next = me.bad ? 0  // no position to go on from
                         : a.next_positions ? ld_index(a.next_positions, b, a.next_is64)
                                            : me.len;
  const long long out0 = (long long)s.fresh;

  // New tokens.  With a tree they are one warp's work (64 nodes at most, two
  // per lane): ancestors by pointer doubling, six rounds of mask |=
  // mask[up], up = up[up] over shuffles, which is as quick for a chain of 64
  // nodes as for a flat tree.
  if (a.parents != nullptr) {
    if (blockIdx.x == 0 && warp == 0 && me.fresh > 0) {
      int up[2];
      unsigned long long mask[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        up[h] = -1;
        mask[h] = 1ull << i;
        if (i < me.fresh && out0 + i < a.capacity) {
          up[h] = a.parents[out0 + i];
          if (up[h] < -1 || up[h] >= i) {  // not above the node: a root
            st |= AKV_SLOTS_BAD_PARENT;
            up[h] = -1;
          }
        }
      }
#pragma unroll
      for (int round = 0; round < 6; ++round) {
        int nu[2];
        unsigned long long nm[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int src = up[h] & 31;
          const unsigned long long m0 = __shfl_sync(0xffffffffu, mask[0], src);
          const unsigned long long m1 = __shfl_sync(0xffffffffu, mask[1], src);
          const int u0 = __shfl_sync(0xffffffffu, up[0], src);
          const int u1 = __shfl_sync(0xffffffffu, up[1], src);
          const bool hi = up[h] >= 32, root = up[h] < 0;
          nm[h] = root ? mask[h] : mask[h] | (hi ? m1 : m0);
          nu[h] = root ? -1 : (hi ? u1 : u0);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          mask[h] = nm[h];
          up[h] = nu[h];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = lane + 32 * h;
        if (i >= me.fresh || out0 + i >= a.capacity) continue;
        const long long t = me.len + i, g = t >> a.shift;
        int slot = -1;
        if (give) {
          const int page = g < old_pages ? last >> a.shift : fresh_page(g - old_pages);
          slot = (page << a.shift) | (int)(t & p_mask);
          row[t] = slot;
        }
        a.slots[out0 + i] = slot;
        a.positions[out0 + i] = (int32_t)(next + __popcll(mask[h]) - 1);
        a.tree_mask[out0 + i] = (int64_t)mask[h];
      }
    }
  } else {
    for (long long i = start; i < me.fresh && out0 + i < a.capacity; i += step) {
      const long long t = me.len + i, g = t >> a.shift;
      int slot = -1;
      if (give) {
        const int page = g < old_pages ? last >> a.shift : fresh_page(g - old_pages);
        slot = (page << a.shift) | (int)(t & p_mask);
        row[t] = slot;
      }
      a.slots[out0 + i] = slot;
      a.positions[out0 + i] = (int32_t)(next + i);
    }
  }

  // Behind the last token no slot and no position of an earlier call stays: a
  // caller may pass the whole vectors on with padded rows.  Entries that hold
  // neither are left as they are.
  {
    const long long stride = (long long)gridDim.y * step;
    for (long long i = (long long)s.all_fresh + (long long)b * step + start; i < a.capacity;
         i += 4 * stride) {
      int slot[4], position[4];  // all loads before the first store
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = i + k * stride < a.capacity;
        slot[k] = in ? a.slots[i + k * stride] : -1;
        position[k] = in ? a.positions[i + k * stride] : 0;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (slot[k] >= 0) a.slots[i + k * stride] = -1;
        if (position[k] > 0) a.positions[i + k * stride] = 0;
      }
    }
  }

  // Block table: the pages of [0, L) from the row, the fresh ones from the
  // ring (the row's new columns are being written by this launch).
  if (a.block_table != nullptr && give) {
    int32_t* out = a.block_table + (long long)b * a.table_stride;
    const int old = (int)old_pages, pages = (int)(old_pages + me.need);
    int g = start;
    // Pages of one slot are a copy: 16 bytes a load where both rows allow it.
    if (a.shift == 0 &&
        ((reinterpret_cast<uintptr_t>(row) | reinterpret_cast<uintptr_t>(out)) & 15) == 0) {
      const int4* from = reinterpret_cast<const int4*>(row);
      int4* to = reinterpret_cast<int4*>(out);
      const int quads = old >> 2;
      int i = start;
      for (; i + 3 * step < quads; i += 4 * step) {
        int4 id[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) id[k] = from[i + k * step];
#pragma unroll
        for (int k = 0; k < 4; ++k) to[i + k * step] = id[k];
      }
      for (; i < quads; i += step) to[i] = from[i];
      g += 4 * quads;
    }
    // Four entries at a time, their loads all before the first store.
    for (; g + 3 * step < old; g += 4 * step) {
      int id[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) id[k] = row[(long long)(g + k * step) << a.shift] >> a.shift;
#pragma unroll
      for (int k = 0; k < 4; ++k) out[g + k * step] = id[k];
    }
    for (; g < pages; g += step)
      out[g] = g < old ? row[(long long)g << a.shift] >> a.shift : fresh_page(g - old);
  }

  if (blockIdx.x == 0 && tid == 0) {
    a.new_offsets[b] = (int32_t)(none ? 0 : s.fresh);
    if (b == a.batch - 1) {
      a.new_offsets[a.batch] = (int32_t)(none ? 0 : s.all_fresh);
      a.totals[0] = (int32_t)(none ? 0 : s.all_fresh);
      a.totals[1] = (int32_t)(refused ? 0 : s.all_need);
      if (short_ring) st |= AKV_SLOTS_RING_UNDERFLOW;
      if (over) st |= AKV_SLOTS_CAPACITY;
    }
  }
  // Status bits gather in arrivals[1] and the last block publishes them (so
  // a call leaves its own status, not a sum over calls) and, with commit,
  // takes the pages: every block has read the ring by then.
  if (st) atomicOr(a.arrivals + 1, (unsigned)st);
  __syncthreads();
  if (warp == 0) {
    int bits = -1;
    if (lane == 0) {
      __threadfence();
      const unsigned blocks = gridDim.x * gridDim.y;
      if (atomicInc(a.arrivals, blocks - 1) == blocks - 1)
        bits = (int)atomicExch(a.arrivals + 1, 0u);
    }
    bits = __shfl_sync(0xffffffffu, bits, 0);
    if (bits < 0) return;  // not the last block
    long long taken = (long long)s.all_need;
    if (a.commit && !refused && (bits & AKV_SLOTS_BAD_PAGE)) {
      __threadfence();
      taken -= return_pages(a, head, taken, lane);
      if (lane == 0) a.totals[1] = (int32_t)taken;
    }
    if (lane == 0) {
      *a.status = bits;
      if (a.commit && !refused) a.ring_state[0] = head + taken;
    }
  }
}

}  // namespace
}  // namespace akv

extern "C" int64_t akv_map_slots_args_bytes(void) { return sizeof(akv_map_slots_args); }

extern "C" int akv_map_slots(const akv_map_slots_args* args, void* stream) {
  AKV_NVTX_RANGE("akv_map_slots");
  using namespace akv;
  if (args == nullptr) return AKV_ERR_INVALID;
  const akv_map_slots_args& x = *args;
  const int64_t page = x.page_size;
  if (x.batch < 0 || x.batch > 65535 || x.rows < 0 || x.columns < 0 || x.row_stride < x.columns ||
      x.ring_capacity <= 0 || x.capacity < 0 || x.capacity > INT32_MAX || page <= 0 ||
      page > 128 || (page & (page - 1)) || page == 2 ||
      (x.block_table && (x.table_columns < 0 || x.table_columns > INT32_MAX / 2 ||
                         x.table_stride < x.table_columns)))
    return AKV_ERR_INVALID;
  if (x.batch == 0) return AKV_OK;
  if (!x.req_to_token || !x.row_ids || !x.raw_lens || !x.new_lens || !x.ring || !x.ring_state ||
      !x.new_offsets || !x.totals || !x.status || !x.workspace ||
      (x.capacity > 0 && (!x.slots || !x.positions)) ||
      (x.parents && x.capacity > 0 && !x.tree_mask))
    return AKV_ERR_INVALID;
  int shift = 0;
  while ((1 << shift) < page) ++shift;
  const int batch = (int)x.batch;
  const bool keep = (x.commit & ~int64_t(1)) == AKV_SLOTS_KEEP_OFFSETS;
  SlotArgs a{x.req_to_token, x.row_stride, x.rows, x.columns, x.row_ids, x.row_ids_is64 != 0,
             x.raw_lens, x.raw_lens_is64 != 0, x.new_lens, x.new_lens_is64 != 0, batch, shift,
             x.ring, reinterpret_cast<long long*>(x.ring_state), x.ring_capacity,
             x.next_positions, x.next_is64 != 0, x.parents, x.capacity, x.new_offsets, x.slots,
             x.positions, x.tree_mask, x.block_table, x.table_stride, x.table_columns, x.totals,
             x.status, x.workspace, keep ? (int)(x.commit & 1) : x.commit != 0, keep};
  // Blocks per request: enough for about six per SM over the batch, no more than its
  // tokens, its table row or its share of the entries behind the last token can use
  // (a capacity of 131,072, one request's tree: one block 178 us, these 5).
  const long long longest =
      std::max<long long>(x.parents ? (x.capacity + batch - 1) / batch : x.capacity,
                          x.block_table ? x.table_columns : 1);
  const long long want = (longest + 4 * kSlotThreads - 1) / (4 * kSlotThreads);
  const long long fit = std::max(1, kNumSMs * 6 / batch);
  const dim3 grid((unsigned)std::max<long long>(1, std::min(want, fit)), batch);
  map_slots_kernel<<<grid, kSlotThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return launch_status();
}
