// Ragged batches over the page pool for MI355X (gfx950), behind include/barq_ragged.h: block tables and slot
// maps built from the requests' lengths, and packed tokens stored through a slot map.
//
// map_slots_kernel.  Request i of row r (length L, mark W in a pool) gets n_i tokens at positions L .. L + n_i - 1.
// Its blocks j in [ceil(W / P), ceil((L + n_i) / P)) are new; ranked over all requests in (request, block)
// order, rank k takes free_pages[top - 1 - k].  The ranks are a prefix sum over at most 256 requests, which every
// workgroup forms for itself from the rows' device state (one request a thread): no workgroup waits for
// another.  A token's page is then the block table's entry where the block is not new, else the free stack's.
// Of a pool's workgroups, the last to have read the state commits it (the pool's arrival counter), while the
// others still write slots: they no longer read what the commit changes.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <new>

#include "barq_kv.h"
#include "barq_kv_commit.h"
#include "barq_ragged.h"
#include "fastdiv.h"

namespace {

using barq_commit::ceil_div_fd;
using barq_commit::checked_page;
using barq_commit::wave_incl_scan;

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kMapRequests = kThreads;  // requests of a launch: one a thread
constexpr int kMapPools = 32;           // pools of a launch (its arguments stay below 4 KB)
constexpr int64_t kI32Max = 0x7fffffff;

struct MapPool {  // the row metadata of a barq_kv_pool
  int32_t* block_table;
  int32_t* seq_lens;
  int32_t* high_water;
  const int32_t* free_pages;
  int32_t* ctrl;
  int64_t num_pages;
};

struct MapArgs {
  MapPool pools[kMapPools];
  int64_t* slots;
  int64_t slot_stride;
  int32_t* positions;
  int32_t* requests;
  int32_t* offsets;
  FastDiv div_page;
  int32_t max_blocks;
  int32_t n;            // requests
  int32_t base;         // the first request's number, of a call in several launches
  int32_t shared;       // this launch writes positions, requests and offsets
  int32_t chunk;        // tokens of a workgroup
  int32_t off[kMapRequests + 1];  // tokens before each request, from the call's first request on
  int32_t row[kMapRequests];
};
static_assert(sizeof(MapArgs) <= 4096, "kernel arguments");

// The last request r of [lo, n) whose tokens (or ranks) start at or before x: off[r] <= x < off[n].
__device__ __forceinline__ int request_of(const int32_t* off, int lo, int n, int x) {
  int hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (off[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__global__ void __launch_bounds__(kThreads) map_slots_kernel(const MapArgs a) {
  __shared__ int32_t s_off[kMapRequests + 1], s_len[kMapRequests], s_first[kMapRequests], s_row[kMapRequests];
  __shared__ int32_t s_rank[kMapRequests + 1], s_sum[kThreads / kWave], s_last;
  const MapPool& p = a.pools[blockIdx.y];
  const int tid = (int)threadIdx.x, mb = a.max_blocks, P = (int)a.div_page.d;
  int len = 0, hw = 0, row = 0, first = 0, news = 0, count = 0, err = 0;
  if (tid < a.n) {
    row = a.row[tid];
    len = p.seq_lens[row];
    hw = p.high_water[row];
    s_off[tid] = a.off[tid];
    count = a.off[tid + 1] - a.off[tid];
    first = ceil_div_fd(hw, a.div_page);
    const int end = ceil_div_fd(len + count, a.div_page);
    if (count > 0) news = max(0, min(end, mb) - first);
    if (end > mb) err |= BARQ_KV_ERRBIT_CAPACITY;
    s_len[tid] = len;
    s_first[tid] = first;
    s_row[tid] = row;
  }
  if (tid == 0) s_off[a.n] = a.off[a.n];
  const int top = p.ctrl[BARQ_KV_CTRL_FREE_TOP];
  const int incl = wave_incl_scan(news);
  if ((tid & (kWave - 1)) == kWave - 1) s_sum[tid / kWave] = incl;
  __syncthreads();
  int before = 0, total_new = 0;
#pragma unroll
  for (int w = 0; w < kThreads / kWave; ++w) {
    if (w < tid / kWave) before += s_sum[w];
    total_new += s_sum[w];
  }
  s_rank[tid] = before + incl - news;
  if (tid == 0) {
    s_rank[a.n] = total_new;
    // Every thread's reads of the rows' state and of the stack's top have returned: they fed the barrier's
    // shared memory.  (s_rank[n] may be thread n's own entry: the same value.)
    s_last = atomicAdd(&p.ctrl[BARQ_KV_CTRL_ARRIVED], 1) == (int)gridDim.x - 1;
  }
  __syncthreads();
  if (s_last) {
    if (tid < a.n) {
      p.seq_lens[row] = len + count;
      p.high_water[row] = max(hw, len + count);
    }
    if (tid == 0) {
      p.ctrl[BARQ_KV_CTRL_FREE_TOP] = max(0, top - total_new);
      atomicExch(&p.ctrl[BARQ_KV_CTRL_ARRIVED], 0);
    }
  }
  if (a.shared && blockIdx.y == 0 && blockIdx.x == 0 && a.offsets) {
    if (tid < a.n) a.offsets[a.base + tid] = a.off[tid];
    if (tid == 0) a.offsets[a.base + a.n] = a.off[a.n];
  }
  // this workgroup's share of the new blocks
  for (int k = (int)blockIdx.x * kThreads + tid; k < total_new; k += (int)gridDim.x * kThreads) {
    const int r = request_of(s_rank, 0, a.n, k);
    const int page = top - 1 - k >= 0 ? checked_page(p.free_pages[top - 1 - k], p.num_pages) : -1;
    if (page < 0) err |= BARQ_KV_ERRBIT_POOL_EXHAUSTED;
    p.block_table[(int64_t)s_row[r] * mb + s_first[r] + (k - s_rank[r])] = page;
  }
  // and of the tokens
  const int t0 = s_off[0] + (int)blockIdx.x * a.chunk;
  const int t1 = min(t0 + a.chunk, s_off[a.n]);
  int64_t* slots = a.slots + (int64_t)blockIdx.y * a.slot_stride;
  int r = -1;
  for (int t = t0 + tid; t < t1; t += kThreads) {
    if (r < 0 || s_off[r + 1] <= t) r = request_of(s_off, r + 1, a.n, t);
    const int pos = s_len[r] + t - s_off[r];
    const int blk = (int)a.div_page.div((uint32_t)pos);
    int page = -1;
    if (blk < mb) {
      const int idx = top - 1 - (s_rank[r] + blk - s_first[r]);
      if (blk < s_first[r]) page = p.block_table[(int64_t)s_row[r] * mb + blk];
      else if (idx >= 0) page = p.free_pages[idx];
      page = checked_page(page, p.num_pages);
    }
    slots[t] = page < 0 ? -1 : (int64_t)page * P + (pos - blk * P);
    if (a.shared && blockIdx.y == 0) {
      if (a.positions) a.positions[t] = pos;
      if (a.requests) a.requests[t] = a.base + r;
    }
  }
  if (err) atomicOr(&p.ctrl[BARQ_KV_CTRL_ERRORS], err);
}

// ---------------------------------------------------------------------------------- stores through a slot map
template <int VB>
struct VecT;
template <>
struct VecT<16> { using T = uint32_t __attribute__((ext_vector_type(4))); };
template <>
struct VecT<8> { using T = uint32_t __attribute__((ext_vector_type(2))); };
template <>
struct VecT<4> { using T = uint32_t; };
template <>
struct VecT<2> { using T = uint16_t; };
template <>
struct VecT<1> { using T = uint8_t; };

struct WriteArgs {
  const int64_t* slots;
  const int64_t* index;
  const char* key;
  const char* value;
  char* key_pages;
  char* value_pages;
  int32_t* errors;
  int64_t num_slots, num_tokens;
  int64_t items;                // vectors of the launch: whole tokens, below 2^31
  int64_t stride_n, stride_h;   // bytes
  int64_t tok_bytes;
  int64_t first_token;
  FastDiv div_vecs;             // vectors of a token
  FastDiv div_head;             // vectors of a head
};

constexpr int kWriteItems = 4;  // vectors of K and of V a thread has in flight

// One vector of a token's K and the same of its V a step: a thread's loads of four tokens' pieces are in
// flight together, and the lanes of a wave take adjacent vectors of one token row.
template <int VB>
__global__ void __launch_bounds__(kThreads) write_slots_kernel(const WriteArgs a) {
  using V = typename VecT<VB>::T;
  const int64_t i0 = (int64_t)blockIdx.x * (kThreads * kWriteItems) + threadIdx.x;
  int64_t slot[kWriteItems], src[kWriteItems];
  int col[kWriteItems];
#pragma unroll
  for (int u = 0; u < kWriteItems; ++u) {
    const uint32_t i = (uint32_t)min(i0 + u * kThreads, a.items - 1);
    const uint32_t t = a.div_vecs.div(i);
    const int64_t j = a.first_token + t;
    col[u] = (int)(i - t * a.div_vecs.d);
    slot[u] = a.slots[j];
    src[u] = a.index ? a.index[j] : j;
  }
  V k[kWriteItems], v[kWriteItems];
  bool live[kWriteItems], bad = false;
#pragma unroll
  for (int u = 0; u < kWriteItems; ++u) {
    const bool in = src[u] >= 0 && src[u] < a.num_tokens && slot[u] < a.num_slots;
    bad |= !in && slot[u] >= 0;
    live[u] = in && slot[u] >= 0 && i0 + u * kThreads < a.items;
    const uint32_t h = a.div_head.div((uint32_t)col[u]);
    const int64_t at = (in ? src[u] : 0) * a.stride_n + (int64_t)h * a.stride_h +
                       (int64_t)((uint32_t)col[u] - h * a.div_head.d) * VB;
    k[u] = __builtin_nontemporal_load((const V*)(a.key + at));
    v[u] = __builtin_nontemporal_load((const V*)(a.value + at));
  }
#pragma unroll
  for (int u = 0; u < kWriteItems; ++u) {
    if (!live[u]) continue;
    const int64_t at = slot[u] * a.tok_bytes + (int64_t)col[u] * VB;
    __builtin_nontemporal_store(k[u], (V*)(a.key_pages + at));
    __builtin_nontemporal_store(v[u], (V*)(a.value_pages + at));
  }
  if (bad) atomicOr(a.errors, BARQ_KV_ERRBIT_BAD_INDEX);
}

bool pool_ok(const barq_kv_pool* p) {
  if (!p || !p->key_pages || !p->value_pages || !p->block_table || !p->seq_lens || !p->high_water || !p->free_pages ||
      !p->ctrl || ((uintptr_t)p->ctrl & 255u) || p->num_pages < 1 || p->max_batch < 1 || p->max_blocks < 1 ||
      p->page_size < 1 || p->kv_heads < 1 || p->head_dim < 1)
    return false;
  if (!(p->elem_bytes == 1 || p->elem_bytes == 2 || p->elem_bytes == 4 || p->elem_bytes == 8)) return false;
  return p->num_pages <= kI32Max && p->max_batch * p->max_blocks <= kI32Max && p->max_blocks * p->page_size <= kI32Max &&
         p->kv_heads * p->head_dim * p->elem_bytes * p->page_size <= kI32Max;
}

int launch(const void* kernel, dim3 grid, void* args, void* stream) {
  void* list[] = {args};
  if (hipLaunchKernel(kernel, grid, dim3(kThreads), list, 0, (hipStream_t)stream) == hipSuccess) return BARQ_KV_OK;
  (void)hipGetLastError();
  return BARQ_KV_ERR_LAUNCH;
}

// Whether rows (of n requests) are distinct and in range, by one bit a row.
bool rows_ok(const int32_t* rows, int64_t n, int64_t max_batch) {
  uint64_t small[16] = {};
  const int64_t words = (max_batch + 63) / 64;
  uint64_t* seen = words <= 16 ? small : new (std::nothrow) uint64_t[words]();
  bool ok = seen != nullptr;
  for (int64_t i = 0; ok && i < n; ++i) {
    const int64_t r = rows[i];
    ok = r >= 0 && r < max_batch && !(seen[r / 64] >> (r % 64) & 1);
    if (ok) seen[r / 64] |= uint64_t(1) << (r % 64);
  }
  if (seen != small) delete[] seen;
  return ok;
}

}  // namespace

extern "C" {

int barq_map_slots(const barq_kv_pool* pools, int64_t num_pools, const int32_t* rows, const int32_t* lengths,
                   int64_t num_rows, int64_t* slots, int64_t slot_stride, int32_t* positions, int32_t* requests,
                   int32_t* offsets, void* stream) {
  if (!pools || num_pools < 1 || num_rows < 0) return BARQ_KV_ERR_INVALID;
  const barq_kv_pool& g = pools[0];
  for (int64_t l = 0; l < num_pools; ++l) {
    const barq_kv_pool& p = pools[l];
    if (!pool_ok(&p) || p.max_batch != g.max_batch || p.max_blocks != g.max_blocks || p.page_size != g.page_size)
      return BARQ_KV_ERR_INVALID;
    for (int64_t m = 0; m < l; ++m)
      if (pools[m].ctrl == p.ctrl || pools[m].seq_lens == p.seq_lens) return BARQ_KV_ERR_INVALID;
  }
  if (num_rows > g.max_batch || (num_rows > 0 && !lengths)) return BARQ_KV_ERR_INVALID;
  if (num_rows == 0) return BARQ_KV_OK;
  int64_t total = 0;
  for (int64_t i = 0; i < num_rows; ++i) {
    if (lengths[i] < 0 || lengths[i] > g.max_blocks * g.page_size) return BARQ_KV_ERR_INVALID;
    total += lengths[i];
  }
  if (total >= (int64_t(1) << 30) || (rows && !rows_ok(rows, num_rows, g.max_batch)) ||
      (total > 0 && (!slots || (num_pools > 1 && slot_stride < total))))
    return BARQ_KV_ERR_INVALID;
  int rc = BARQ_KV_OK;
  for (int64_t l0 = 0; l0 < num_pools && rc == BARQ_KV_OK; l0 += kMapPools) {
    const int set = (int)std::min<int64_t>(kMapPools, num_pools - l0);
    int32_t at = 0;
    for (int64_t i0 = 0; i0 < num_rows && rc == BARQ_KV_OK; i0 += kMapRequests) {
      MapArgs a = {};
      for (int k = 0; k < set; ++k) {
        const barq_kv_pool& p = pools[l0 + k];
        a.pools[k] = MapPool{p.block_table, p.seq_lens, p.high_water, p.free_pages, p.ctrl, p.num_pages};
      }
      a.slots = slots + l0 * slot_stride;
      a.slot_stride = slot_stride;
      a.positions = positions;
      a.requests = requests;
      a.offsets = offsets;
      a.div_page = FastDiv::make((uint32_t)g.page_size);
      a.max_blocks = (int32_t)g.max_blocks;
      a.n = (int32_t)std::min<int64_t>(kMapRequests, num_rows - i0);
      a.base = (int32_t)i0;
      a.shared = l0 == 0;
      const int32_t from = at;
      for (int i = 0; i < a.n; ++i) {
        a.off[i] = at;
        a.row[i] = rows ? rows[i0 + i] : (int32_t)(i0 + i);
        at += lengths[i0 + i];
      }
      a.off[a.n] = at;
      // 2,048 tokens a workgroup, more where the launch would pass 2,048 workgroups.
      const int64_t most = std::max<int64_t>(1, 2048 / set);
      a.chunk = (int32_t)std::max<int64_t>(2048, (at - from + most - 1) / most);
      const uint32_t tiles = (uint32_t)std::max<int64_t>(1, ((int64_t)(at - from) + a.chunk - 1) / a.chunk);
      rc = launch((const void*)&map_slots_kernel, dim3(tiles, (uint32_t)set), &a, stream);
    }
  }
  return rc;
}

int barq_write_slots(const barq_kv_pool* pool, const int64_t* slots, const int64_t* index, int64_t count,
                     const void* key, const void* value, int64_t num_tokens, int64_t stride_n, int64_t stride_h,
                     void* stream) {
  if (!pool_ok(pool) || count < 0 || num_tokens < 0 || stride_n < 0 || stride_h < 0) return BARQ_KV_ERR_INVALID;
  if (count == 0) return BARQ_KV_OK;
  if (!slots || !key || !value || num_tokens < 1 || (!index && num_tokens < count)) return BARQ_KV_ERR_INVALID;
  const int64_t es = pool->elem_bytes, head = pool->head_dim * es, tok = pool->kv_heads * head;
  uint64_t bits = (uint64_t)head | (uint64_t)(stride_n * es) | (uint64_t)(uintptr_t)key |
                  (uint64_t)(uintptr_t)value | (uint64_t)(uintptr_t)pool->key_pages |
                  (uint64_t)(uintptr_t)pool->value_pages;
  if (pool->kv_heads > 1) bits |= (uint64_t)(stride_h * es);
  int vb = 16;
  while (bits & (uint64_t)(vb - 1)) vb >>= 1;
  WriteArgs a;
  a.slots = slots;
  a.index = index;
  a.key = (const char*)key;
  a.value = (const char*)value;
  a.key_pages = (char*)pool->key_pages;
  a.value_pages = (char*)pool->value_pages;
  a.errors = pool->ctrl + BARQ_KV_CTRL_ERRORS;
  a.num_slots = pool->num_pages * pool->page_size;
  a.num_tokens = num_tokens;
  a.stride_n = stride_n * es;
  a.stride_h = stride_h * es;
  a.tok_bytes = tok;
  a.div_vecs = FastDiv::make((uint32_t)(tok / vb));
  a.div_head = FastDiv::make((uint32_t)(head / vb));
  const void* kernel = vb == 16  ? (const void*)&write_slots_kernel<16>
                       : vb == 8 ? (const void*)&write_slots_kernel<8>
                       : vb == 4 ? (const void*)&write_slots_kernel<4>
                       : vb == 2 ? (const void*)&write_slots_kernel<2>
                                 : (const void*)&write_slots_kernel<1>;
  const int64_t vecs = tok / vb, step = std::max<int64_t>(1, (int64_t(1) << 30) / vecs);  // tokens of a launch
  int rc = BARQ_KV_OK;
  for (a.first_token = 0; a.first_token < count && rc == BARQ_KV_OK; a.first_token += step) {
    a.items = std::min(step, count - a.first_token) * vecs;
    const int64_t blocks = (a.items + kThreads * kWriteItems - 1) / (kThreads * kWriteItems);
    rc = launch(kernel, dim3((uint32_t)blocks), &a, stream);
  }
  return rc;
}

}  // extern "C"
