// Block tables and slot maps of a paged cache, built on the GPU from request
// lengths, and the return of finished requests' pages.
//
// Request b has c_b cached tokens on ceil(c_b / P) pages of P tokens and gets
// n_b more. It takes need_b = ceil((c_b + n_b) / P) - ceil(c_b / P) pages from a
// ring of free pages, in request order: with the exclusive prefix sums
// first_b = sum_{a<b} need_a the pages are ring[(head + first_b + i) mod size].
// Token j of request b sits at position p = c_b + j, slot page(p / P) * P + p mod
// P, and at row cu_b + j of the packed tensors, cu = prefix sums of n.
//
// Latency bounds a decode step (a few KB), the 12 bytes written a token a long
// prefill. So it is ONE launch without any wait between CTAs: every CTA scans
// the lengths itself (a few KB from L2, kept in shared memory) and then fills its
// own share of the slots and table entries, finding a token's request by binary
// search. A token on a page that this call allocates takes the page number from
// the ring, never from the table row that another CTA is writing. All or
// nothing: where pages, table columns or slots run out nothing is allocated and
// the device error word says so, since the host is not asked.
#include <cuda_runtime.h>

#include "common.cuh"
#include "kv4_layout.cuh"
#include "tilemix_b200.h"

namespace tilemix {
namespace tables {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kMaxBatch = 8192;
constexpr int kFew = 16;  // new tokens a request that a thread fills in by itself

struct Args {
  const int32_t* cached;
  const int32_t* fresh;
  int32_t* table;
  int64_t table_stride;
  int cols;
  const int32_t* ring;
  int64_t capacity;
  const int64_t* span;
  int batch, page;
  int64_t n_slots;
  int64_t* slots;
  int32_t* positions;
  int32_t* cu;
  int32_t* kv_lens;
  int64_t* span_out;
  int vec;  // slots and positions take 16-byte stores
  int* err;
};

// Largest b with start[b] <= i (start ascending, start[0] = 0): the request that owns item i.
__device__ __forceinline__ int owner(const int32_t* start, int n, int32_t i) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (start[mid] <= i)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// kRun: consecutive tokens a thread fills in. 4 where stores are the work (mostly of one request and one page:
// one lookup, whole 16-byte stores), 1 where the chain of lookups is.
template <int kRun>
__global__ void __launch_bounds__(kThreads) build_kernel(const Args a) {
  extern __shared__ int32_t sh[];
  int32_t* s_cu = sh;                     // [batch + 1] token offsets
  int32_t* s_first = sh + a.batch + 1;    // [batch + 1] page offsets
  __shared__ long long part_tok[kWarps], part_page[kWarps];
  __shared__ int bad, crowded;  // some length is impossible; some request has many new tokens
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad = crowded = 0;
  __syncthreads();

  // Exclusive scan of (n_b, need_b): each thread owns a run of requests. Sums in 64 bits, so that
  // lengths that cannot be served do not wrap into ones that can.
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  const long long most = static_cast<long long>(a.cols) * a.page;
  const long long head = a.span[0], tail = a.span[1];
  long long tok = 0, pages = 0;
  bool mine_bad = false, many = false;
  for (int b = b0; b < b1; ++b) {
    const long long c = a.cached[b], n = a.fresh[b];
    if (c < 0 || n < 0 || c + n > most || c + n > 0x7fffffffll - a.page) {
      mine_bad = true;
      continue;
    }
    tok += n;
    pages += (c + n + a.page - 1) / a.page - (c + a.page - 1) / a.page;
    many |= n > kFew;
  }
  if (mine_bad) bad = 1;
  if (many) crowded = 1;
  long long inc_tok = tok, inc_page = pages;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, inc_tok, o), p = __shfl_up_sync(0xffffffffu, inc_page, o);
    if (lane >= o) {
      inc_tok += t;
      inc_page += p;
    }
  }
  if (lane == 31) {
    part_tok[warp] = inc_tok;
    part_page[warp] = inc_page;
  }
  __syncthreads();
  long long base_tok = 0, base_page = 0, all_tok = 0, all_page = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) {
      base_tok += part_tok[w];
      base_page += part_page[w];
    }
    all_tok += part_tok[w];
    all_page += part_page[w];
  }
  const bool fail = bad != 0 || head < 0 || tail < head || tail - head > a.capacity || all_page > tail - head ||
                    all_tok > a.n_slots;
  if (!fail) {
    long long t = base_tok + inc_tok - tok, p = base_page + inc_page - pages;
    for (int b = b0; b < b1; ++b) {
      const long long c = a.cached[b], n = a.fresh[b];
      s_cu[b] = static_cast<int32_t>(t);
      s_first[b] = static_cast<int32_t>(p);
      t += n;
      p += (c + n + a.page - 1) / a.page - (c + a.page - 1) / a.page;
    }
    if (tid == 0) {
      s_cu[a.batch] = static_cast<int32_t>(all_tok);
      s_first[a.batch] = static_cast<int32_t>(all_page);
    }
  }
  __syncthreads();

  if (blockIdx.x == 0) {
    for (int b = tid; b < a.batch; b += kThreads) {
      a.cu[b] = fail ? 0 : s_cu[b];
      a.kv_lens[b] = a.cached[b] + (fail ? 0 : a.fresh[b]);
    }
    if (tid == 0) {
      a.cu[a.batch] = fail ? 0 : s_cu[a.batch];
      a.span_out[0] = head + (fail ? 0 : all_page);
      a.span_out[1] = tail;
      if (fail) record_error(a.err, kErrCachePlan);
    }
  }

  const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * kThreads + tid;
  // the capacity fits 31 bits; a counter of pages ever taken rarely needs the long division
  const int64_t head0 = fail || a.capacity == 0 ? 0
                        : head <= 0xffffffffll  ? static_cast<uint32_t>(head) % static_cast<uint32_t>(a.capacity)
                                                : head % a.capacity;
  auto from_ring = [&](int64_t off) {
    const int64_t at = head0 + off;
    return a.ring[at >= a.capacity ? at - a.capacity : at];
  };
  if (!fail) {
    for (int64_t i = first; i < all_page; i += stride) {
      const int b = owner(s_first, a.batch, static_cast<int32_t>(i));
      const int held = (a.cached[b] + a.page - 1) / a.page;
      a.table[b * a.table_stride + held + (i - s_first[b])] = from_ring(i);
    }
  }
  // A decode step (one CTA, a few tokens a request): each thread fills in its own requests' tokens, without a
  // search.
  if (kRun == 1 && gridDim.x == 1 && !fail && !crowded) {
    long long row = base_tok + inc_tok - tok, need = base_page + inc_page - pages;
    for (int b = b0; b < b1; ++b) {
      const int c = a.cached[b], n = a.fresh[b], held = (c + a.page - 1) / a.page;
      int col = c / a.page, at = c - col * a.page;
      int32_t page = -1;
      for (int k = 0; k < n; ++k) {
        if (k == 0 || at == a.page) {
          if (at == a.page) ++col, at = 0;
          page = col < held ? a.table[b * a.table_stride + col] : from_ring(need + col - held);
          if (page < 0) record_error(a.err, kErrCachePage);
        }
        a.slots[row + k] = page < 0 ? -1 : static_cast<int64_t>(page) * a.page + at;
        a.positions[row + k] = c + k;
        ++at;
      }
      row += n;
      need += (c + n + a.page - 1) / a.page - held;
    }
    for (int64_t i = all_tok + tid; i < a.n_slots; i += kThreads) {
      a.slots[i] = -1;
      a.positions[i] = 0;
    }
    return;
  }
  for (int64_t i0 = kRun * first; i0 < a.n_slots; i0 += kRun * stride) {
    long long s4[kRun];
    int p4[kRun];
    int left = 0;  // tokens that still belong to the page at hand
#pragma unroll
    for (int k = 0; k < kRun; ++k) {
      const int64_t i = i0 + k;
      s4[k] = -1;
      p4[k] = 0;
      if (fail || i >= all_tok) continue;
      if (k > 0 && left > 0) {
        s4[k] = s4[k - 1] < 0 ? -1 : s4[k - 1] + 1;
        p4[k] = p4[k - 1] + 1;
        --left;
        continue;
      }
      const int b = owner(s_cu, a.batch, static_cast<int32_t>(i));
      const int c = a.cached[b];
      const int held = (c + a.page - 1) / a.page;
      p4[k] = c + static_cast<int32_t>(i) - s_cu[b];
      const int col = p4[k] / a.page, in_page = p4[k] - col * a.page;
      const int32_t page = col < held ? a.table[b * a.table_stride + col] : from_ring(s_first[b] + col - held);
      if (page >= 0)
        s4[k] = static_cast<int64_t>(page) * a.page + in_page;
      else
        record_error(a.err, kErrCachePage);
      left = min(a.page - in_page, s_cu[b + 1] - static_cast<int32_t>(i)) - 1;
    }
    if (kRun == 4 && a.vec && i0 + 4 <= a.n_slots) {
      reinterpret_cast<longlong2*>(a.slots + i0)[0] = make_longlong2(s4[0], s4[kRun > 1 ? 1 : 0]);
      reinterpret_cast<longlong2*>(a.slots + i0)[1] = make_longlong2(s4[kRun > 2 ? 2 : 0], s4[kRun > 3 ? 3 : 0]);
      *reinterpret_cast<int4*>(a.positions + i0) =
          make_int4(p4[0], p4[kRun > 1 ? 1 : 0], p4[kRun > 2 ? 2 : 0], p4[kRun > 3 ? 3 : 0]);
    } else {
#pragma unroll
      for (int k = 0; k < kRun; ++k)
        if (i0 + k < a.n_slots) {
          a.slots[i0 + k] = s4[k];
          a.positions[i0 + k] = p4[k];
        }
    }
  }
}

struct ReleaseArgs {
  int32_t* lens;
  const uint8_t* done;
  int32_t* table;
  int64_t table_stride;
  int cols;
  int32_t* ring;
  int64_t capacity;
  int64_t* span;
  int batch, page;
  int* err;
};

// One CTA: finished requests are rare, and the lengths, the table and the ring's end are changed in
// place. A thread walks the pages of its requests: 0.3 ms for 256 requests of 8192 tokens on pages of 16, 1.1 ms
// for one of 131,072, bound by the chain of a load and two stores a page. Pages go back in request order, so the
// ring's content does not depend on the schedule.
__global__ void __launch_bounds__(kThreads) release_kernel(const ReleaseArgs a) {
  __shared__ long long part[kWarps];
  __shared__ int bad;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (tid == 0) bad = 0;
  __syncthreads();
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = min(tid * per, a.batch), b1 = min(b0 + per, a.batch);
  long long mine = 0;
  bool mine_bad = false;
  for (int b = b0; b < b1; ++b) {
    if (!a.done[b]) continue;
    const long long held = (static_cast<long long>(a.lens[b]) + a.page - 1) / a.page;
    if (a.lens[b] < 0 || held > a.cols)
      mine_bad = true;
    else
      mine += held;
  }
  if (mine_bad) bad = 1;
  long long inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long t = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += t;
  }
  if (lane == 31) part[warp] = inc;
  __syncthreads();
  long long base = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    if (w < warp) base += part[w];
    all += part[w];
  }
  const long long head = a.span[0], tail = a.span[1];
  const bool fail = bad != 0 || head < 0 || tail < head || tail - head + all > a.capacity;
  __syncthreads();  // every thread has read the span before it changes
  if (fail) {
    if (tid == 0) record_error(a.err, kErrCachePlan);
    return;
  }
  long long at = tail + base + inc - mine;
  for (int b = b0; b < b1; ++b) {
    if (!a.done[b]) continue;
    const int held = static_cast<int>((static_cast<long long>(a.lens[b]) + a.page - 1) / a.page);
    int32_t* row = a.table + b * a.table_stride;
    for (int i = 0; i < held; ++i, ++at) {
      a.ring[at % a.capacity] = row[i];
      row[i] = -1;
    }
    a.lens[b] = 0;
  }
  if (tid == 0) a.span[1] = tail + all;
}

}  // namespace tables
}  // namespace tilemix

extern "C" int tm_build_block_tables(const tm_block_tables_params* p, int* error_flag, void* stream) {
  using namespace tilemix::tables;
  if (p == nullptr) return TM_ERR_NULL;
  if (p->batch < 0 || p->n_slots < 0 || p->cols < 0 || p->capacity < 0) return TM_ERR_SHAPE;
  if (p->page_size < 16 || p->page_size % 16 != 0) return TM_ERR_SHAPE;
  if (!p->free_span || !p->free_span_out || !p->cu_seqlens) return TM_ERR_NULL;
  if (p->batch > 0 && (!p->cached_lens || !p->new_lens || !p->kv_lens)) return TM_ERR_NULL;
  if (p->n_slots > 0 && (!p->slots || !p->positions)) return TM_ERR_NULL;
  if (p->batch > 0 && p->cols > 0 && !p->block_table) return TM_ERR_NULL;
  if (p->capacity > 0 && !p->free_pages) return TM_ERR_NULL;
  // The scan's two arrays live in shared memory; token and page offsets are 32-bit.
  if (p->batch > kMaxBatch || p->n_slots > 0x7fffffffll || p->capacity > 0x7fffffffll) return TM_ERR_UNSUPPORTED;
  if ((p->batch > 0 && (p->kv_lens == p->cached_lens || p->kv_lens == p->new_lens)) || p->free_span_out == p->free_span)
    return TM_ERR_UNSUPPORTED;  // other CTAs still read the inputs while the outputs are written
  Args a{p->cached_lens, p->new_lens,  p->block_table, p->table_stride, p->cols,        p->free_pages,
         p->capacity,    p->free_span, p->batch,       p->page_size,    p->n_slots,     p->slots,
         p->positions,   p->cu_seqlens, p->kv_lens,    p->free_span_out,
         tilemix::kv4::aligned(p->slots, 16) && tilemix::kv4::aligned(p->positions, 16), error_flag};
  const size_t smem = 2 * sizeof(int32_t) * (static_cast<size_t>(p->batch) + 1);
  constexpr int kMostSmem = 2 * 4 * (kMaxBatch + 1);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  // One CTA for what a decode step has; else one token a thread until every SM has its threads, four beyond
  // (557,056 tokens: 10.3 us at two a thread, 8.0 at four; 256 single tokens: 6.8 and 11).
  if (p->n_slots <= 148 * kThreads) {
    if (!tilemix::allow_smem<build_kernel<1>, kMostSmem>()) return TM_ERR_LAUNCH;
    const int64_t ctas = p->n_slots <= 4 * kThreads ? 1 : (p->n_slots + kThreads - 1) / kThreads;
    build_kernel<1><<<static_cast<unsigned>(ctas), kThreads, smem, st>>>(a);
  } else {
    if (!tilemix::allow_smem<build_kernel<4>, kMostSmem>()) return TM_ERR_LAUNCH;
    const int64_t want = (p->n_slots + 4 * kThreads - 1) / (4 * kThreads);
    build_kernel<4><<<static_cast<unsigned>(want > 296 ? 296 : want), kThreads, smem, st>>>(a);
  }
  return cudaGetLastError() == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}

extern "C" int tm_release_pages(int32_t* lens, const uint8_t* done, int32_t* block_table, int64_t table_stride,
                                int cols, int32_t* free_pages, int64_t capacity, int64_t* free_span, int batch,
                                int page_size, int* error_flag, void* stream) {
  using namespace tilemix::tables;
  if (batch < 0 || cols < 0 || capacity < 0) return TM_ERR_SHAPE;
  if (page_size < 16 || page_size % 16 != 0) return TM_ERR_SHAPE;
  if (batch == 0) return TM_OK;
  if (!lens || !done || !free_span || (cols > 0 && !block_table) || (capacity > 0 && !free_pages)) return TM_ERR_NULL;
  if (capacity > 0x7fffffffll) return TM_ERR_UNSUPPORTED;
  ReleaseArgs a{lens, done, block_table, table_stride, cols, free_pages, capacity, free_span, batch, page_size,
                error_flag};
  release_kernel<<<1, kThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
  return cudaGetLastError() == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}
