// Attention over the paged 4-bit key/value cache (kv4_layout.cuh): a few query
// tokens a request against all of its cached keys.
//
//   o_r = sum_j softmax_j(scale q_r . k_j) v_j,  k_j = s n + m, v_j likewise,
// in one pass with the running maximum and sum of the softmax. Rows are the
// (query token, query head) pairs that share a KV head, 8 a tile.
//
// The cache's bytes bound it (5 bits a value; 4 D FLOPs per 1.25 D bytes and
// row is far from any tensor-core limit), so what matters is that the loads never
// pause and that the codes are unpacked in few instructions:
//   * the key axis is split over CTAs, and inside a CTA over warps; each warp has
//     its own ring of bulk copies (32 keys a stage, K and V and their scales
//     adjacent in one block) and its own softmax state, so no warp ever waits for
//     another before the end;
//   * keys are the M side of mma.m16n8k16 (S^T = K Q^T, O^T = V^T P^T): 8 rows
//     fill N, so a group of 3 to 8 query heads wastes little, where rows on the M
//     side would fill 16. tcgen05 would need the unpacked operand written to
//     shared memory first, which costs more than the unpacking itself;
//   * a lane's share of a row is one shared-memory load in the order the operands
//     want. Scores come from the codes themselves, masked out of the word as fp16
//     subnormals, with scale and minimum in fp32: k is never rounded. A v is made
//     from its code by OR-ing it into the mantissa of 1024, one exact add (or FMA)
//     and one FMA with the group's scale and minimum, which rounds it to fp16 once
//     (the tensor core's operand type); p is rounded to fp16 as the prefill's
//     kernels do, times 2^15; scores, maxima, sums and the output accumulate in fp32.
// 64 requests of 512 to 8192 keys (24 query heads, 8 of 128 cached): 84 us, 4.2
// TB/s, where the bytes alone would take 54; one request of 131,072 keys 45 us (26).
// What bounds it is a step's instructions, the unpacking of V first among them,
// issued in 57 % of the cycles by the three warps a scheduler that the registers
// leave room for. More rows than a tile has pass over the keys again and unpack
// them anew: 2048 new tokens behind 16,384 keys take 2.5 ms, 180 TFLOP/s.
// Rows with no key left give 0. Keys past the length or masked are excluded by
// selecting, and a V of theirs that is not finite by a zero scale, so infinities
// and NaN there do not leak.
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "kv4_layout.cuh"
#include "tilemix_b200.h"

namespace tilemix {
namespace kv4 {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kStages = 2;  // 10 KB a warp in flight, 120 KB an SM; three measured no faster
constexpr int kStepBlocks = 2;                        // 16-key blocks a step
constexpr int kStepKeys = kStepBlocks * kBlockTokens;
constexpr int kChunkKeys = kStepKeys * kAttnWarps;    // keys of one step of every warp: the unit of work
constexpr int kSms = 148;
// What a run of chunks costs beside its chunks (queries, pages, merge and store), in chunks. Without it a CTA
// with several short requests was the last to end: 64 requests of 512 to 8192 keys took 94 us, 82 so (89 with 1, 83
// with 2).
constexpr int kSetup = 4;

// The softmax weights and their sums carry a factor of 2^15, which cancels in the end: the largest is 2^15 instead of 1,
// still exact in fp16, and a weight keeps fp16's 11 bits down to 2^-29 of the largest. Without it those under 2^-14
// lost bits and those under 2^-25 all of them: behind one key that drew nearly all of a row, 8192 keys of 2^-25.5 of its
// weight each came out a quarter too small.
constexpr float kWeightBits = 15.f;

// CTAs an SM of the kernel for head_dim d and nt row tiles, by registers and shared memory.
constexpr int resident(int d, int nt) { return d == 128 && nt == 2 ? 2 : 3; }

struct AttnArgs {
  const __half* q;
  int64_t q_st, q_sh;
  const uint8_t* pool;
  int64_t pages;
  int64_t page_stride;  // bytes from page to page (all heads)
  int page_bytes;       // bytes of one head of a page
  int page_blocks;      // 16-token blocks a page
  const int32_t* table;
  int64_t table_stride;
  int cols;
  const int32_t* kv_lens;
  const int32_t* cu;  // NULL: one query token a request
  const uint8_t* mask;
  int64_t mask_stride;
  int mask_cols;
  __half* out;
  int64_t o_st, o_sh;
  int64_t q_tokens;
  int batch, heads_q, heads_k, group;
  int max_q;
  int64_t max_kv;  // most keys a request may have: its bound and its table row's
  int causal;
  float scale_log2;
  int ctas;            // CTAs that share the work
  int32_t* starts;     // [batch + 1] first chunk of each request, written by CTA 0 for the join
  float* part_o;       // [2 ctas][rows of a tile][D]
  float2* part_ml;     // [2 ctas][rows of a tile] (max in log2 units, sum)
  int* err;
};

// A request's share of the work.
struct Request {
  int q0, n_q;   // its query tokens, at most max_q of them
  int kv;        // its keys, at most max_kv of them
  int tiles;     // row tiles a KV head
  int chunks;    // chunks of kChunkKeys keys of one (KV head, row tile), at least 1
  int cost;      // those and kSetup, times the KV heads and row tiles: its length in the work list
};

template <int NT>
__device__ __forceinline__ Request request_of(const AttnArgs& a, int b) {
  Request r;
  r.q0 = b;
  int q1 = b + 1;
  if (a.cu != nullptr) {
    r.q0 = a.cu[b];
    q1 = a.cu[b + 1];
  }
  // the subtraction may wrap where one of the two is negative, and is not used then
  r.n_q = min(static_cast<int>(static_cast<uint32_t>(q1) - static_cast<uint32_t>(r.q0)), a.max_q);
  if (r.q0 < 0 || q1 < r.q0 || r.q0 + static_cast<int64_t>(r.n_q) > a.q_tokens) r.n_q = 0;
  r.kv = static_cast<int>(min(static_cast<int64_t>(max(a.kv_lens[b], 0)), a.max_kv));
  r.tiles = (r.n_q * a.group + 8 * NT - 1) / (8 * NT);
  r.chunks = max(1, (r.kv + kChunkKeys - 1) / kChunkKeys);
  r.cost = r.tiles * a.heads_k * (r.chunks + kSetup);
  return r;
}

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// D = A B
__device__ __forceinline__ void mma16816_new(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}

// D = A[16 x 8] B[8 x 8]
__device__ __forceinline__ void mma1688(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm(
      "mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0), "f"(0.f));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t lop_and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(m), "r"(o));  // (x & m) | o
  return y;
}

__device__ __forceinline__ __half2 as_h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Codes of a word as fp16 subnormals, n 2^-24 in the even pairs and 16 n 2^-24 in the odd ones: pair i holds nibbles i
// and i + 4. One instruction a pair, and the tensor core multiplies subnormals exactly.
__device__ __forceinline__ void spread8(uint32_t w, uint32_t (&o)[4]) {
  const uint32_t w8 = w >> 8;
  o[0] = w & 0x000F000Fu;
  o[1] = w & 0x00F000F0u;
  o[2] = w8 & 0x000F000Fu;
  o[3] = w8 & 0x00F000F0u;
}

// The values s n + m of a word's codes as fp16 pairs (s, m of the pair's two halves): the codes in the mantissa of
// 1024, brought to n exactly, one FMA.
__device__ __forceinline__ void unpack8(uint32_t w, __half2 s, __half2 m, uint32_t (&o)[4]) {
  const __half2 k1024 = as_h2(0x64006400u), r16 = as_h2(0x2C002C00u), k64 = as_h2(0xD400D400u);  // 1024, 1/16, -64
  const uint32_t magic = 0x64006400u, w8 = w >> 8;
  o[0] = as_u32(__hfma2(__hsub2(as_h2(lop_and_or(w, 0x000F000Fu, magic)), k1024), s, m));
  o[1] = as_u32(__hfma2(__hfma2(as_h2(lop_and_or(w, 0x00F000F0u, magic)), r16, k64), s, m));
  o[2] = as_u32(__hfma2(__hsub2(as_h2(lop_and_or(w8, 0x000F000Fu, magic)), k1024), s, m));
  o[3] = as_u32(__hfma2(__hfma2(as_h2(lop_and_or(w8, 0x00F000F0u, magic)), r16, k64), s, m));
}

template <int N>
struct Words {
  uint32_t w[N];
};

template <int N>
__device__ __forceinline__ Words<N> load_words(const uint8_t* p) {
  Words<N> r;
  if constexpr (N == 4) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
  } else if constexpr (N == 2) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    r.w[0] = v.x, r.w[1] = v.y;
  } else {
    r.w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
  return r;
}

// The work of a call is the list of all chunks: by request, then KV head, then row tile, then key, with kSetup
// places in front of each (KV head, row tile). CTA c takes places [c per, (c + 1) per), whatever requests they
// belong to, so ragged lengths leave no CTA behind; a (KV head, row tile) that several CTAs share leaves partial
// states for the join, one that a CTA has whole is written at once. A CTA's first run of chunks may continue another's (slot 2 c), its last may be continued
// (slot 2 c + 1).
template <int D, int NT>
__global__ void __launch_bounds__(kAttnThreads, resident(D, NT)) attn_kernel(const AttnArgs a) {
  using L = Layout<D>;
  constexpr int G = L::kGroups;
  constexpr int kRows = 8 * NT;
  constexpr int kStageBytes = kStepBlocks * L::kBlockBytes;
  constexpr int kState = NT * (8 * G + 4);  // floats of a lane's state (o, m, l)
  extern __shared__ __align__(128) uint8_t smem[];
  float* sh_state = reinterpret_cast<float*>(smem + kAttnWarps * kStages * kStageBytes);  // [warps][kState][32]
  __shared__ __align__(8) uint64_t bars[kAttnWarps][kStages];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;
  // Set up beside the kernel before (programmatic dependent launch), whose end is waited for before anything is
  // read; then the join may be set up in the same way.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  uint8_t* ring = smem + warp * kStages * kStageBytes;
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    fence_mbarrier_init();
  }

  // Where this CTA's chunks begin: every warp scans the requests for itself, a run of them a lane.
  const int run = (a.batch + 31) / 32;
  const int rb0 = min(lane * run, a.batch), rb1 = min(rb0 + run, a.batch);
  int mine = 0;
  for (int b = rb0; b < rb1; ++b) {
    const Request r = request_of<NT>(a, b);
    mine += r.cost;
  }
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  const int total = __shfl_sync(0xffffffffu, inc, 31);
  const int per = (total + a.ctas - 1) / a.ctas;
  int pos = per * static_cast<int>(blockIdx.x);
  const int end = min(total, pos + per);
  if (blockIdx.x == gridDim.x - 1 && warp == kAttnWarps - 1) {  // for the join; this CTA has the least to do
    int at = inc - mine;
    for (int b = rb0; b < rb1; ++b) {
      a.starts[b] = at;
      const Request r = request_of<NT>(a, b);
      at += r.cost;
      // more keys or query tokens than the call said there may be, offsets that are not rows of q in order, a negative
      // length: what is beyond is left out
      if (r.kv != a.kv_lens[b] || r.q0 < 0 || (a.cu != nullptr && a.cu[b + 1] != static_cast<int64_t>(r.q0) + r.n_q))
        record_error(a.err, kErrCachePlan);
    }
    if (lane == 0) a.starts[a.batch] = total;
  }
  if (pos >= end) return;
  int b = 0, b_start = 0;
  const int owner = __ffs(__ballot_sync(0xffffffffu, inc > pos)) - 1;
  if (lane == owner) {
    b = rb0;
    b_start = inc - mine;
    while (true) {
      const Request r = request_of<NT>(a, b);
      if (pos < b_start + r.cost) break;
      b_start += r.cost;
      ++b;
    }
  }
  b = __shfl_sync(0xffffffffu, b, owner);
  b_start = __shfl_sync(0xffffffffu, b_start, owner);
  Request rq = request_of<NT>(a, b);

  // The current run of chunks: one (request, KV head, row tile), keys [key0, key1).
  int hk, row0, chunk0, n_chunks, key0, blk1, steps;
  // false: the CTA's range ends in front of the next chunk
  auto locate = [&]() {
    const int off = pos - b_start;
    const int unit = off / (rq.chunks + kSetup), in_unit = off - unit * (rq.chunks + kSetup);
    const int lead = max(0, kSetup - in_unit);
    chunk0 = max(0, in_unit - kSetup);
    n_chunks = min(rq.chunks - chunk0, end - pos - lead);
    if (n_chunks <= 0) return false;
    pos += lead + n_chunks;
    hk = unit / rq.tiles;
    row0 = (unit - hk * rq.tiles) * kRows;
    key0 = chunk0 * kChunkKeys;
    const int key1 = min(rq.kv, key0 + n_chunks * kChunkKeys);
    blk1 = (key1 + kBlockTokens - 1) / kBlockTokens;
    const int all_steps = (blk1 - key0 / kBlockTokens + kStepBlocks - 1) / kStepBlocks;
    steps = all_steps > warp ? (all_steps - warp + kAttnWarps - 1) / kAttnWarps : 0;
    return true;
  };
  if (!locate()) return;

  // Bulk copies of the warp's steps: blocks key0 / 16 + 2 (warp + kAttnWarps i). Each lane looks up one step of
  // the next 32 (its pages, the addresses of its blocks) and issues that step's copies itself when its turn
  // comes, so a step costs a few instructions. Steps of all runs count on through the ring's stages.
  const uint8_t* src[kStepBlocks];  // the lane's step; NULL: past the run's end, or its page is outside the pool
  bool joined = false;              // the lane's two blocks are adjacent: one copy
  uint32_t absent[kStepBlocks];     // bit i: step i of the 32 lacks the block (a step past the end is none)
  int issued = 0;                   // steps of the current run whose copies are under way
  int in_stage = 0;                 // stage of the next step to issue
  uint32_t stage_bad = 0;           // bit (kStepBlocks stage + block): not in the stage
  int all_issued = 0;
  auto first_of = [&](int i) { return key0 / kBlockTokens + kStepBlocks * (warp + kAttnWarps * i); };
  auto issue = [&]() {
    if ((issued & 31) == 0) {
      const int32_t* row = a.table + b * a.table_stride;
#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u) {
        const int blk = first_of(issued + lane) + u;
        src[u] = nullptr;
        if (blk < blk1) {
          const int col = blk / a.page_blocks;
          const int64_t page = row[col];
          if (page >= 0 && page < a.pages)
            src[u] = a.pool + page * a.page_stride + static_cast<int64_t>(hk) * a.page_bytes +
                     static_cast<int64_t>(blk - col * a.page_blocks) * L::kBlockBytes;
          else
            record_error(a.err, kErrCachePage);
        }
        absent[u] = __ballot_sync(0xffffffffu, src[u] == nullptr && first_of(issued + lane) < blk1);
      }
      joined = src[0] != nullptr && src[1] == src[0] + L::kBlockBytes;
    }
    if ((absent[0] | absent[1] | stage_bad) != 0) {
      uint32_t bad = 0;
#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u) bad |= ((absent[u] >> (issued & 31)) & 1u) << u;
      const int at = kStepBlocks * in_stage;
      stage_bad = (stage_bad & ~(((1u << kStepBlocks) - 1) << at)) | bad << at;
    }
    if (lane == (issued & 31)) {
      uint8_t* dst = ring + in_stage * kStageBytes;
      uint64_t* full = &bar[in_stage];
      if (joined) {
        mbar_arrive_expect_tx(full, kStageBytes);
        bulk_load(dst, src[0], kStageBytes, full);
      } else {
        mbar_arrive_expect_tx(full, ((src[0] != nullptr) + (src[1] != nullptr)) * L::kBlockBytes);
#pragma unroll
        for (int u = 0; u < kStepBlocks; ++u)
          if (src[u] != nullptr) bulk_load(dst + u * L::kBlockBytes, src[u], L::kBlockBytes, full);
      }
    }
    ++issued;
    ++all_issued;
    in_stage = in_stage == kStages - 1 ? 0 : in_stage + 1;
  };
  __syncwarp();
  while (issued < steps && issued < kStages) issue();

  // Operand rows of the mma <-> tokens of a block: rows 2 i, 2 i + 1 (+ 8) are tokens i, i + 4 (+ 8), so
  // that the four keys of a lane's V operand are t, t + 4, t + 8, t + 12 and a quad reads whole rows.
  const int tok_g = (g >> 1) + (g & 1) * 4;
  int s = 0;           // stage of the next step to consume, and its phase
  uint32_t phase = 0;
  bool ok = true;

  while (true) {
    // Queries as the B operand: tile x, column g = row row0 + 8 x + g, the K order of a lane's channels.
    // Scores are formed from the codes themselves, as subnormals: s (q' . n 2^-24) + m (sum q' 2^-24), the
    // group's scale applied in fp32, its minimum in an mma as (m, m 2^-10) times the sum as two fp16 numbers (the
    // rest after the first times 2^10, clear of the subnormals). Channels on odd nibbles, 16 n, have q' / 16. q' is
    // q times a power of two that brings the row's largest magnitude to [2^14, 2^15): q' / 16 keeps its bits.
    // Padding rows are 0.
    uint32_t qf[NT][2 * G][2], qsum[NT];
    float cs[NT][2];     // log2 units a score unit of columns 2 t and 2 t + 1
    int lim[NT][2];                 // keys [0, lim) visible to them; padding rows see what the last row sees
    const int n_rows = rq.n_q * a.group;
    // Keys in front of the request's first query token, by the lengths as they were given: max_q and max_kv leave tokens
    // and keys out and do not move the others. Query token i sees before + i + 1 keys, which is at most the length.
    // Looked up anew for each run: held with the request it cost a register of the loop below (64 requests of 512 to
    // 8192 keys: 88 us, 86 so).
    const int before = max(a.kv_lens[b], 0) - (a.cu != nullptr ? a.cu[b + 1] - a.cu[b] : 1);
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int r = row0 + 8 * x + g;
      const __half* qr = a.q + static_cast<int64_t>(rq.q0 + r / a.group) * a.q_st +
                         static_cast<int64_t>(hk * a.group + r % a.group) * a.q_sh;
      uint4 v[G];
      float top = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        v[j] = make_uint4(0, 0, 0, 0);
        if (r < n_rows) v[j] = __ldg(reinterpret_cast<const uint4*>(qr + 32 * j + 8 * t));
        const __half2 m2 = __hmax2(__hmax2(__habs2(as_h2(v[j].x)), __habs2(as_h2(v[j].y))),
                                   __hmax2(__habs2(as_h2(v[j].z)), __habs2(as_h2(v[j].w))));
        top = fmaxf(top, fmaxf(__low2float(m2), __high2float(m2)));
      }
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // 2^(14 - floor(log2 top)) by its exponent bits
      const uint32_t ex = __float_as_uint(top) >> 23;
      const bool norm = top > 0.f && top <= 65504.f;
      const float up = norm ? __uint_as_float((268u - ex) << 23) : 1.f;
      const float down = norm  // its inverse, times 2^24
                              ? __uint_as_float((ex + 10u) << 23) : 16777216.f;
      float sum_j = 0.f;
#pragma unroll
      for (int j = 0; j < G; ++j) {
        const float2 c01 = __half22float2(as_h2(v[j].x)), c23 = __half22float2(as_h2(v[j].y));
        const float2 c45 = __half22float2(as_h2(v[j].z)), c67 = __half22float2(as_h2(v[j].w));
        const float u16 = up * 0.0625f;
        const __half2 p0 = __floats2half2_rn(c01.x * up, c45.x * up), p1 = __floats2half2_rn(c01.y * u16, c45.y * u16);
        const __half2 p2 = __floats2half2_rn(c23.x * up, c67.x * up), p3 = __floats2half2_rn(c23.y * u16, c67.y * u16);
        qf[x][2 * j][0] = as_u32(p0);
        qf[x][2 * j][1] = as_u32(p1);
        qf[x][2 * j + 1][0] = as_u32(p2);
        qf[x][2 * j + 1][1] = as_u32(p3);
        const float2 f0 = __half22float2(p0), f1 = __half22float2(p1), f2 = __half22float2(p2), f3 = __half22float2(p3);
        const float lo = f0.x + f0.y + f2.x + f2.y, hi = f1.x + f1.y + f3.x + f3.y;
        float sum = lo + 16.f * hi;
#pragma unroll
        for (int d = 1; d <= 2; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (t == j) sum_j = sum * 5.9604644775390625e-8f;  // 2^-24
      }
      const __half sum_hi = __float2half_rn(sum_j);
      qsum[x] = as_u32(__halves2half2(sum_hi, __float2half_rn((sum_j - __half2float(sum_hi)) * 1024.f)));
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int src = (2 * t + c) * 4;
        cs[x][c] = fmaxf(a.scale_log2 * __shfl_sync(0xffffffffu, down, src), 1.17549435e-38f);  // > 0: -inf stays -inf
        const int rc = min(row0 + 8 * x + 2 * t + c, n_rows - 1);
        lim[x][c] = a.causal ? min(rq.kv, before + rc / a.group + 1) : rq.kv;
      }
    }
    int lim_lo = rq.kv, lim_hi = rq.kv;
    if (a.causal) {
      lim_lo = min(rq.kv, before + row0 / a.group + 1);
      lim_hi = min(rq.kv, before + (min(row0 + kRows, n_rows) - 1) / a.group + 1);
    }
    const uint8_t* mask = a.mask != nullptr ? a.mask + b * a.mask_stride : nullptr;

    float o[NT][2 * G][4];
    // Running maximum in the scores' units, and in log2 units less kWeightBits (-inf and 0 while there is none), and
    // running sum. The maximum moves with every larger score: letting it lag by up to 2^8 saved rescales (83 us against
    // 85 for 64 requests of 512 to 8192 keys), but then the heaviest weight is no longer a power of two, exact in fp16
    // (error 3.2e-4 against 2.9e-4).
    float m[NT][2], mc[NT][2], l[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x) {
#pragma unroll
      for (int i = 0; i < 2 * G; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[x][i][c] = 0.f;
#pragma unroll
      for (int c = 0; c < 2; ++c) m[x][c] = -CUDART_INF_F, mc[x][c] = 0.f, l[x][c] = 0.f;
    }

    // One step: 32 keys from stage s; `live`: those that count for any row.
    // What a step does for keys that do not count is kept to two short branches: a second copy of the whole step
    // without them ran no faster where it was used, and the last step of every run then met cold instructions
    // (64 ragged requests 96 us, 84 with lengths that fill their steps).
    auto step = [&](const int key, const uint32_t live) {
      uint8_t* st = ring + s * kStageBytes;
      if (live != 0xffffffffu || (lim_lo < lim_hi && key + kStepKeys > lim_lo)) {
        // Keys that do not count, or only for some rows, have a weight of 0, and 0 times a V that is not finite
        // (infinities, NaN, what an absent block's stage happens to hold) would be NaN: its scale and minimum become
        // 0, and the rows that do see it get the NaN here. Where all are finite nothing is stored, and the next copy
        // into the stage needs no fence.
        uint8_t* vs = st + lane / kBlockTokens * L::kBlockBytes + L::kOffVScale;
        auto sm_of = [&](int j) { return reinterpret_cast<uint16_t*>(vs + L::v_scale(j, lane % kBlockTokens)); };
        // 15 s + |m| is finite under these (2^11, 2^15); beyond, an unused token's bytes may stand for an infinity
        auto beyond = [](const uint16_t* sm, int s, int m) { return (sm[0] & 0x7FFF) >= s || (sm[4] & 0x7FFF) >= m; };
        bool any = false;
#pragma unroll
        for (int j = 0; j < G; ++j) any |= beyond(sm_of(j), 0x6800, 0x7800);
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
          for (int j = 0; j < G; ++j) {
            uint16_t* sm = sm_of(j);
            const bool bad = beyond(sm, 0x7C00, 0x7C00);
            const uint32_t keys = __ballot_sync(0xffffffffu, bad) & live;
            if (bad || !((live >> lane) & 1)) sm[0] = sm[4] = 0;
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const int n = lim[x][c] - key;
                const uint32_t sees = n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
                if (keys & sees)
                  o[x][2 * j][c] = o[x][2 * j][c + 2] = o[x][2 * j + 1][c] = o[x][2 * j + 1][c + 2] = CUDART_NAN_F;
              }
          }
          fence_proxy_async_smem();  // before the next copy into this stage
          __syncwarp();
        }
      }

      float sc[kStepBlocks][NT][4];
#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u) {
        const uint8_t* blk = st + u * L::kBlockBytes;
        const uint8_t* ks = blk + L::kOffKScale + tok_g * L::kScaleBytes;
        const Words<G> ka = load_words<G>(blk + tok_g * L::kRowBytes + t * (4 * G));
        const Words<G> kb = load_words<G>(blk + (tok_g + 8) * L::kRowBytes + t * (4 * G));
        const Words<G> sa = load_words<G>(ks), sb = load_words<G>(ks + 8 * L::kScaleBytes);
        const uint32_t ma = *reinterpret_cast<const uint32_t*>(ks + t % G * 4);
        const uint32_t mb = *reinterpret_cast<const uint32_t*>(ks + 8 * L::kScaleBytes + t % G * 4);
        const __half2 halves = as_h2(0x14003C00u);  // 1, 2^-10
        const __half2 m_a = __hmul2(__high2half2(as_h2(ma)), halves), m_b = __hmul2(__high2half2(as_h2(mb)), halves);
#pragma unroll
        for (int x = 0; x < NT; ++x)
          mma1688(sc[u][x], as_u32(m_a), as_u32(m_b), qsum[x]);
#pragma unroll
        for (int j = 0; j < G; ++j) {
          uint32_t pa[4], pb[4];
          spread8(ka.w[j], pa);
          spread8(kb.w[j], pb);
          const float fa = __low2float(as_h2(sa.w[j])), fb = __low2float(as_h2(sb.w[j]));
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            float acc[4];
            mma16816_new(acc, pa[0], pb[0], pa[1], pb[1], qf[x][2 * j][0], qf[x][2 * j][1]);
            mma16816(acc, pa[2], pb[2], pa[3], pb[3], qf[x][2 * j + 1][0], qf[x][2 * j + 1][1]);
            sc[u][x][0] = fmaf(fa, acc[0], sc[u][x][0]);
            sc[u][x][1] = fmaf(fa, acc[1], sc[u][x][1]);
            sc[u][x][2] = fmaf(fb, acc[2], sc[u][x][2]);
            sc[u][x][3] = fmaf(fb, acc[3], sc[u][x][3]);
          }
        }
      }

      if (live != 0xffffffffu) {
#pragma unroll
        for (int u = 0; u < kStepBlocks; ++u)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const bool dead = !((live >> (tok_g + kBlockTokens * u + 8 * h)) & 1);
#pragma unroll
            for (int x = 0; x < NT; ++x)
#pragma unroll
              for (int c = 0; c < 2; ++c)
                if (dead) sc[u][x][2 * h + c] = -CUDART_INF_F;
          }
      }
      if (key + kStepKeys > lim_lo) {  // some row's last keys
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int left = lim[x][c] - key - tok_g;  // the row sees this many keys from the lane's first on
#pragma unroll
            for (int u = 0; u < kStepBlocks; ++u)
#pragma unroll
              for (int h = 0; h < 2; ++h)
                if (kBlockTokens * u + 8 * h >= left) sc[u][x][2 * h + c] = -CUDART_INF_F;
          }
      }
      float base[NT][2];
      bool moved = false;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float top = fmaxf(sc[0][x][c], sc[0][x][c + 2]);
#pragma unroll
          for (int u = 1; u < kStepBlocks; ++u) top = fmaxf(top, fmaxf(sc[u][x][c], sc[u][x][c + 2]));
          base[x][c] = top;
          moved |= top > m[x][c];
        }
      // The maxima are joined across the lanes only when some lane's own is beyond the running one.
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          float f[2];
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float top = base[x][c];
#pragma unroll
            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            top = fmaxf(m[x][c], top);
            // By the rounded maxima, which the weights are relative to. m = -inf: nothing summed yet, and 0 stays 0
            const float now = top == -CUDART_INF_F ? 0.f : fmaf(top, cs[x][c], -kWeightBits);
            f[c] = m[x][c] == -CUDART_INF_F ? 0.f : ex2_approx(mc[x][c] - now);
            m[x][c] = top;
            mc[x][c] = now;
            l[x][c] *= f[c];
          }
#pragma unroll
          for (int k = 0; k < 2 * G; ++k) {
            o[x][k][0] *= f[0];
            o[x][k][1] *= f[1];
            o[x][k][2] *= f[0];
            o[x][k][3] *= f[1];
          }
        }
      }

#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u) {
        const uint8_t* blk = st + u * L::kBlockBytes + L::kOffV;
        uint32_t pf[NT][2];
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          float p[4];
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            p[c] = ex2_approx(fmaf(sc[u][x][c], cs[x][c & 1], -mc[x][c & 1]));
            l[x][c & 1] += p[c];
          }
          pf[x][0] = transpose8x8(pack_half2_rn(p[0], p[1]));
          pf[x][1] = transpose8x8(pack_half2_rn(p[2], p[3]));
        }
        constexpr int W = G / 2;  // words of a lane's share of a V row: two groups a word
        Words<W> v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = load_words<W>(blk + (t + 4 * k) * L::kRowBytes + g * (2 * G));
#pragma unroll
        for (int j = 0; j < G; ++j) {
          const Words<4> vs = load_words<4>(blk + 16 * L::kRowBytes + (j * 4 + t) * 16);
          const uint32_t sel = (j & 1) ? 0x7632u : 0x5410u;
          uint32_t e[4], f[4];
          unpack8(__byte_perm(v[0].w[j / 2], v[1].w[j / 2], sel), as_h2(vs.w[0]), as_h2(vs.w[2]), e);
          unpack8(__byte_perm(v[2].w[j / 2], v[3].w[j / 2], sel), as_h2(vs.w[1]), as_h2(vs.w[3]), f);
#pragma unroll
          for (int x = 0; x < NT; ++x) {
            mma16816(o[x][2 * j], e[0], e[1], f[0], f[1], pf[x][0], pf[x][1]);
            mma16816(o[x][2 * j + 1], e[2], e[3], f[2], f[3], pf[x][0], pf[x][1]);
          }
        }
      }
    };

    // The key mask is read two steps ahead: one key of the step a lane (8 requests of several query tokens: 41 us with
    // one step, 39 with two).
    auto mask_of = [&](int i) {
      const int key = key0 + kStepKeys * (warp + kAttnWarps * i) + lane;
      return i < steps && key < min(lim_hi, a.mask_cols) ? static_cast<uint32_t>(mask[key]) : 0u;
    };
    uint32_t mask_now = 0, mask_next = 0;
    if (mask != nullptr) mask_now = mask_of(0), mask_next = mask_of(1);
    // The first steps of a run without a mask are plain: every key counts for every row.
    const int first_key = key0 + kStepKeys * warp, stride = kStepKeys * kAttnWarps;
    const int n_plain = mask != nullptr || lim_lo < first_key + kStepKeys ? 0 : (lim_lo - kStepKeys - first_key) / stride + 1;
    for (int i = 0; i < steps; ++i) {
      const int key = first_key + stride * i;
      uint32_t live = 0xffffffffu;  // which of the step's keys count for any row, a bit each
      if (i >= n_plain || stage_bad != 0) {
        const uint32_t bad = (stage_bad >> (kStepBlocks * s)) & ((1u << kStepBlocks) - 1);
        live = __ballot_sync(0xffffffffu, !((bad >> (lane / kBlockTokens)) & 1) && key + lane < lim_hi &&
                                              (mask == nullptr || mask_now != 0));
        if (mask != nullptr) mask_now = mask_next, mask_next = mask_of(i + 2);
      }
      if (!mbar_wait_spin(&bar[s], phase, a.err, kErrTimeoutFull)) {
        ok = false;
        break;
      }
      step(key, live);
      __syncwarp();  // every lane has read the stage
      if (++s == kStages) s = 0, phase ^= 1;
      if (issued < steps) issue();
    }
    if (!ok) {  // a copy did not arrive: wait (bounded) for what is in flight
      for (int k = 0; k < kStages; ++k)
        if (all_issued > k) mbar_wait(&bar[k], ((all_issued - 1 - k) / kStages) & 1, a.err, kErrTimeoutDrain);
    }
    ok = !__syncthreads_or(!ok);
    if (!ok) return;  // the whole CTA, with the error word set

    // The next run's copies start before this run's states are merged and written.
    const int o_b_q0 = rq.q0, o_row0 = row0, o_hk = hk, o_chunk0 = chunk0;
    const bool whole = chunk0 == 0 && n_chunks == rq.chunks;
    bool more = pos < end;
    if (more) {
      while (pos >= b_start + rq.cost) {
        b_start += rq.cost;
        rq = request_of<NT>(a, ++b);
      }
      more = locate();
    }
    if (more) {
      issued = 0;
      while (issued < steps && issued < kStages) issue();
    }

#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c)  // log2 units from here on, less kWeightBits in all parts
        m[x][c] = m[x][c] == -CUDART_INF_F ? m[x][c] : mc[x][c];
    // Merge the warps' states, a share of the channel groups each.
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[x][c] += __shfl_xor_sync(0xffffffffu, l[x][c], d);
    {
      float* to = sh_state + warp * kState * 32 + lane;
#pragma unroll
      for (int x = 0; x < NT; ++x) {
#pragma unroll
        for (int k = 0; k < 2 * G; ++k)
#pragma unroll
          for (int c = 0; c < 4; ++c) to[(x * 8 * G + 4 * k + c) * 32] = o[x][k][c];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          to[(NT * 8 * G + 4 * x + c) * 32] = m[x][c];
          to[(NT * 8 * G + 4 * x + 2 + c) * 32] = l[x][c];
        }
      }
    }
    __syncthreads();
    if (warp < G) {
      const int j = warp;
      static_assert(G <= kAttnWarps, "a channel group a warp");
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = 8 * x + 2 * t + c;
          if (o_row0 + r >= n_rows) continue;
          const float* from = sh_state + lane;
          float mw[kAttnWarps], top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
          for (int w = 0; w < kAttnWarps; ++w) {
            mw[w] = from[(w * kState + NT * 8 * G + 4 * x + c) * 32];
            top = fmaxf(top, mw[w]);
          }
          const float ref = top == -CUDART_INF_F ? 0.f : top;
          float v[4] = {};  // channels 32 j + 4 g ..
#pragma unroll
          for (int w = 0; w < kAttnWarps; ++w) {
            const float f = ex2_approx(mw[w] - ref);
            sum += f * from[(w * kState + NT * 8 * G + 4 * x + 2 + c) * 32];
#pragma unroll
            for (int i = 0; i < 4; ++i)  // accumulator 2 j + i / 2, row g or g + 8
              v[i] += f * from[(w * kState + x * 8 * G + 4 * (2 * j + i / 2) + c + 2 * (i & 1)) * 32];
          }
          if (whole) {
            const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays
            __half* dst = a.out + static_cast<int64_t>(o_b_q0 + (o_row0 + r) / a.group) * a.o_st +
                          static_cast<int64_t>(o_hk * a.group + (o_row0 + r) % a.group) * a.o_sh + 32 * j + 4 * g;
            *reinterpret_cast<uint2*>(dst) =
                make_uint2(pack_half2_rn(v[0] * inv, v[1] * inv), pack_half2_rn(v[2] * inv, v[3] * inv));
          } else {
            const int64_t at = (2 * static_cast<int64_t>(blockIdx.x) + (o_chunk0 == 0 ? 1 : 0)) * kRows + r;
            *reinterpret_cast<float4*>(a.part_o + at * D + 32 * j + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
            if (g == 0 && j == 0) a.part_ml[at] = make_float2(top, sum);
          }
        }
    }
    if (!more) return;
  }
}

// Joins the partial states of a row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s. One CTA a row, the parts
// dealt to its warps, so that a long request's parts (one from every CTA of the machine) are read in a few
// round trips.
template <int D, int NT>
__global__ void __launch_bounds__(kAttnThreads) join_kernel(const AttnArgs a) {
  constexpr int V = D / 32;  // channels a lane
  __shared__ float sh_o[kAttnWarps][D], sh_m[kAttnWarps], sh_l[kAttnWarps];
  const int b = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Request rq = request_of<NT>(a, b);  // inputs: there since before the attention kernel began
  const int i = blockIdx.x;
  // The attention kernel has ended, its writes are visible. Every CTA waits, those without a row too: the join must
  // not be over before the attention is.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (i >= rq.n_q * a.heads_q) return;
  const int token = i / a.heads_q, hq = i - token * a.heads_q;
  const int hk = hq / a.group, row = token * a.group + hq - hk * a.group;
  const int tile = row / (8 * NT), r = row - tile * (8 * NT);
  const int total = a.starts[a.batch], per = (total + a.ctas - 1) / a.ctas;
  const int first = a.starts[b] + (hk * rq.tiles + tile) * (rq.chunks + kSetup) + kSetup;
  const int c0 = first / per, c1 = (first + rq.chunks - 1) / per;
  if (c0 == c1) return;  // one CTA had it whole and wrote it
  auto slot = [&](int c) { return (2 * static_cast<int64_t>(c) + (c == c0 ? 1 : 0)) * (8 * NT) + r; };
  // Each warp with a running maximum of its own, kFlight parts in flight.
  constexpr int kFlight = 8;
  using Vec = std::conditional_t<V == 4, float4, float2>;
  float acc[V] = {}, sum = 0.f, top = -CUDART_INF_F;
  for (int c = c0 + warp; c <= c1; c += kFlight * kAttnWarps) {
    float2 ml[kFlight];
    Vec v[kFlight];
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const int at_c = c + k * kAttnWarps;
      ml[k] = make_float2(-CUDART_INF_F, 0.f);
      v[k] = Vec{};
      if (at_c <= c1) {
        const int64_t at = slot(at_c);
        ml[k] = a.part_ml[at];
        v[k] = *reinterpret_cast<const Vec*>(a.part_o + at * D + lane * V);
      }
    }
    float now = top;
#pragma unroll
    for (int k = 0; k < kFlight; ++k) now = fmaxf(now, ml[k].x);
    const float ref = now == -CUDART_INF_F ? 0.f : now;
    const float keep = ex2_approx(top - ref);
    sum *= keep;
#pragma unroll
    for (int e = 0; e < V; ++e) acc[e] *= keep;
#pragma unroll
    for (int k = 0; k < kFlight; ++k) {
      const float f = ex2_approx(ml[k].x - ref);  // 0 for a part that is not there
      const float* ve = reinterpret_cast<const float*>(&v[k]);
      sum += f * ml[k].y;
#pragma unroll
      for (int e = 0; e < V; ++e) acc[e] += f * ve[e];
    }
    top = now;
  }
#pragma unroll
  for (int e = 0; e < V; ++e) sh_o[warp][lane * V + e] = acc[e];
  if (lane == 0) sh_m[warp] = top, sh_l[warp] = sum;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= D) return;
  top = sh_m[0];
#pragma unroll
  for (int w = 1; w < kAttnWarps; ++w) top = fmaxf(top, sh_m[w]);
  const float ref = top == -CUDART_INF_F ? 0.f : top;
  float o = 0.f;
  sum = 0.f;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    const float f = ex2_approx(sh_m[w] - ref);
    sum += f * sh_l[w];
    o += f * sh_o[w][d];
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays
  a.out[static_cast<int64_t>(rq.q0 + token) * a.o_st + static_cast<int64_t>(hq) * a.o_sh + d] = __float2half_rn(o * inv);
}

struct Plan {
  int nt, ctas;
  int64_t starts_bytes, part_o_bytes, part_ml_bytes;
  int64_t bytes() const { return starts_bytes + part_o_bytes + part_ml_bytes; }
};

// Two row tiles a CTA where more than 8 rows share a KV head: the unpacking is shared. Four, at head_dim 64, leave two
// CTAs an SM and measured slower (8 requests of up to 15 query tokens: 44 us against 41). As many CTAs as are
// resident at once, or as there can be chunks.
static Plan plan_of(const tm_kv4_attn_params* p) {
  Plan r{};
  const int64_t rows = static_cast<int64_t>(p->max_seqlen_q) * (p->heads_q / p->heads_k);
  r.nt = rows > 8 ? 2 : 1;
  const int64_t tiles = (rows + 8 * r.nt - 1) / (8 * r.nt);
  const int64_t chunks = p->max_kv_len / kChunkKeys + 1 + kSetup;
  const int64_t most = static_cast<int64_t>(p->batch) * p->heads_k * tiles;
  const int64_t slots = kSms * resident(p->head_dim, r.nt);
  r.ctas = static_cast<int>(most >= slots || chunks >= slots || most * chunks >= slots ? slots : most * chunks);
  r.starts_bytes = (static_cast<int64_t>(p->batch) + 4) / 4 * 16;
  r.part_o_bytes = 2ll * r.ctas * 8 * r.nt * p->head_dim * 4;
  r.part_ml_bytes = 2ll * r.ctas * 8 * r.nt * 8;
  return r;
}

static int check(const tm_kv4_attn_params* p) {
  if (p == nullptr) return TM_ERR_NULL;
  if (p->batch < 0 || p->q_tokens < 0 || p->heads_q <= 0 || p->heads_k <= 0 || p->heads_q % p->heads_k != 0)
    return TM_ERR_SHAPE;
  if (p->num_pages < 0 || p->cols < 0 || p->max_seqlen_q < 0 || p->max_kv_len < 0) return TM_ERR_SHAPE;
  if (p->page_size < kBlockTokens || p->page_size % kBlockTokens != 0) return TM_ERR_SHAPE;
  if (p->head_dim != 64 && p->head_dim != 128) return TM_ERR_UNSUPPORTED;
  if (p->batch > 65535 || p->max_seqlen_q > 65535 || p->heads_q > 32767 || p->max_kv_len > (1 << 30))
    return TM_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(p->page_size) * 20 * 128 / kBlockTokens > 0x7fffffffll) return TM_ERR_UNSUPPORTED;
  if (p->batch == 0 || p->q_tokens == 0 || p->max_seqlen_q == 0) return TM_OK;
  if (!p->q || !p->out || !p->kv_lens || (p->num_pages > 0 && !p->pool) || (p->cols > 0 && !p->block_table))
    return TM_ERR_NULL;
  if (p->cu_seqlens_q == nullptr && (p->max_seqlen_q != 1 || p->q_tokens < p->batch)) return TM_ERR_SHAPE;
  if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->pool, 16)) return TM_ERR_ALIGN;
  // of one token or head the stride to the next is never used
  if (p->q_tokens > 1 && (p->q_stride_tok % 8 || p->o_stride_tok % 8)) return TM_ERR_ALIGN;
  if (p->heads_q > 1 && (p->q_stride_head % 8 || p->o_stride_head % 8)) return TM_ERR_ALIGN;
  if (p->key_mask != nullptr && p->mask_cols < 0) return TM_ERR_SHAPE;
  // Positive: maxima are taken before scaling. At most 2^80: |q . k| < 2^40, so a score in log2 units stays finite.
  if (!(p->sm_scale > 0.f) || p->sm_scale > 1.2089258e24f) return TM_ERR_SHAPE;
  // the chunks of the work list are counted in 32 bits, with room for the last CTA's end
  const double rows = static_cast<double>(p->max_seqlen_q) * p->heads_q;
  if (p->batch * (rows / 8 + p->heads_k) * (p->max_kv_len / kChunkKeys + 1.0 + kSetup) > 2147480000.0)
    return TM_ERR_UNSUPPORTED;
  return TM_OK;
}

template <int D, int NT>
static cudaError_t launch(const AttnArgs& a, cudaStream_t st) {
  constexpr int smem = kAttnWarps * kStages * kStepBlocks * Layout<D>::kBlockBytes +
                       kAttnWarps * NT * (8 * Layout<D>::kGroups + 4) * 32 * 4;
  if (!allow_smem<attn_kernel<D, NT>, smem>()) return cudaErrorInvalidValue;
  // Both kernels are set up while the one before them ends (programmatic dependent launch) and wait for it.
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  cfg.stream = st;
  cfg.blockDim = dim3(kAttnThreads);
  cfg.gridDim = dim3(static_cast<unsigned>(a.ctas));
  cfg.dynamicSmemBytes = smem;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, attn_kernel<D, NT>, a);
  if (e != cudaSuccess) return e;
  cfg.gridDim = dim3(static_cast<unsigned>(static_cast<int64_t>(a.max_q) * a.heads_q), static_cast<unsigned>(a.batch));
  cfg.dynamicSmemBytes = 0;
  return cudaLaunchKernelEx(&cfg, join_kernel<D, NT>, a);
}

}  // namespace kv4
}  // namespace tilemix

extern "C" int tm_kv4_attn_workspace(const tm_kv4_attn_params* p, int64_t* bytes) {
  using namespace tilemix::kv4;
  if (bytes == nullptr) return TM_ERR_NULL;
  *bytes = 0;
  const int rc = check(p);
  if (rc != TM_OK || p->batch == 0 || p->q_tokens == 0 || p->max_seqlen_q == 0) return rc;
  *bytes = plan_of(p).bytes();
  return TM_OK;
}

extern "C" int tm_kv4_attn(const tm_kv4_attn_params* p, void* workspace, int64_t workspace_bytes, int* error_flag,
                           void* stream) {
  using namespace tilemix::kv4;
  const int rc = check(p);
  if (rc != TM_OK || p->batch == 0 || p->q_tokens == 0 || p->max_seqlen_q == 0) return rc;
  const Plan r = plan_of(p);
  if (workspace == nullptr) return TM_ERR_NULL;
  if (workspace_bytes < r.bytes()) return TM_ERR_SHAPE;
  if (!aligned(workspace, 16)) return TM_ERR_ALIGN;
  AttnArgs a{};
  a.q = static_cast<const __half*>(p->q);
  a.q_st = p->q_stride_tok;
  a.q_sh = p->q_stride_head;
  a.pool = static_cast<const uint8_t*>(p->pool);
  a.pages = p->num_pages;
  a.page_blocks = p->page_size / kBlockTokens;
  a.page_bytes = a.page_blocks * block_bytes(p->head_dim);
  a.page_stride = static_cast<int64_t>(a.page_bytes) * p->heads_k;
  a.table = p->block_table;
  a.table_stride = p->table_stride;
  a.cols = p->cols;
  a.kv_lens = p->kv_lens;
  a.cu = p->cu_seqlens_q;
  a.mask = p->key_mask;
  a.mask_stride = p->mask_stride;
  a.mask_cols = p->mask_cols;
  a.out = static_cast<__half*>(p->out);
  a.o_st = p->o_stride_tok;
  a.o_sh = p->o_stride_head;
  a.q_tokens = p->q_tokens;
  a.heads_q = p->heads_q;
  a.heads_k = p->heads_k;
  a.group = p->heads_q / p->heads_k;
  a.batch = p->batch;
  a.max_q = p->max_seqlen_q;
  const int64_t room = static_cast<int64_t>(p->cols) * p->page_size;
  a.max_kv = p->max_kv_len < room ? p->max_kv_len : room;
  a.causal = p->causal;
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  a.ctas = r.ctas;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  a.starts = reinterpret_cast<int32_t*>(ws);
  a.part_o = reinterpret_cast<float*>(ws + r.starts_bytes);
  a.part_ml = reinterpret_cast<float2*>(ws + r.starts_bytes + r.part_o_bytes);
  a.err = error_flag;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (p->head_dim == 128)
    e = r.nt == 2 ? launch<128, 2>(a, st) : launch<128, 1>(a, st);
  else
    e = r.nt == 2 ? launch<64, 2>(a, st) : launch<64, 1>(a, st);
  return e == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}
