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
//     want; a code becomes fp16 by OR-ing it into the mantissa of 1024 (even
//     nibbles: 1024 + n, odd: 1024 + 16 n) and one exact add or FMA, the value by
//     one FMA with the group's scale and minimum. That FMA rounds k and v to fp16
//     once (the tensor core's operand type); p is rounded to fp16 as the prefill's
//     kernels do; scores, maxima, sums and the output accumulate in fp32.
// Rows with no key left give 0. Keys past the length or masked are excluded by
// selecting, and their V by zero scales, so infinities and NaN there do not leak.
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"
#include "kv4_layout.cuh"
#include "tilemix_b200.h"

namespace tilemix {
namespace kv4 {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = 32 * kAttnWarps;
constexpr int kStages = 3;
constexpr int kStepBlocks = 2;                        // 16-key blocks a step
constexpr int kStepKeys = kStepBlocks * kBlockTokens;
constexpr int kChunkKeys = kStepKeys * kAttnWarps;    // keys of one step of every warp
constexpr int kSms = 148;

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
  int heads_q, heads_k, group, row_tiles;  // row_tiles: CTAs along the rows of a (request, KV head)
  int max_q;
  int causal;
  float scale_log2;
  int chunk;   // keys a split
  int splits;  // splits of the longest request
  float* part_o;   // [splits][q_tokens][heads_q][D]
  float2* part_ml; // [splits][q_tokens][heads_q] (max in log2 units, sum)
  int* err;
};

__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

__device__ __forceinline__ uint32_t lop_and_or(uint32_t x, uint32_t m, uint32_t o) {
  uint32_t y;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(y) : "r"(x), "r"(m), "r"(o));  // (x & m) | o
  return y;
}

__device__ __forceinline__ __half2 as_h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ uint32_t as_u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Eight codes of a word as four fp16 pairs of values: pair i holds nibbles i and i + 4, value = s n + m.
__device__ __forceinline__ void unpack8(uint32_t w, __half2 s, __half2 m, uint32_t (&o)[4]) {
  const uint32_t magic = 0x64006400u;
  const __half2 k1024 = as_h2(0x64006400u), r16 = as_h2(0x2C002C00u), k64 = as_h2(0xD400D400u);  // 1024, 1/16, -64
  const uint32_t w8 = w >> 8;
  const __half2 n0 = __hsub2(as_h2(lop_and_or(w, 0x000F000Fu, magic)), k1024);
  const __half2 n1 = __hfma2(as_h2(lop_and_or(w, 0x00F000F0u, magic)), r16, k64);
  const __half2 n2 = __hsub2(as_h2(lop_and_or(w8, 0x000F000Fu, magic)), k1024);
  const __half2 n3 = __hfma2(as_h2(lop_and_or(w8, 0x00F000F0u, magic)), r16, k64);
  o[0] = as_u32(__hfma2(n0, s, m));
  o[1] = as_u32(__hfma2(n1, s, m));
  o[2] = as_u32(__hfma2(n2, s, m));
  o[3] = as_u32(__hfma2(n3, s, m));
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

// One CTA: one (request, KV head, tile of 8 NT rows, split of the keys).
template <int D, int NT>
__global__ void __launch_bounds__(kAttnThreads) attn_kernel(const AttnArgs a) {
  using L = Layout<D>;
  constexpr int G = L::kGroups;
  constexpr int kRows = 8 * NT;
  constexpr int kStageBytes = kStepBlocks * L::kBlockBytes;
  constexpr int kRingBytes = kAttnWarps * kStages * kStageBytes;
  static_assert(kAttnWarps * kRows * D * 4 <= kRingBytes, "the merge reuses the ring");
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint64_t bars[kAttnWarps][kStages];
  __shared__ float sh_m[kAttnWarps][kRows], sh_l[kAttnWarps][kRows];

  const int b = blockIdx.y, split = blockIdx.z;
  const int hk = blockIdx.x / a.row_tiles, row0 = (blockIdx.x % a.row_tiles) * kRows;
  int q0 = b, n_q = 1;
  if (a.cu != nullptr) {
    q0 = a.cu[b];
    n_q = min(a.cu[b + 1] - q0, a.max_q);
  }
  if (q0 < 0 || n_q <= 0 || q0 + static_cast<int64_t>(n_q) > a.q_tokens) return;
  const int n_rows = n_q * a.group;
  if (row0 >= n_rows) return;
  const int64_t cap = static_cast<int64_t>(a.cols) * a.page_blocks * kBlockTokens;
  const int kv = static_cast<int>(min(static_cast<int64_t>(max(a.kv_lens[b], 0)),
                                      min(cap, static_cast<int64_t>(a.chunk) * a.splits)));
  const int parts = max(1, (kv + a.chunk - 1) / a.chunk);
  if (split >= parts) return;
  if (kv < a.kv_lens[b] && threadIdx.x == 0) record_error(a.err, kErrCachePlan);  // longer than the table or max_kv_len
  const int key0 = split * a.chunk, key1 = min(kv, key0 + a.chunk);  // this CTA's keys
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int g = lane >> 2, t = lane & 3;

  uint8_t* ring = smem + warp * kStages * kStageBytes;
  uint64_t* bar = bars[warp];
  if (lane == 0) {
    for (int s = 0; s < kStages; ++s) mbar_init(&bar[s], 1);
    fence_mbarrier_init();
  }
  __syncwarp();

  // The warp's steps: blocks key0 / 16 + 2 (warp + kAttnWarps i).
  const int blk0 = key0 / kBlockTokens, blk1 = (key1 + kBlockTokens - 1) / kBlockTokens;
  const int all_steps = (blk1 - blk0 + kStepBlocks - 1) / kStepBlocks;
  const int steps = all_steps > warp ? (all_steps - warp + kAttnWarps - 1) / kAttnWarps : 0;

  // Page numbers of 32 steps at a time, one step a lane.
  const int32_t* row = a.table + b * a.table_stride;
  const uint8_t* head_base = a.pool + static_cast<int64_t>(hk) * a.page_bytes;
  int32_t pid[kStepBlocks];
  int issued = 0;
  uint32_t stage_bad = 0;  // bit (kStepBlocks stage + block): the block's page is outside the pool
  auto issue = [&]() {
    if ((issued & 31) == 0) {
#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u) {
        const int blk = blk0 + kStepBlocks * (warp + kAttnWarps * (issued + lane)) + u;
        pid[u] = blk < blk1 ? row[blk / a.page_blocks] : 0;
        if (blk < blk1 && (pid[u] < 0 || pid[u] >= a.pages)) {
          record_error(a.err, kErrCachePage);
          pid[u] = -1;
        }
      }
    }
    const int s = issued % kStages;
    const int first = blk0 + kStepBlocks * (warp + kAttnWarps * issued);
    int page[kStepBlocks];
    uint32_t bytes = 0;
#pragma unroll
    for (int u = 0; u < kStepBlocks; ++u) {
      page[u] = __shfl_sync(0xffffffffu, pid[u], issued & 31);
      const uint32_t bit = 1u << (kStepBlocks * s + u);
      const bool have = first + u < blk1;
      if (have && page[u] >= 0) {
        bytes += L::kBlockBytes;
        stage_bad &= ~bit;
      } else {
        page[u] = -1;
        stage_bad |= bit;
      }
    }
    if (lane == 0) {
      mbar_arrive_expect_tx(&bar[s], bytes);
#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u)
        if (page[u] >= 0)
          bulk_load(ring + s * kStageBytes + u * L::kBlockBytes,
                    head_base + page[u] * a.page_stride +
                        static_cast<int64_t>((first + u) % a.page_blocks) * L::kBlockBytes,
                    L::kBlockBytes, &bar[s]);
    }
    ++issued;
  };
  for (int s = 0; s < kStages && issued < steps; ++s) issue();

  // Queries as the B operand: tile x, column g = row row0 + 8 x + g; the K order of a lane's channels.
  // Padding rows are 0 and see what the last row sees.
  uint32_t qf[NT][2 * G][2];
  int lim[NT][2];  // keys [0, lim) visible to the rows of columns 2 t and 2 t + 1
  int lim_lo = 0x7fffffff, lim_hi = 0;
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int r = row0 + 8 * x + g;
    const __half* qr = a.q + static_cast<int64_t>(q0 + r / a.group) * a.q_st +
                       static_cast<int64_t>(hk * a.group + r % a.group) * a.q_sh;
#pragma unroll
    for (int j = 0; j < G; ++j) {
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < n_rows) v = __ldg(reinterpret_cast<const uint4*>(qr + 32 * j + 8 * t));
      // channel i with channel i + 4, as a word's nibbles unpack
      qf[x][2 * j][0] = __byte_perm(v.x, v.z, 0x5410);
      qf[x][2 * j][1] = __byte_perm(v.x, v.z, 0x7632);
      qf[x][2 * j + 1][0] = __byte_perm(v.y, v.w, 0x5410);
      qf[x][2 * j + 1][1] = __byte_perm(v.y, v.w, 0x7632);
    }
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int rc = min(row0 + 8 * x + 2 * t + c, n_rows - 1);
      lim[x][c] = a.causal ? min(kv, kv - n_q + rc / a.group + 1) : kv;
    }
  }
  {
    const int first_row = row0, last_row = min(row0 + kRows, n_rows) - 1;
    lim_lo = a.causal ? min(kv, kv - n_q + first_row / a.group + 1) : kv;
    lim_hi = a.causal ? min(kv, kv - n_q + last_row / a.group + 1) : kv;
  }
  const uint8_t* mask = a.mask != nullptr ? a.mask + b * a.mask_stride : nullptr;

  float o[NT][2 * G][4];
  float m[NT][2], l[NT][2];
#pragma unroll
  for (int x = 0; x < NT; ++x) {
#pragma unroll
    for (int i = 0; i < 2 * G; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) o[x][i][c] = 0.f;
#pragma unroll
    for (int c = 0; c < 2; ++c) m[x][c] = -CUDART_INF_F, l[x][c] = 0.f;
  }

  // Operand rows of the mma <-> tokens of a block: rows 2 i, 2 i + 1 (+ 8) are tokens i, i + 4 (+ 8), so
  // that the four keys of a lane's V operand are t, t + 4, t + 8, t + 12 and a quad reads whole rows.
  const int tok_g = (g >> 1) + (g & 1) * 4;
  bool ok = true;
  for (int i = 0; i < steps; ++i) {
    const int s = i % kStages;
    const int key = key0 + kStepKeys * (warp + kAttnWarps * i);
    const uint32_t bad = (stage_bad >> (kStepBlocks * s)) & ((1u << kStepBlocks) - 1);
    // Which of the step's keys count for any row: bit `token` of block u.
    const bool plain = bad == 0 && mask == nullptr && key + kStepKeys <= lim_lo;
    uint32_t live[kStepBlocks];
    if (!plain) {
#pragma unroll
      for (int u = 0; u < kStepBlocks; ++u) {
        const int kk = key + kBlockTokens * u + lane;
        bool on = lane < kBlockTokens && !((bad >> u) & 1) && kk < lim_hi;
        if (on && mask != nullptr) on = kk < a.mask_cols && mask[kk] != 0;
        live[u] = __ballot_sync(0xffffffffu, on);
      }
    }
    if (!mbar_wait_spin(&bar[s], (i / kStages) & 1, a.err, kErrTimeoutFull)) {
      ok = false;
      break;
    }
    const uint8_t* st = ring + s * kStageBytes;

    float sc[kStepBlocks][NT][4];
#pragma unroll
    for (int u = 0; u < kStepBlocks; ++u) {
      const uint8_t* blk = st + u * L::kBlockBytes;
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 4; ++c) sc[u][x][c] = 0.f;
      const Words<G> ka = load_words<G>(blk + tok_g * L::kRowBytes + t * (4 * G));
      const Words<G> kb = load_words<G>(blk + (tok_g + 8) * L::kRowBytes + t * (4 * G));
      const Words<G> sa = load_words<G>(blk + L::kOffKScale + tok_g * L::kScaleBytes);
      const Words<G> sb = load_words<G>(blk + L::kOffKScale + (tok_g + 8) * L::kScaleBytes);
#pragma unroll
      for (int j = 0; j < G; ++j) {
        uint32_t pa[4], pb[4];
        unpack8(ka.w[j], __low2half2(as_h2(sa.w[j])), __high2half2(as_h2(sa.w[j])), pa);
        unpack8(kb.w[j], __low2half2(as_h2(sb.w[j])), __high2half2(as_h2(sb.w[j])), pb);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          mma16816(sc[u][x], pa[0], pb[0], pa[1], pb[1], qf[x][2 * j][0], qf[x][2 * j][1]);
          mma16816(sc[u][x], pa[2], pb[2], pa[3], pb[3], qf[x][2 * j + 1][0], qf[x][2 * j + 1][1]);
        }
      }
    }

    // Scores in log2 units, the excluded ones -inf.
#pragma unroll
    for (int u = 0; u < kStepBlocks; ++u)
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float v = sc[u][x][c] * a.scale_log2;
          if (!plain) {
            const int tok = tok_g + (c >> 1) * 8;
            if (!((live[u] >> tok) & 1) || key + kBlockTokens * u + tok >= lim[x][c & 1]) v = -CUDART_INF_F;
          }
          sc[u][x][c] = v;
        }
    float base[NT][2];
#pragma unroll
    for (int x = 0; x < NT; ++x)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = fmaxf(sc[0][x][c], sc[0][x][c + 2]);
#pragma unroll
        for (int u = 1; u < kStepBlocks; ++u) top = fmaxf(top, fmaxf(sc[u][x][c], sc[u][x][c + 2]));
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        base[x][c] = fmaxf(m[x][c], top);
      }
    bool moved = false;
#pragma unroll
    for (int x = 0; x < NT; ++x) moved |= base[x][0] > m[x][0] || base[x][1] > m[x][1];
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int x = 0; x < NT; ++x) {
        // m = -inf: nothing summed yet (0 times anything below); base = -inf then stays so
        const float f0 = m[x][0] == base[x][0] ? 1.f : ex2_approx(m[x][0] - base[x][0]);
        const float f1 = m[x][1] == base[x][1] ? 1.f : ex2_approx(m[x][1] - base[x][1]);
        l[x][0] *= f0;
        l[x][1] *= f1;
#pragma unroll
        for (int k = 0; k < 2 * G; ++k) {
          o[x][k][0] *= f0;
          o[x][k][1] *= f1;
          o[x][k][2] *= f0;
          o[x][k][3] *= f1;
        }
        m[x][0] = base[x][0];
        m[x][1] = base[x][1];
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
          const float mx = m[x][c & 1];
          p[c] = ex2_approx(sc[u][x][c] - (mx == -CUDART_INF_F ? 0.f : mx));
          l[x][c & 1] += p[c];
        }
        pf[x][0] = transpose8x8(pack_half2_rn(p[0], p[1]));
        pf[x][1] = transpose8x8(pack_half2_rn(p[2], p[3]));
      }
      constexpr int W = G / 2;  // words of a lane's share of a V row: two groups a word
      Words<W> v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = load_words<W>(blk + (t + 4 * k) * L::kRowBytes + g * (2 * G));
      uint32_t keep0 = 0xffffffffu, keep1 = 0xffffffffu;
      if (!plain) {
        const uint32_t on = live[u] >> t;
        keep0 = ((on & 1u) ? 0xffffu : 0u) | ((on & 0x10u) ? 0xffff0000u : 0u);
        keep1 = ((on & 0x100u) ? 0xffffu : 0u) | ((on & 0x1000u) ? 0xffff0000u : 0u);
      }
#pragma unroll
      for (int j = 0; j < G; ++j) {
        Words<4> vs = load_words<4>(blk + 16 * L::kRowBytes + (j * 4 + t) * 16);
        if (!plain) {
          vs.w[0] &= keep0;
          vs.w[1] &= keep1;
          vs.w[2] &= keep0;
          vs.w[3] &= keep1;
        }
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
    __syncwarp();  // every lane has read the stage
    if (issued < steps) issue();
  }
  if (!ok) {  // a copy did not arrive: wait (bounded) for what is in flight; the other warps still meet below
    for (int s = 0; s < kStages; ++s) {
      const int last = (issued - 1 - s) / kStages;
      if (issued > s) mbar_wait(&bar[s], last & 1, a.err, kErrTimeoutDrain);
    }
  }

  // Merge the warps' states.
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
#pragma unroll
      for (int d = 4; d < 32; d <<= 1) l[x][c] += __shfl_xor_sync(0xffffffffu, l[x][c], d);
      if (g == 0) {
        sh_m[warp][8 * x + 2 * t + c] = m[x][c];
        sh_l[warp][8 * x + 2 * t + c] = l[x][c];
      }
    }
  __syncthreads();  // also: no warp's copies are in flight any more, the rings are free
  float* so = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int x = 0; x < NT; ++x)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      float* dst = so + (warp * kRows + 8 * x + 2 * t + c) * D + 4 * g;
#pragma unroll
      for (int j = 0; j < G; ++j)
        *reinterpret_cast<float4*>(dst + 32 * j) = make_float4(o[x][2 * j][c], o[x][2 * j][c + 2],
                                                               o[x][2 * j + 1][c], o[x][2 * j + 1][c + 2]);
    }
  __syncthreads();
  for (int i = tid; i < kRows * (D / 4); i += kAttnThreads) {
    const int r = i / (D / 4), d = i % (D / 4) * 4;
    if (row0 + r >= n_rows) break;
    float top = sh_m[0][r];
#pragma unroll
    for (int w = 1; w < kAttnWarps; ++w) top = fmaxf(top, sh_m[w][r]);
    const float ref = top == -CUDART_INF_F ? 0.f : top;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kAttnWarps; ++w) {
      const float f = ex2_approx(sh_m[w][r] - ref);
      const float4 v = *reinterpret_cast<const float4*>(so + (w * kRows + r) * D + d);
      sum += f * sh_l[w][r];
      acc.x += f * v.x;
      acc.y += f * v.y;
      acc.z += f * v.z;
      acc.w += f * v.w;
    }
    const int64_t token = q0 + (row0 + r) / a.group;
    const int hq = hk * a.group + (row0 + r) % a.group;
    if (parts == 1) {
      const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);  // NaN stays
      *reinterpret_cast<uint2*>(a.out + token * a.o_st + hq * a.o_sh + d) =
          make_uint2(pack_half2_rn(acc.x * inv, acc.y * inv), pack_half2_rn(acc.z * inv, acc.w * inv));
    } else {
      const int64_t at = (static_cast<int64_t>(split) * a.q_tokens + token) * a.heads_q + hq;
      *reinterpret_cast<float4*>(a.part_o + at * D + d) = acc;
      if (d == 0) a.part_ml[at] = make_float2(top, sum);
    }
  }
}

// Joins the splits of a row: o = sum_s 2^(m_s - m) o_s / sum_s 2^(m_s - m) l_s. One warp a row.
template <int D>
__global__ void __launch_bounds__(kAttnThreads) join_kernel(const AttnArgs a) {
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  int q0 = b, n_q = 1;
  if (a.cu != nullptr) {
    q0 = a.cu[b];
    n_q = min(a.cu[b + 1] - q0, a.max_q);
  }
  if (q0 < 0 || n_q <= 0 || q0 + static_cast<int64_t>(n_q) > a.q_tokens) return;
  const int i = blockIdx.x * kAttnWarps + (threadIdx.x >> 5);
  if (i >= n_q * a.heads_q) return;
  const int64_t cap = static_cast<int64_t>(a.cols) * a.page_blocks * kBlockTokens;
  const int kv = static_cast<int>(min(static_cast<int64_t>(max(a.kv_lens[b], 0)),
                                      min(cap, static_cast<int64_t>(a.chunk) * a.splits)));
  const int parts = max(1, (kv + a.chunk - 1) / a.chunk);
  if (parts == 1) return;  // written by its only CTA
  const int64_t token = q0 + i / a.heads_q;
  const int hq = i % a.heads_q;
  const int64_t row = token * a.heads_q + hq, step = a.q_tokens * a.heads_q;
  float top = -CUDART_INF_F;
  for (int s = lane; s < parts; s += 32) top = fmaxf(top, a.part_ml[row + s * step].x);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  const float ref = top == -CUDART_INF_F ? 0.f : top;
  constexpr int V = D / 32;  // channels a lane
  float acc[V] = {}, sum = 0.f;
  for (int s = 0; s < parts; ++s) {
    const float2 ml = a.part_ml[row + s * step];
    const float f = ex2_approx(ml.x - ref);
    sum += f * ml.y;
    const float* o = a.part_o + (row + s * step) * D + lane * V;
    if constexpr (V == 4) {
      const float4 v = *reinterpret_cast<const float4*>(o);
      acc[0] += f * v.x, acc[1] += f * v.y, acc[2] += f * v.z, acc[3] += f * v.w;
    } else {
      const float2 v = *reinterpret_cast<const float2*>(o);
      acc[0] += f * v.x, acc[1] += f * v.y;
    }
  }
  const float inv = sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum);
  __half* dst = a.out + token * a.o_st + hq * a.o_sh + lane * V;
  if constexpr (V == 4)
    *reinterpret_cast<uint2*>(dst) =
        make_uint2(pack_half2_rn(acc[0] * inv, acc[1] * inv), pack_half2_rn(acc[2] * inv, acc[3] * inv));
  else
    *reinterpret_cast<uint32_t*>(dst) = pack_half2_rn(acc[0] * inv, acc[1] * inv);
}

struct Plan {
  int nt, row_tiles, chunk, splits;
  int64_t part_o_bytes, part_ml_bytes;
};

// Shape of the launch, from host-known sizes alone. Two row tiles a CTA where more than 8 rows share a KV
// head (the unpacking is shared; four would spill). The key axis is cut so that about `kWaves` CTAs fall on
// every slot of the machine, but not into pieces under 256 keys, whose start and join would cost more than
// they save.
static Plan plan_of(const tm_kv4_attn_params* p) {
  Plan r{};
  const int rows = p->max_seqlen_q * (p->heads_q / p->heads_k);
  r.nt = rows > 8 ? 2 : 1;
  r.row_tiles = (rows + 8 * r.nt - 1) / (8 * r.nt);
  const int64_t units = static_cast<int64_t>(p->batch) * p->heads_k * r.row_tiles;
  constexpr int64_t kSlots = kSms * 3, kWaves = 3;
  const int64_t keys = p->max_kv_len > 0 ? p->max_kv_len : 1;
  int64_t chunk = (keys * units + kSlots * kWaves - 1) / (kSlots * kWaves);
  if (chunk < 256) chunk = 256;
  chunk = (chunk + kChunkKeys - 1) / kChunkKeys * kChunkKeys;
  r.splits = static_cast<int>((keys + chunk - 1) / chunk);
  r.chunk = static_cast<int>(chunk);
  if (r.splits > 1) {
    const int64_t n = static_cast<int64_t>(r.splits) * p->q_tokens * p->heads_q;
    r.part_o_bytes = n * p->head_dim * 4;
    r.part_ml_bytes = n * 8;
  }
  return r;
}

static int check(const tm_kv4_attn_params* p) {
  if (p == nullptr) return TM_ERR_NULL;
  if (p->batch < 0 || p->q_tokens < 0 || p->heads_q <= 0 || p->heads_k <= 0 || p->heads_q % p->heads_k != 0)
    return TM_ERR_SHAPE;
  if (p->num_pages < 0 || p->cols < 0 || p->max_seqlen_q < 0 || p->max_kv_len < 0) return TM_ERR_SHAPE;
  if (p->page_size < kBlockTokens || p->page_size % kBlockTokens != 0) return TM_ERR_SHAPE;
  if (p->head_dim != 64 && p->head_dim != 128) return TM_ERR_UNSUPPORTED;
  if (p->batch > 65535 || p->max_seqlen_q > 65535 || p->heads_q > 65535 || p->max_kv_len > (1 << 30))
    return TM_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(p->page_size) * 20 * 128 / kBlockTokens > 0x7fffffffll) return TM_ERR_UNSUPPORTED;
  if (p->batch == 0 || p->q_tokens == 0 || p->max_seqlen_q == 0) return TM_OK;
  if (!p->q || !p->out || !p->kv_lens || (p->num_pages > 0 && !p->pool) || (p->cols > 0 && !p->block_table))
    return TM_ERR_NULL;
  if (p->cu_seqlens_q == nullptr && (p->max_seqlen_q != 1 || p->q_tokens < p->batch)) return TM_ERR_SHAPE;
  if (!aligned(p->q, 16) || !aligned(p->out, 16) || !aligned(p->pool, 16)) return TM_ERR_ALIGN;
  if (p->q_stride_tok % 8 || p->q_stride_head % 8 || p->o_stride_tok % 8 || p->o_stride_head % 8) return TM_ERR_ALIGN;
  if (p->key_mask != nullptr && p->mask_cols < 0) return TM_ERR_SHAPE;
  const Plan r = plan_of(p);
  if (r.splits > 65535) return TM_ERR_UNSUPPORTED;
  return TM_OK;
}

template <int D, int NT>
static cudaError_t launch(const AttnArgs& a, int batch, cudaStream_t st) {
  constexpr int smem = kAttnWarps * kStages * kStepBlocks * Layout<D>::kBlockBytes;
  cudaError_t e = cudaFuncSetAttribute(attn_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid(a.heads_k * a.row_tiles, batch, a.splits);
  attn_kernel<D, NT><<<grid, kAttnThreads, smem, st>>>(a);
  if (a.splits > 1) {
    const dim3 jg((a.max_q * a.heads_q + kAttnWarps - 1) / kAttnWarps, batch);
    join_kernel<D><<<jg, kAttnThreads, 0, st>>>(a);
  }
  return cudaGetLastError();
}

}  // namespace kv4
}  // namespace tilemix

extern "C" int tm_kv4_attn_workspace(const tm_kv4_attn_params* p, int64_t* bytes) {
  using namespace tilemix::kv4;
  if (bytes == nullptr) return TM_ERR_NULL;
  *bytes = 0;
  const int rc = check(p);
  if (rc != TM_OK || p->batch == 0 || p->q_tokens == 0 || p->max_seqlen_q == 0) return rc;
  const Plan r = plan_of(p);
  *bytes = r.part_o_bytes + r.part_ml_bytes;
  return TM_OK;
}

extern "C" int tm_kv4_attn(const tm_kv4_attn_params* p, void* workspace, int64_t workspace_bytes, void* stream) {
  using namespace tilemix::kv4;
  const int rc = check(p);
  if (rc != TM_OK || p->batch == 0 || p->q_tokens == 0 || p->max_seqlen_q == 0) return rc;
  const Plan r = plan_of(p);
  const int64_t need = r.part_o_bytes + r.part_ml_bytes;
  if (need > 0 && workspace == nullptr) return TM_ERR_NULL;
  if (workspace_bytes < need) return TM_ERR_SHAPE;
  if (need > 0 && !aligned(workspace, 16)) return TM_ERR_ALIGN;
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
  a.row_tiles = r.row_tiles;
  a.max_q = p->max_seqlen_q;
  a.causal = p->causal;
  a.scale_log2 = p->sm_scale * 1.4426950408889634f;
  a.chunk = r.chunk;
  a.splits = r.splits;
  a.part_o = static_cast<float*>(workspace);
  a.part_ml = reinterpret_cast<float2*>(static_cast<uint8_t*>(workspace) + r.part_o_bytes);
  a.err = p->error_flag;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e;
  if (p->head_dim == 128)
    e = r.nt == 2 ? launch<128, 2>(a, p->batch, st) : launch<128, 1>(a, p->batch, st);
  else
    e = r.nt == 2 ? launch<64, 2>(a, p->batch, st) : launch<64, 1>(a, p->batch, st);
  return e == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}
