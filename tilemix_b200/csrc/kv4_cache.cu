// Append to and read back from the paged 4-bit key/value cache (kv4_layout.cuh).
//
// Append, for each group of 32 channels of one (token, KV head) row x:
//   m = min x, s = (max x - m) / 15 rounded down to fp16, n = min(rint((x - m) / s), 15)
// and the cache stands for s n + m (never beyond the row's range, hence finite in
// fp16: that is what rounding s down is for), differences and quotients in fp32. A group whose values
// are equal (or closer than 15 fp16 subnormal steps) has s = 0 and n = 0; a group
// with an infinity or a NaN reads back as NaN. Read back is the reverse, rounded
// to fp16 once.
//
// HBM should bound both on a prefill (2 bytes + 5 bits a value); append is bound
// by the instructions it issues (in 75 % of its active cycles, the ALU and FMA
// pipes 57 and 48 % busy), so a thread has 16 channels of K and of V, two
// lanes a group: what a token and head cost (slot, addresses, scales) and the
// shuffles are shared by twice the values. 32768 tokens of 8 heads of 128: 38 us
// (51 with 8 channels a thread) where 27 would carry the bytes. Read back: 34 us
// for the same, 8 channels a thread; 16 took a third fewer instructions and the
// same time, so it waits for memory, not for its instructions.
#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"
#include "kv4_layout.cuh"
#include "tilemix_b200.h"

namespace tilemix {
namespace kv4 {

// A CTA takes 16 consecutive tokens of one head, D / 16 (append) or D / 8 lanes a token: consecutive tokens mostly
// share a block, whose V scales (2 bytes a token in 8 places) then leave, or come, as whole sectors.
template <int D>
constexpr int kAppendThreads = kBlockTokens * D / 16;
template <int D>
constexpr int kReadThreads = kBlockTokens * D / 8;

struct Pages {
  uint32_t heads;
  int bytes;        // of one head of a page
  uint32_t blocks;  // 16-token blocks a page
  int shift;        // log2 of them, or -1
};

struct AppendArgs {
  const __half* k;
  const __half* v;
  int k_st, k_sh, v_st, v_sh;
  uint8_t* pool;
  int n_tokens;
  int64_t n_slots;  // pages * page size
  const int64_t* slots;
  Pages pages;
  int* err;
};

// Where a slot's 16-token block of a head is. Blocks, tokens and strides are counted in 32 bits (the entry points
// see to it) and page sizes that are powers of two divide by a shift: 64-bit products and a division by the page
// size were a third of the kernels' instructions.
__device__ __forceinline__ int64_t block_offset(int64_t slot, int head, const Pages& p, int block_bytes) {
  const uint32_t blk = static_cast<uint32_t>(slot >> 4);
  const uint32_t page = p.shift >= 0 ? blk >> p.shift : blk / p.blocks;
  return static_cast<int64_t>(page * p.heads + head) * p.bytes +
         static_cast<int64_t>(blk - page * p.blocks) * block_bytes;
}

__device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ uint32_t u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

__device__ __forceinline__ uint64_t pair(float lo, float hi) {
  return static_cast<uint64_t>(__float_as_uint(hi)) << 32 | __float_as_uint(lo);
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}

// a / b from an approximate reciprocal of b and one residual correction (Markstein): q0 is within a few units in
// the last place, the residual a - q0 b is exact in an FMA, and its product with r errs by 2^-22 of a unit, so
// the quotient is that of an IEEE division unless it lies that near half way between two fp32 numbers; a
// quotient half way between two codes is representable and comes out exact.
__device__ __forceinline__ float quotient(float a, float b, float r) {
  const float q0 = __fmul_rn(a, r);
  return __fmaf_rn(__fmaf_rn(-q0, b, a), r, q0);
}

// Codes of a lane's 16 channels in nibble order (channel i at nibble i) and the
// group's (s, m) as a half2. Two neighbouring lanes hold the group.
__device__ __forceinline__ uint2 quantise16(const uint4& x0, const uint4& x1, __half2* sm) {
  const uint32_t in[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
  __half2 lo2 = h2(in[0]), hi2 = lo2;
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo2 = __hmin2_nan(lo2, h2(in[i]));
    hi2 = __hmax2_nan(hi2, h2(in[i]));
  }
  // (min, -max) in one register, so the two reductions share their shuffle
  __half2 ext = __halves2half2(__hmin_nan(__low2half(lo2), __high2half(lo2)),
                               __hneg(__hmax_nan(__low2half(hi2), __high2half(hi2))));
  ext = __hmin2_nan(ext, h2(__shfl_xor_sync(0xffffffffu, u32(ext), 1)));
  const float lo = __low2float(ext), hi = -__high2float(ext);
  const __half sh = __float2half_rd(quotient(__fsub_rn(hi, lo), 15.f, 1.f / 15.f));
  const float s = __half2float(sh);
  *sm = __halves2half2(sh, __low2half(ext));
  const bool ok = s > 0.f && s < CUDART_INF_F;
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(s));
  const uint64_t r2 = pair(r, r), ns2 = pair(-s, -s), nlo2 = pair(-lo, -lo);
  const uint64_t magic2 = 0x4B4000004B400000ull;  // 1.5 * 2^23: rounds to nearest even in the low bits
  uint64_t e[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float2 f = __half22float2(h2(in[i]));
    e[i] = add2(pair(f.x, f.y), nlo2);
  }
  // s is rounded down by less than 2^-10, so the largest quotient stays under 15.5, except where s is
  // subnormal: there x - m is cut at 15 s.
  if (__any_sync(0xffffffffu, s < 6.103515625e-5f)) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      e[i] = pair(fminf(__uint_as_float(static_cast<uint32_t>(e[i])), 15.f * s),
                  fminf(__uint_as_float(static_cast<uint32_t>(e[i] >> 32)), 15.f * s));
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint64_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint64_t q0 = mul2(e[4 * h + i], r2);
      u[i] = add2(fma2(fma2(q0, ns2, e[4 * h + i]), r2, q0), magic2);
    }
    // sum of (0x4B400000 + n_i) 16^i modulo 2^32, less the constants'
    w[h] = static_cast<uint32_t>(u[3] >> 32);
#pragma unroll
    for (int i = 6; i >= 0; --i) w[h] = (w[h] << 4) + static_cast<uint32_t>(u[i / 2] >> (32 * (i % 2)));
    w[h] = ok ? w[h] - (0x4B400000u + 0xB4000000u + 0x40000000u) : 0u;
  }
  return make_uint2(w[0], w[1]);
}

template <int D>
__global__ void __launch_bounds__(kAppendThreads<D>) append_kernel(const AppendArgs a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 16;  // lanes a row
  __shared__ uint8_t* sh_block[kBlockTokens];  // each token's block, NULL: it is not stored
  __shared__ int sh_at[kBlockTokens];          // its place there
  __shared__ __half sh_scale[kBlockTokens][L::kGroups][2];
  const int head = blockIdx.x, in_cta = threadIdx.x / kLanes;
  const int tok = (blockIdx.z * gridDim.y + blockIdx.y) * kBlockTokens + in_cta;
  const int l = threadIdx.x % kLanes;
  const int j = l >> 1, p = l & 1;  // channels 32 j + 16 p ..
  const bool there = tok < a.n_tokens;  // tokens behind the last one stay for the shuffles
  const int64_t slot = there ? a.slots[tok] : -1;
  const bool fits = slot >= 0 && slot < a.n_slots;
  uint4 xk[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)}, xv[2] = {xk[0], xk[0]};
  if (fits) {
    const uint4* k = reinterpret_cast<const uint4*>(a.k + static_cast<int64_t>(tok) * a.k_st +
                                                    (static_cast<int64_t>(head) * a.k_sh + 16 * l));
    const uint4* v = reinterpret_cast<const uint4*>(a.v + static_cast<int64_t>(tok) * a.v_st +
                                                    (static_cast<int64_t>(head) * a.v_sh + 16 * l));
    xk[0] = __ldcs(k);
    xk[1] = __ldcs(k + 1);
    xv[0] = __ldcs(v);
    xv[1] = __ldcs(v + 1);
  }
  __half2 ks, vs;
  const uint2 kw = quantise16(xk[0], xk[1], &ks), vw = quantise16(xv[0], xv[1], &vs);
  // A V chunk holds 4 channels of each group, and a lane has four chunks' worth of its own: lanes of groups j and
  // j ^ 1 trade halves, so that each stores two chunks' 32-bit words. The even group's lane keeps chunks 4 p and
  // 4 p + 1, the odd one's the two after them.
  const bool odd = j & 1;
  const uint32_t other = __shfl_xor_sync(0xffffffffu, odd ? vw.x : vw.y, 2);
  const uint32_t mine = odd ? vw.y : vw.x;
  const uint32_t va = odd ? other : mine, vb = odd ? mine : other;  // of the even and the odd group
  const int in_block = static_cast<int>(slot) & (kBlockTokens - 1);
  uint8_t* blk = fits ? a.pool + block_offset(slot, head, a.pages, L::kBlockBytes) : nullptr;
  if (p == 0) {
    sh_scale[in_cta][j][0] = __low2half(vs);
    sh_scale[in_cta][j][1] = __high2half(vs);
    if (j == 0) {
      sh_block[in_cta] = blk;
      sh_at[in_cta] = in_block;
      if (there && (slot >= a.n_slots || slot < -1)) record_error(a.err, kErrCacheSlot);
    }
  }
  if (fits) {
    uint32_t* kc = reinterpret_cast<uint32_t*>(blk + in_block * L::kRowBytes + (2 * p * L::kGroups + j) * 4);
    kc[0] = kw.x;
    kc[L::kGroups] = kw.y;
    uint8_t* vc = blk + L::kOffV + in_block * L::kRowBytes + (4 * p + 2 * odd) * (2 * L::kGroups) + (j & ~1) * 2;
    *reinterpret_cast<uint32_t*>(vc) = __byte_perm(va, vb, 0x5410);
    *reinterpret_cast<uint32_t*>(vc + 2 * L::kGroups) = __byte_perm(va, vb, 0x7632);
    if (p == 0) *reinterpret_cast<__half2*>(blk + L::kOffKScale + in_block * L::kScaleBytes + j * 4) = ks;
  }
  __syncthreads();
  // The V scales, a thread each, in the order in which a block holds them if its tokens follow on from the
  // first one's slot (any other order is as right, only slower).
  const int i = threadIdx.x;
  static_assert(kAppendThreads<D> == kBlockTokens * L::kGroups * 2, "one V scale or minimum a thread");
  const int quarter = i & 3, which = (i >> 2) & 1, tt = (i >> 3) & 3, jj = i >> 5;
  const int first = sh_block[0] == nullptr ? 0 : sh_at[0];
  const int token = (4 * quarter + tt - first) & (kBlockTokens - 1);
  uint8_t* to = sh_block[token];
  if (to != nullptr)
    *reinterpret_cast<__half*>(to + L::kOffVScale + L::v_scale(jj, sh_at[token]) + 8 * which) =
        sh_scale[token][jj][which];
}

struct ReadArgs {
  const uint8_t* pool;
  const int64_t* slots;
  int n_tokens;
  int64_t n_slots;
  Pages pages;
  __half* k;
  __half* v;
  int* err;
};

// Eight values in channel order: codes OR-ed into the mantissa of 1024 as pairs (i, i + 4), brought to n
// exactly, one fp16 FMA (one rounding), then put side by side.
__device__ __forceinline__ uint4 dequant8(uint32_t w, __half s, __half m) {
  const __half2 s2 = __half2half2(s), m2 = __half2half2(m);
  const __half2 k1024 = h2(0x64006400u), r16 = h2(0x2C002C00u), k64 = h2(0xD400D400u);  // 1024, 1/16, -64
  const uint32_t w8 = w >> 8;
  const uint32_t a = u32(__hfma2(__hsub2(h2((w & 0x000F000Fu) | 0x64006400u), k1024), s2, m2));
  const uint32_t b = u32(__hfma2(__hfma2(h2((w & 0x00F000F0u) | 0x64006400u), r16, k64), s2, m2));
  const uint32_t c = u32(__hfma2(__hsub2(h2((w8 & 0x000F000Fu) | 0x64006400u), k1024), s2, m2));
  const uint32_t d = u32(__hfma2(__hfma2(h2((w8 & 0x00F000F0u) | 0x64006400u), r16, k64), s2, m2));
  return make_uint4(__byte_perm(a, b, 0x5410), __byte_perm(c, d, 0x5410), __byte_perm(a, b, 0x7632),
                    __byte_perm(c, d, 0x7632));
}

template <int D>
__global__ void __launch_bounds__(kReadThreads<D>) read_kernel(const ReadArgs a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8;
  const int head = blockIdx.x;
  const int tok = (blockIdx.z * gridDim.y + blockIdx.y) * kBlockTokens + threadIdx.x / kLanes;
  const int l = threadIdx.x % kLanes;
  const int j = l >> 2, t = l & 3;
  const bool there = tok < a.n_tokens;  // tokens behind the last one stay for the shuffle
  const int64_t slot = there ? a.slots[tok] : -1;
  const bool fits = slot >= 0 && slot < a.n_slots;
  uint32_t kw = 0, vpair = 0;
  __half2 ks = __half2half2(__ushort_as_half(0));
  __half vs = __ushort_as_half(0), vm = vs;
  if (fits) {
    const int in_block = static_cast<int>(slot) & (kBlockTokens - 1);
    const uint8_t* blk = a.pool + block_offset(slot, head, a.pages, L::kBlockBytes);
    kw = *reinterpret_cast<const uint32_t*>(blk + in_block * L::kRowBytes + (t * L::kGroups + j) * 4);
    vpair = *reinterpret_cast<const uint32_t*>(blk + L::kOffV + in_block * L::kRowBytes +
                                               (2 * t + (j & 1)) * (2 * L::kGroups) + (j & ~1) * 2);
    ks = *reinterpret_cast<const __half2*>(blk + L::kOffKScale + in_block * L::kScaleBytes + j * 4);
    const __half* v = reinterpret_cast<const __half*>(blk + L::kOffVScale + L::v_scale(j, in_block));
    vs = v[0];
    vm = v[4];
  }
  // the lane holds chunk 2 t (+ 1) of groups j and j ^ 1 and trades one half
  const uint32_t other = __shfl_xor_sync(0xffffffffu, vpair, 4);
  const uint32_t vw = (j & 1) ? __byte_perm(other, vpair, 0x7632) : __byte_perm(vpair, other, 0x5410);
  if (!there) return;
  uint4 ok = make_uint4(0, 0, 0, 0), ov = ok;
  if (fits) {
    ok = dequant8(kw, __low2half(ks), __high2half(ks));
    ov = dequant8(vw, vs, vm);
  } else if (slot != -1 && l == 0) {
    record_error(a.err, kErrCacheSlot);
  }
  const int64_t at = static_cast<int64_t>(tok * a.pages.heads + head) * D + 8 * l;
  __stcs(reinterpret_cast<uint4*>(a.k + at), ok);
  __stcs(reinterpret_cast<uint4*>(a.v + at), ov);
}

// Heads fastest: the heads of 16 tokens are neighbours in memory.
static dim3 grid_of(int64_t groups, int heads) {
  const unsigned y = static_cast<unsigned>(groups < 65535 ? groups : 65535);
  return dim3(static_cast<unsigned>(heads), y, static_cast<unsigned>((groups + y - 1) / y));
}

// TM_OK and the pool's shape for the kernels, or why not. The grid's last dimension is rounded up to whole layers of
// 65,535 CTAs, so a CTA's first token may be up to 2^20 behind the last one and has to stay below 2^31.
static int pages_of(int64_t n_tokens, int64_t num_pages, int heads, int head_dim, int page_size, Pages* p) {
  const int64_t blocks = page_size / kBlockTokens, bytes = blocks * block_bytes(head_dim);
  if (bytes > 0x7fffffffll || num_pages * blocks > 0x7fffffffll || num_pages * heads > 0x7fffffffll ||
      (n_tokens + kBlockTokens) * heads > 0x7fffffffll || n_tokens > 0x7fffffffll - (1 << 20))
    return TM_ERR_UNSUPPORTED;
  p->heads = static_cast<uint32_t>(heads);
  p->bytes = static_cast<int>(bytes);
  p->blocks = static_cast<uint32_t>(blocks);
  p->shift = -1;
  for (int k = 0; k < 31; ++k)
    if (blocks == (1ll << k)) p->shift = k;
  return TM_OK;
}

}  // namespace kv4
}  // namespace tilemix

extern "C" int tm_kv4_append(const void* k, int64_t k_stride_tok, int64_t k_stride_head, const void* v,
                             int64_t v_stride_tok, int64_t v_stride_head, int64_t n_tokens, const int64_t* slots,
                             void* pool, int64_t num_pages, int heads, int head_dim, int page_size, int* error_flag,
                             void* stream) {
  using namespace tilemix::kv4;
  if (n_tokens < 0 || num_pages < 0 || heads <= 0 || page_size < 16 || page_size % 16 != 0) return TM_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return TM_ERR_UNSUPPORTED;
  if (n_tokens == 0) return TM_OK;
  if (!k || !v || !slots || (num_pages > 0 && !pool)) return TM_ERR_NULL;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(pool, 16) || !aligned(slots, 8)) return TM_ERR_ALIGN;
  AppendArgs a{};
  // of one token or head the stride to the next is never used
  const bool toks = n_tokens > 1, hs = heads > 1;
  const int64_t strides[4] = {toks ? k_stride_tok : 0, hs ? k_stride_head : 0, toks ? v_stride_tok : 0,
                              hs ? v_stride_head : 0};
  int* const to[4] = {&a.k_st, &a.k_sh, &a.v_st, &a.v_sh};
  for (int i = 0; i < 4; ++i) {
    if (strides[i] % 8 != 0) return TM_ERR_ALIGN;
    if (strides[i] > 0x7fffffffll || strides[i] < -0x7fffffffll) return TM_ERR_UNSUPPORTED;
    *to[i] = static_cast<int>(strides[i]);
  }
  if (pages_of(n_tokens, num_pages, heads, head_dim, page_size, &a.pages) != TM_OK) return TM_ERR_UNSUPPORTED;
  a.k = static_cast<const __half*>(k);
  a.v = static_cast<const __half*>(v);
  a.pool = static_cast<uint8_t*>(pool);
  a.n_tokens = static_cast<int>(n_tokens);
  a.n_slots = num_pages * page_size;
  a.slots = slots;
  a.err = error_flag;
  const int64_t groups = (n_tokens + kBlockTokens - 1) / kBlockTokens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    append_kernel<128><<<grid_of(groups, heads), kAppendThreads<128>, 0, st>>>(a);
  else
    append_kernel<64><<<grid_of(groups, heads), kAppendThreads<64>, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}

extern "C" int tm_kv4_read(const void* pool, int64_t num_pages, int heads, int head_dim, int page_size,
                           const int64_t* slots, int64_t n_tokens, void* k, void* v, int* error_flag, void* stream) {
  using namespace tilemix::kv4;
  if (n_tokens < 0 || num_pages < 0 || heads <= 0 || page_size < 16 || page_size % 16 != 0) return TM_ERR_SHAPE;
  if (head_dim != 64 && head_dim != 128) return TM_ERR_UNSUPPORTED;
  if (n_tokens == 0) return TM_OK;
  if (!k || !v || !slots || (num_pages > 0 && !pool)) return TM_ERR_NULL;
  if (!aligned(k, 16) || !aligned(v, 16) || !aligned(pool, 16) || !aligned(slots, 8)) return TM_ERR_ALIGN;
  ReadArgs a{};
  if (pages_of(n_tokens, num_pages, heads, head_dim, page_size, &a.pages) != TM_OK) return TM_ERR_UNSUPPORTED;
  a.pool = static_cast<const uint8_t*>(pool);
  a.slots = slots;
  a.n_tokens = static_cast<int>(n_tokens);
  a.n_slots = num_pages * page_size;
  a.k = static_cast<__half*>(k);
  a.v = static_cast<__half*>(v);
  a.err = error_flag;
  const int64_t groups = (n_tokens + kBlockTokens - 1) / kBlockTokens;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    read_kernel<128><<<grid_of(groups, heads), kReadThreads<128>, 0, st>>>(a);
  else
    read_kernel<64><<<grid_of(groups, heads), kReadThreads<64>, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}
