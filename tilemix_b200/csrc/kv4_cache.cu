// Append to and read back from the paged 4-bit key/value cache (kv4_layout.cuh).
//
// Append, for each group of 32 channels of one (token, KV head) row x:
//   m = min x, s = (max x - m) / 15 rounded down to fp16, n = min(rint((x - m) / s), 15)
// and the cache stands for s n + m (never beyond the row's range, hence finite in
// fp16: that is what rounding s down is for). Both fp32 differences and quotients round
// once (IEEE), so the codes do not depend on the schedule. A group whose values
// are equal (or closer than 15 fp16 subnormal steps) has s = 0 and n = 0; a group
// with an infinity or a NaN reads back as NaN. Read back is the reverse, rounded
// to fp16 once.
//
// HBM bounds both on a prefill (2 bytes + 5 bits a value). A thread holds 8
// channels of K and of V (two 16-byte loads in flight), four lanes a group.
#include <cuda_fp16.h>

#include "common.cuh"
#include "kv4_layout.cuh"
#include "tilemix_b200.h"

namespace tilemix {
namespace kv4 {

constexpr int kThreads = 256;

struct AppendArgs {
  const __half* k;
  const __half* v;
  int64_t k_st, k_sh, v_st, v_sh;
  uint8_t* pool;
  int64_t n_tokens;
  int64_t n_slots;  // pages * page size
  const int64_t* slots;
  int heads, page, page_bytes;
  int* err;
};

__device__ __forceinline__ __half2 h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ uint32_t u32(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }

// Codes of a lane's 8 channels in nibble order (channel i at nibble i) and the
// group's (s, m) as a half2. Four consecutive lanes hold the group.
__device__ __forceinline__ uint32_t quantise8(const uint4& x, __half2* sm) {
  const __half2 a = h2(x.x), b = h2(x.y), c = h2(x.z), d = h2(x.w);
  __half2 lo2 = __hmin2_nan(__hmin2_nan(a, b), __hmin2_nan(c, d));
  __half2 hi2 = __hmax2_nan(__hmax2_nan(a, b), __hmax2_nan(c, d));
  // (min, -max) in one register, so the two reductions share their shuffles
  __half2 ext = __halves2half2(__hmin_nan(__low2half(lo2), __high2half(lo2)),
                               __hneg(__hmax_nan(__low2half(hi2), __high2half(hi2))));
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) ext = __hmin2_nan(ext, h2(__shfl_xor_sync(0xffffffffu, u32(ext), o)));
  const float lo = __low2float(ext), hi = -__high2float(ext);
  const __half sh = __float2half_rd(__fdiv_rn(__fsub_rn(hi, lo), 15.f));
  const float s = __half2float(sh);
  *sm = __halves2half2(sh, __low2half(ext));
  if (!(s > 0.f) || !isfinite(s)) return 0u;
  // IEEE quotient from the correctly rounded reciprocal and one residual correction (Markstein):
  // s is an fp16 value and 0 <= x - m <= 2^17, far from under- and overflow.
  const float r = __frcp_rn(s);
  const float f[8] = {__low2float(a), __high2float(a), __low2float(b), __high2float(b),
                      __low2float(c), __high2float(c), __low2float(d), __high2float(d)};
  uint32_t w = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float e = __fsub_rn(f[i], lo);
    const float q0 = __fmul_rn(e, r);
    const float q = __fmaf_rn(__fmaf_rn(-q0, s, e), r, q0);
    // round to nearest even in the low mantissa bits of 1.5 * 2^23
    const uint32_t n = __float_as_uint(__fadd_rn(fminf(q, 15.f), 12582912.f)) & 15u;
    w |= n << (4 * i);
  }
  return w;
}

template <int D>
__global__ void __launch_bounds__(kThreads) append_kernel(const AppendArgs a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8;  // lanes a row
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  const int l = threadIdx.x % kLanes;
  const int j = l >> 2, t = l & 3;
  // Items behind the last one stay for the shuffles.
  const bool there = item < a.n_tokens * a.heads;
  const int64_t tok = there ? item / a.heads : 0;
  const int head = there ? static_cast<int>(item - tok * a.heads) : 0;
  const int64_t slot = there ? a.slots[tok] : -1;
  const bool fits = slot >= 0 && slot < a.n_slots;
  uint4 xk = make_uint4(0, 0, 0, 0), xv = xk;
  if (fits) {
    xk = __ldcs(reinterpret_cast<const uint4*>(a.k + tok * a.k_st + head * a.k_sh + 8 * l));
    xv = __ldcs(reinterpret_cast<const uint4*>(a.v + tok * a.v_st + head * a.v_sh + 8 * l));
  }
  __half2 ks, vs;
  const uint32_t kw = quantise8(xk, &ks), vw = quantise8(xv, &vs);
  // A V chunk holds 4 channels of each group: lanes of groups j and j ^ 1 trade halves, so that each
  // stores one 32-bit word. The even group's lane keeps chunk 2t, the odd one's chunk 2t + 1.
  const uint32_t other = __shfl_xor_sync(0xffffffffu, vw, 4);
  const uint32_t vpair = (j & 1) ? __byte_perm(other, vw, 0x7632) : __byte_perm(vw, other, 0x5410);
  if (!fits) {
    if (there && (slot >= a.n_slots || slot < -1) && l == 0) record_error(a.err, kErrCacheSlot);
    return;
  }
  const int64_t page = slot / a.page;
  const int in_page = static_cast<int>(slot - page * a.page), in_block = in_page % kBlockTokens;
  uint8_t* blk = a.pool + (page * a.heads + head) * a.page_bytes +
                 static_cast<int64_t>(in_page / kBlockTokens) * L::kBlockBytes;
  *reinterpret_cast<uint32_t*>(blk + in_block * L::kRowBytes + (t * L::kGroups + j) * 4) = kw;
  const int g = 2 * t + (j & 1);
  *reinterpret_cast<uint32_t*>(blk + L::kOffV + in_block * L::kRowBytes + g * (2 * L::kGroups) + (j & ~1) * 2) = vpair;
  if (t == 0) {
    *reinterpret_cast<__half2*>(blk + L::kOffKScale + in_block * L::kScaleBytes + j * 4) = ks;
    __half* p = reinterpret_cast<__half*>(blk + L::kOffVScale + L::v_scale(j, in_block));
    p[0] = __low2half(vs);
    p[4] = __high2half(vs);
  }
}

struct ReadArgs {
  const uint8_t* pool;
  const int64_t* slots;
  int64_t n_tokens, n_slots;
  int heads, page, page_bytes;
  __half* k;
  __half* v;
  int* err;
};

__device__ __forceinline__ uint4 dequant8(uint32_t w, float s, float m) {
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = pack_half2_rn(__fmaf_rn(static_cast<float>((w >> (8 * i)) & 15u), s, m),
                         __fmaf_rn(static_cast<float>((w >> (8 * i + 4)) & 15u), s, m));
  return make_uint4(o[0], o[1], o[2], o[3]);
}

template <int D>
__global__ void __launch_bounds__(kThreads) read_kernel(const ReadArgs a) {
  using L = Layout<D>;
  constexpr int kLanes = D / 8;
  const int64_t item = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) / kLanes;
  if (item >= a.n_tokens * a.heads) return;
  const int l = threadIdx.x % kLanes;
  const int j = l >> 2, t = l & 3;
  const int64_t tok = item / a.heads;
  const int head = static_cast<int>(item - tok * a.heads);
  const int64_t slot = a.slots[tok];
  uint4 ok = make_uint4(0, 0, 0, 0), ov = ok;
  if (slot >= 0 && slot < a.n_slots) {
    const int64_t page = slot / a.page;
    const int in_page = static_cast<int>(slot - page * a.page), in_block = in_page % kBlockTokens;
    const uint8_t* blk = a.pool + (page * a.heads + head) * a.page_bytes +
                         static_cast<int64_t>(in_page / kBlockTokens) * L::kBlockBytes;
    const uint32_t kw = *reinterpret_cast<const uint32_t*>(blk + in_block * L::kRowBytes + (t * L::kGroups + j) * 4);
    const uint8_t* vr = blk + L::kOffV + in_block * L::kRowBytes + 2 * j;
    const uint32_t v0 = *reinterpret_cast<const uint16_t*>(vr + (2 * t) * (2 * L::kGroups));
    const uint32_t v1 = *reinterpret_cast<const uint16_t*>(vr + (2 * t + 1) * (2 * L::kGroups));
    const __half2 ks = *reinterpret_cast<const __half2*>(blk + L::kOffKScale + in_block * L::kScaleBytes + j * 4);
    const __half* vs = reinterpret_cast<const __half*>(blk + L::kOffVScale + L::v_scale(j, in_block));
    ok = dequant8(kw, __low2float(ks), __high2float(ks));
    ov = dequant8(v0 | v1 << 16, __half2float(vs[0]), __half2float(vs[4]));
  } else if (slot != -1 && l == 0) {
    record_error(a.err, kErrCacheSlot);
  }
  const int64_t at = item * D + 8 * l;
  __stcs(reinterpret_cast<uint4*>(a.k + at), ok);
  __stcs(reinterpret_cast<uint4*>(a.v + at), ov);
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
  if (k_stride_tok % 8 || k_stride_head % 8 || v_stride_tok % 8 || v_stride_head % 8) return TM_ERR_ALIGN;
  const int64_t page_bytes = static_cast<int64_t>(page_size) / kBlockTokens * block_bytes(head_dim);
  const int64_t blocks = (n_tokens * heads * (head_dim / 8) + kThreads - 1) / kThreads;
  if (page_bytes > 0x7fffffffll || blocks > 0x7fffffffll) return TM_ERR_UNSUPPORTED;
  AppendArgs a{static_cast<const __half*>(k), static_cast<const __half*>(v), k_stride_tok, k_stride_head,
               v_stride_tok, v_stride_head, static_cast<uint8_t*>(pool), n_tokens, num_pages * page_size, slots,
               heads, page_size, static_cast<int>(page_bytes), error_flag};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    append_kernel<128><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(a);
  else
    append_kernel<64><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(a);
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
  const int64_t page_bytes = static_cast<int64_t>(page_size) / kBlockTokens * block_bytes(head_dim);
  const int64_t blocks = (n_tokens * heads * (head_dim / 8) + kThreads - 1) / kThreads;
  if (page_bytes > 0x7fffffffll || blocks > 0x7fffffffll) return TM_ERR_UNSUPPORTED;
  ReadArgs a{static_cast<const uint8_t*>(pool), slots, n_tokens, num_pages * page_size, heads, page_size,
             static_cast<int>(page_bytes), static_cast<__half*>(k), static_cast<__half*>(v), error_flag};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    read_kernel<128><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(a);
  else
    read_kernel<64><<<static_cast<unsigned>(blocks), kThreads, 0, st>>>(a);
  return cudaGetLastError() == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}
