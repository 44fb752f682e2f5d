// Linear layer in 8-bit integers: per-token quantiser and the integer matrix
// product with a scale for each token and each output channel.
//
//   s_t = max_k |x_tk| / 127,  x8_tk = round_half_away(127 x_tk / max_k |x_tk|)
//   y_tn = (sum_k x8_tk w8_nk) s_t w_n + b_n
//
// The sum is exact (int32: up to 133,000 terms of 127 * 127), so its order, the
// split of K and the tile do not change the result; scales and bias are applied
// in fp32 and y is rounded once.
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math_constants.h>

#include <type_traits>

#include "common.cuh"
#include "kv4_layout.cuh"
#include "tilemix_b200.h"

namespace tilemix {

PFN_cuTensorMapEncodeTiled_v12000 encode_fn();  // attn_api.cu

namespace linear {

using kv4::aligned;

// ----------------------------------------------------------------------------
// Quantiser
// ----------------------------------------------------------------------------
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w);
template <>
__device__ __forceinline__ float2 unpack2<__half>(uint32_t w) {
  return __half22float2(*reinterpret_cast<__half2*>(&w));
}
template <>
__device__ __forceinline__ float2 unpack2<__nv_bfloat16>(uint32_t w) {
  return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w));
}
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// max that keeps a NaN
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct RowScale {
  float k;     // codes are round(k x / amax), k = 127 times a power of two
  QuantDiv d;  // division by amax (times that power of two)
  bool ok;
};

// k x is exact in fp32 (x has at most 11 significant bits), and the quotient is the IEEE one (common.cuh), so a
// quotient half way between two codes is exact and the others are too far from one (2^-19 relative) for their
// rounding to matter: the code is that of exact arithmetic.
__device__ __forceinline__ RowScale row_scale(float amax) {
  // bf16 rows reach from 1e-40 to 3e38: a power of two on both sides of the quotient keeps the product, the
  // reciprocal and the residual normal.
  const float p = amax < 5.421010862e-20f ? 1.844674407e19f : amax > 1.844674407e19f ? 5.421010862e-20f : 1.f;  // 2^+-64
  RowScale s;
  s.k = 127.f * p;
  s.ok = amax > 0.f && amax <= 3.4028235e38f;
  s.d.init(s.ok ? amax * p : 1.f);
  return s;
}

template <typename T>
__device__ __forceinline__ uint2 codes8(const uint4& v, const RowScale& s) {
  const uint32_t in[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[8];  // codes in the low bytes
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<T>(in[i]);
    quant_code_pair<kNumericsExact>(f.x * s.k, f.y * s.k, s.d, &c[2 * i], &c[2 * i + 1]);
  }
  return make_uint2(__byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410));
}

template <int kThreads>
__device__ __forceinline__ float block_max(float m) {
  __shared__ float red[kThreads / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  m = red[threadIdx.x % (kThreads / 32)];
#pragma unroll
  for (int o = kThreads / 64; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}

// One CTA a row, the row held in registers between the two uses (kVec 16-byte pieces a thread; 0: any length,
// read twice). 8192 rows of 4096: 22.8 us, 4.4 TB/s; the codes' arithmetic bounds it (an issue in 75 % of the active
// cycles, the FMA and ALU pipes 52 and 49 % busy, 14 % of the time start and tail). A row with an infinity or a NaN gets that scale and codes 0, so that its outputs are NaN.
template <typename T, int kVec, int kThreads>
__global__ void __launch_bounds__(kThreads) quant_rows_kernel(const T* x, int64_t x_stride, int cols, int8_t* out,
                                                             int64_t out_stride, float* scale) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product that follows may load its weights
  const T* row = x + blockIdx.x * x_stride;
  int8_t* dst = out + blockIdx.x * out_stride;
  float m = 0.f;
  if constexpr (kVec > 0) {
    uint4 v[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int c = (i * kThreads + threadIdx.x) * 8;
      v[i] = c < cols ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0, 0, 0, 0);
      const uint32_t w[4] = {v[i].x, v[i].y, v[i].z, v[i].w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<T>(w[e]);
        m = max_nan(m, max_nan(fabsf(f.x), fabsf(f.y)));
      }
    }
    m = block_max<kThreads>(m);
    const RowScale s = row_scale(m);
#pragma unroll
    for (int i = 0; i < kVec; ++i) {
      const int c = (i * kThreads + threadIdx.x) * 8;
      if (c < cols) *reinterpret_cast<uint2*>(dst + c) = s.ok ? codes8<T>(v[i], s) : make_uint2(0, 0);
    }
  } else {
    for (int c = threadIdx.x; c < cols; c += kThreads) m = max_nan(m, fabsf(to_float(row[c])));
    m = block_max<kThreads>(m);
    const RowScale s = row_scale(m);
    for (int c = threadIdx.x; c < cols; c += kThreads) {
      uint32_t code, unused;
      quant_code_pair<kNumericsExact>(to_float(row[c]) * s.k, 0.f, s.d, &code, &unused);
      dst[c] = s.ok ? static_cast<int8_t>(code & 0xffu) : int8_t(0);
    }
  }
  if (threadIdx.x == 0) scale[blockIdx.x] = __fdiv_rn(m, 127.f);
}

// Rows that do not start on 16 bytes, value by value: kWarps warps a row, up to 32 values a thread in registers. One
// warp (eight rows a CTA) where a row fits it: 3944 rows of 323 take 3.4 us, 19 with 1024 threads a row that read it
// twice; 4096 rows of 5003 with eight 19, 41 so. Longer rows are read twice (4096 of 18947: 101 us, 131 with 1024
// threads that hold them).
template <typename T, int kWarps>
__global__ void __launch_bounds__(256) quant_odd_kernel(const T* x, int64_t x_stride, unsigned rows, int cols,
                                                        int8_t* out, int64_t out_stride, float* scale) {
  static_assert(kWarps == 1 || kWarps == 8, "eight warps a CTA");
  constexpr int kPer = 32;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");  // a product that follows may load its weights
  constexpr int kRow = 32 * kWarps;
  const unsigned r = kWarps == 1 ? blockIdx.x * 8 + threadIdx.x / 32 : blockIdx.x;
  const int t = threadIdx.x % kRow;
  if (r >= rows) return;  // a whole warp, and only where no one waits for it
  const T* row = x + r * x_stride + t;
  int8_t* dst = out + r * out_stride + t;
  const int n = cols > t ? (cols - t + kRow - 1) / kRow : 0;  // values of this thread
  T v[kPer];
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < n) v[i] = row[i * kRow];
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (i < n) m = max_nan(m, fabsf(to_float(v[i])));
  if constexpr (kWarps == 1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
  } else {
    m = block_max<kRow>(m);
  }
  const RowScale s = row_scale(m);
#pragma unroll
  for (int i = 0; i < kPer; i += 2) {
    if (i >= n) break;
    const bool two = i + 1 < n;
    uint32_t c[2];
    quant_code_pair<kNumericsExact>(to_float(v[i]) * s.k, two ? to_float(v[i + 1]) * s.k : 0.f, s.d, &c[0], &c[1]);
    dst[i * kRow] = s.ok ? static_cast<int8_t>(c[0] & 0xffu) : int8_t(0);
    if (two) dst[(i + 1) * kRow] = s.ok ? static_cast<int8_t>(c[1] & 0xffu) : int8_t(0);
  }
  if (t == 0) scale[r] = __fdiv_rn(m, 127.f);
}

template <typename T, int kVec, int kThreads>
static void run_quant(const T* x, int64_t xs, unsigned rows, int cols, int8_t* out, int64_t os, float* scale,
                      cudaStream_t st) {
  quant_rows_kernel<T, kVec, kThreads><<<rows, kThreads, 0, st>>>(x, xs, cols, out, os, scale);
}

// 1024 threads a row where rows are fewer than SMs (64 rows of 18944: 11 us with 256 threads that read it twice,
// 5 us so), 256 where they are many: a CTA's reduction then hides behind the others' loads (4096 rows of 18944: 120 us
// with 1024 threads, 58 so).
template <typename T>
static void launch_quant(const void* x, int64_t xs, int64_t rows, int cols, int8_t* out, int64_t os, float* scale,
                         cudaStream_t st) {
  const T* p = static_cast<const T*>(x);
  const unsigned g = static_cast<unsigned>(rows);
  const bool vec = cols % 8 == 0 && aligned(x, 16) && xs % 8 == 0 && aligned(out, 8) && os % 8 == 0;
  if (cols > 32768 || (!vec && (cols > 8192 || rows < 148)))
    run_quant<T, 0, 1024>(p, xs, g, cols, out, os, scale, st);
  else if (!vec && cols <= 1024)
    quant_odd_kernel<T, 1><<<(g + 7) / 8, 256, 0, st>>>(p, xs, g, cols, out, os, scale);
  else if (!vec)
    quant_odd_kernel<T, 8><<<g, 256, 0, st>>>(p, xs, g, cols, out, os, scale);
  else if (cols <= 2048)
    run_quant<T, 1, 256>(p, xs, g, cols, out, os, scale, st);
  else if (rows < 148) {
    if (cols <= 8192)
      run_quant<T, 1, 1024>(p, xs, g, cols, out, os, scale, st);
    else if (cols <= 16384)
      run_quant<T, 2, 1024>(p, xs, g, cols, out, os, scale, st);
    else
      run_quant<T, 4, 1024>(p, xs, g, cols, out, os, scale, st);
  } else if (cols <= 4096)
    run_quant<T, 2, 256>(p, xs, g, cols, out, os, scale, st);
  else if (cols <= 8192)
    run_quant<T, 4, 256>(p, xs, g, cols, out, os, scale, st);
  else if (cols <= 16384)
    run_quant<T, 8, 256>(p, xs, g, cols, out, os, scale, st);
  else if (cols <= 24576)
    run_quant<T, 12, 256>(p, xs, g, cols, out, os, scale, st);
  else
    run_quant<T, 8, 512>(p, xs, g, cols, out, os, scale, st);
}

// ----------------------------------------------------------------------------
// Matrix product
// ----------------------------------------------------------------------------
// D[128 x BN] = A[128 x K] B[BN x K]^T on tcgen05 kind::i8, both operands K-major in 128-byte swizzled tiles
// that TMA brings (it fills rows and columns past the ends with zeros), int32 accumulators in TMEM, two of
// them, so that one tile's epilogue runs under the next tile's products. With many tokens they are the A side
// (a lane of TMEM is a token); with few, the weights are, and the tokens are the N side, as narrow as they
// are (a lane is a channel): the tensor core then never works on padding rows and the weights stream through.
// A split of K is a cluster of CTAs, one part each, whose int32 partial tiles are added through distributed
// shared memory: exact, so without an effect on the result, and without a workspace. 64 tokens of 18944 -> 3584: 19 us,
// the weights at 3.5 TB/s from HBM (13.6 us from L2: about 5 us are the start, the first loads and the split's sum).
constexpr int kBM = 128, kBK = 128;
constexpr int kGemmThreads = 256;
constexpr int kMaxSplit = 8;
constexpr int kMaxSplitBN = 128;  // widest tile whose K is cut
constexpr int kSms = 148;

struct GemmArgs {
  int rows_a, rows_b;
  int k_tiles, split;
  int bn;  // columns a tile (the pair kernel's; the others know theirs)
  int tiles_a, tiles_b;
  const float* scale_a;  // of the lanes' rows
  const float* scale_b;  // of the columns' rows
  const void* bias;      // optional, of the channels, in the output's type
  void* out;             // [tokens, channels], row stride ldo
  int64_t ldo;
  int vec;  // rows of `out` take 16-byte stores
  // Launched beside the quantiser that makes x8 and its scales (programmatic dependent launch): what the kernels
  // before that one wrote, the weights among it, is there already. Without it everything before is waited for.
  int beside;
  int* err;
};

__device__ __forceinline__ void tma_load_2d_e(void* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ int32_t ld_cluster(uint32_t saddr, uint32_t rank) {
  int32_t v;
  asm volatile(
      "{\n\t.reg .b32 a;\n\t"
      "mapa.shared::cluster.u32 a, %1, %2;\n\t"
      "ld.shared::cluster.b32 %0, [a];\n\t}"
      : "=r"(v)
      : "r"(saddr), "r"(rank)
      : "memory");
  return v;
}

__device__ __forceinline__ void store_one(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void store_one(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store_one(float* p, float v) { *p = v; }
__device__ __forceinline__ float load_one(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float load_one(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load_one(const float* p) { return *p; }
__device__ __forceinline__ uint32_t pack2(const __half*, float a, float b) { return pack_half2_rn(a, b); }
__device__ __forceinline__ uint32_t pack2(const __nv_bfloat16*, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <int BN>
struct GemmShape {
  static constexpr int kStageBytes = (kBM + BN) * kBK;
  static constexpr int kStages = BN >= 256 ? 4 : BN >= 128 ? 5 : BN >= 64 ? 7 : 8;  // what fits, one CTA an SM
  // behind the ring: scales and biases of the columns of two tiles, and with the tokens on the lanes a
  // 4 KB piece of output for each epilogue warp
  static constexpr int kOffCols = kStages * kStageBytes;
  static constexpr int kOffPieces = kOffCols + 2 * 2 * BN * 4;
  static constexpr int smem(bool token_lanes) { return kOffPieces + (token_lanes ? 4 * 4096 : 0) + 1024; }
  static constexpr int kTmemCols = 2 * BN < 32 ? 32 : 2 * BN;
  static constexpr bool kSplits = BN <= kMaxSplitBN;
};

// y = sum * token scale * channel scale + bias, the token's scale first on either side, so that every launch
// shape gives the same bits.
__device__ __forceinline__ float scaled(uint32_t acc, float token, float channel, float bias) {
  return fmaf(static_cast<float>(static_cast<int32_t>(acc)) * token, channel, bias);
}

// kCols consecutive columns of this lane's row, stored one by one; col_scale / col_bias: of those columns.
template <int kCols, bool kTokenLanes, typename OutT>
__device__ __forceinline__ void emit(const uint32_t* acc, const GemmArgs& g, int a, int b0, float row_scale,
                                     float row_bias, const float* col_scale, const float* col_bias) {
  if (a >= g.rows_a) return;
  OutT* out = static_cast<OutT*>(g.out);
#pragma unroll
  for (int c = 0; c < kCols; ++c) {
    const int b = b0 + c;
    if (b >= g.rows_b) break;
    if (kTokenLanes)
      store_one(out + a * g.ldo + b, scaled(acc[c], row_scale, col_scale[c], col_bias[c]));
    else
      store_one(out + b * g.ldo + a, scaled(acc[c], col_scale[c], row_scale, row_bias));
  }
}

// With the tokens on the lanes: kRowBytes of each of a warp's 32 rows through shared memory, so that they are
// stored as whole sectors side by side (a lane's own row would be 32 separate pieces a store). 16-byte pieces are
// swizzled by the row against bank conflicts.
// `load(c, sums)` brings the lane's sums of columns c .. of the piece.
template <typename OutT, int kRowBytes, typename Load>
__device__ __forceinline__ void emit_rows(Load load, uint8_t* piece, const GemmArgs& g, int a0, int b0,
                                          float row_scale, const float* col_scale, const float* col_bias) {
  constexpr int kCols = kRowBytes / sizeof(OutT), kPer = 16 / sizeof(OutT), kChunks = kRowBytes / 16;
  constexpr int kLoad = kCols < 32 ? kCols : 32;  // columns a load
  const int lane = threadIdx.x & 31;
  auto at = [](int row, int chunk) { return row * kRowBytes + ((chunk ^ (row * kRowBytes / 128 & (kChunks - 1))) << 4); };
#pragma unroll
  for (int h = 0; h < kCols / kLoad; ++h) {
    uint32_t r[kLoad];
    load(kLoad * h, r);
#pragma unroll
    for (int c = 0; c < kLoad; c += kPer) {
      float v[kPer];
#pragma unroll
      for (int i = 0; i < kPer; i += 4) {
        const float4 cs = *reinterpret_cast<const float4*>(col_scale + kLoad * h + c + i);
        const float4 cb = *reinterpret_cast<const float4*>(col_bias + kLoad * h + c + i);
        v[i] = scaled(r[c + i], row_scale, cs.x, cb.x);
        v[i + 1] = scaled(r[c + i + 1], row_scale, cs.y, cb.y);
        v[i + 2] = scaled(r[c + i + 2], row_scale, cs.z, cb.z);
        v[i + 3] = scaled(r[c + i + 3], row_scale, cs.w, cb.w);
      }
      uint4 w;
      if constexpr (sizeof(OutT) == 2)
        w = make_uint4(pack2(static_cast<const OutT*>(nullptr), v[0], v[1]),
                       pack2(static_cast<const OutT*>(nullptr), v[2], v[3]),
                       pack2(static_cast<const OutT*>(nullptr), v[4], v[5]),
                       pack2(static_cast<const OutT*>(nullptr), v[6], v[7]));
      else
        w = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
      *reinterpret_cast<uint4*>(piece + at(lane, (kLoad * h + c) / kPer)) = w;
    }
  }
  __syncwarp();
  OutT* out = static_cast<OutT*>(g.out);
  if (g.vec) {
    const int chunk = lane % kChunks, b = b0 + chunk * kPer;
#pragma unroll
    for (int i = 0; i < kChunks; ++i) {
      const int row = 32 / kChunks * i + lane / kChunks;
      if (a0 + row < g.rows_a && b < g.rows_b) {
        const uint4 w = *reinterpret_cast<const uint4*>(piece + at(row, chunk));
        OutT* dst = out + static_cast<int64_t>(a0 + row) * g.ldo + b;
        if (b + kPer <= g.rows_b) {
          *reinterpret_cast<uint4*>(dst) = w;
        } else {
          const OutT* e = reinterpret_cast<const OutT*>(&w);
#pragma unroll
          for (int k = 0; k < kPer; ++k)
            if (b + k < g.rows_b) dst[k] = e[k];
        }
      }
    }
  } else {
    // Rows that do not start on 16 bytes: a value a lane, side by side (3944 x 323 -> 4663 took 102 us with eight a
    // lane, 51 so).
    constexpr int kWide = kCols < 32 ? kCols : 32, kStep = 32 / kWide;
    const int col = lane % kWide, rows = min(32, g.rows_a - a0);
#pragma unroll 4
    for (int row = lane / kWide; row < rows; row += kStep) {
      OutT* dst = out + static_cast<int64_t>(a0 + row) * g.ldo + b0;
#pragma unroll
      for (int c = col; c < kCols; c += kWide)
        if (b0 + c < g.rows_b) dst[c] = *reinterpret_cast<const OutT*>(piece + at(row, c / kPer) + c % kPer * sizeof(OutT));
    }
  }
  __syncwarp();
}

// emit_rows' sums from TMEM.
struct FromTmem {
  uint32_t taddr;
  __device__ __forceinline__ void operator()(int c, uint32_t (&r)[32]) const {
    tmem_ld32(taddr + c, r);
    tmem_wait_ld();
  }
  __device__ __forceinline__ void operator()(int c, uint32_t (&r)[16]) const {
    tmem_ld16(taddr + c, r);
    tmem_wait_ld();
  }
};

// The sum over the cluster of kSplit partial tiles of this rank's columns, with the loads of several columns and
// all parts in flight together.
template <int kSplit, int BN, bool kTokenLanes, typename OutT>
__device__ __forceinline__ void reduce_split(uint32_t red, uint8_t* piece, const GemmArgs& g, int a0, int b0, int rank,
                                             float row_scale, float row_bias, const float* col_scale,
                                             const float* col_bias) {
  constexpr int kCols = BN / kSplit;
  auto sums = [&](int c, auto& sum) {
    constexpr int n = sizeof(sum) / 4, kFlight = n < 32 / kSplit ? n : 32 / kSplit;
#pragma unroll
    for (int i0 = 0; i0 < n; i0 += kFlight) {
      int32_t part[kSplit][kFlight];
#pragma unroll
      for (int p = 0; p < kSplit; ++p)
#pragma unroll
        for (int i = 0; i < kFlight; ++i) part[p][i] = ld_cluster(red + (c + i0 + i) * (kBM * 4), p);
#pragma unroll
      for (int i = 0; i < kFlight; ++i) {
        int32_t v = part[0][i];
#pragma unroll
        for (int p = 1; p < kSplit; ++p) v += part[p][i];
        sum[i0 + i] = static_cast<uint32_t>(v);
      }
    }
  };
  if constexpr (kTokenLanes) {
    constexpr int kRowBytes = kCols * static_cast<int>(sizeof(OutT)) < 128 ? kCols * static_cast<int>(sizeof(OutT)) : 128;
    constexpr int kStep = kRowBytes / static_cast<int>(sizeof(OutT));
    for (int c = rank * kCols; c < (rank + 1) * kCols; c += kStep)
      emit_rows<OutT, kRowBytes>([&](int at, auto& sum) { sums(c + at, sum); }, piece, g, a0, b0 + c, row_scale,
                                 col_scale + c, col_bias + c);
  } else {
    constexpr int kStep = kCols < 8 ? kCols : 8;
    for (int c = rank * kCols; c < (rank + 1) * kCols; c += kStep) {
      uint32_t sum[kStep];
      sums(c, sum);
      emit<kStep, kTokenLanes, OutT>(sum, g, a0 + (threadIdx.x & 31), b0 + c, row_scale, row_bias, col_scale + c,
                                     col_bias + c);
    }
  }
}

template <int BN, bool kTokenLanes, typename OutT>
__global__ void __launch_bounds__(kGemmThreads) gemm_kernel(const __grid_constant__ CUtensorMap map_a,
                                                           const __grid_constant__ CUtensorMap map_b,
                                                           const GemmArgs g) {
  using S = GemmShape<BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[S::kStages], empty[S::kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = g.split > 1 ? blockIdx.x % g.split : 0;
  const int first_tile = g.split > 1 ? blockIdx.x / g.split : blockIdx.x;
  const int tile_step = g.split > 1 ? g.tiles_a * g.tiles_b : gridDim.x;
  const int tiles = g.tiles_a * g.tiles_b;
  const int k0 = static_cast<int>(static_cast<int64_t>(g.k_tiles) * rank / g.split);
  const int k1 = static_cast<int>(static_cast<int64_t>(g.k_tiles) * (rank + 1) / g.split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 4);
    }
    fence_mbarrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 2) {
    tmem_alloc(&tmem_base, S::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  // Tiles in groups of 16 A tiles, A fastest: a group's A tiles and the B tiles in work stay in L2.
  auto tile_at = [&](int t, int* ta, int* tb) {
    const int group = t / (16 * g.tiles_b), first = group * 16;
    const int wide = min(16, g.tiles_a - first), r = t - group * 16 * g.tiles_b;
    *ta = first + r % wide;
    *tb = r / wide;
  };

  bool ok = true;
  float row_scale = 0.f, row_bias = 0.f;
  if (warp == 0) {
    // The weights do not depend on the kernel before (the quantiser, when this one was launched beside it): those
    // of the first stages are under way before its end is waited for.
    int s = 0, used = 0, early = 0;
    uint32_t phase = 0;
    if (first_tile < tiles) {
      int ta, tb;
      tile_at(first_tile, &ta, &tb);
      early = min(S::kStages, k1 - k0);
      for (int i = 0; i < early; ++i) {
        uint8_t* st = smem + i * S::kStageBytes;
        mbar_arrive_expect_tx_e(&full[i], S::kStageBytes);
        if (kTokenLanes)
          tma_load_2d_e(st + kBM * kBK, &map_b, &full[i], (k0 + i) * kBK, tb * BN);
        else
          tma_load_2d_e(st, &map_a, &full[i], (k0 + i) * kBK, ta * kBM);
      }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int t = first_tile; t < tiles && ok; t += tile_step) {
      int ta, tb;
      tile_at(t, &ta, &tb);
      for (int k = k0; k < k1; ++k) {
        uint8_t* st = smem + s * S::kStageBytes;
        const bool half = used < early;  // its weights are under way
        if (!half) {
          if (!mbar_wait_spin(&empty[s], phase ^ 1, g.err, kErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          mbar_arrive_expect_tx_e(&full[s], S::kStageBytes);
        }
        if (!half || kTokenLanes) tma_load_2d_e(st, &map_a, &full[s], k * kBK, ta * kBM);
        if (!half || !kTokenLanes) tma_load_2d_e(st + kBM * kBK, &map_b, &full[s], k * kBK, tb * BN);
        ++used;
        if (++s == S::kStages) s = 0, phase ^= 1;
      }
    }
    if (!ok) {  // the copies in flight land before the shared memory is given up
      for (int i = 0; i < S::kStages && used > i; ++i) {
        const int last = (used - 1 - i) / S::kStages;
        mbar_wait(&full[i], last & 1, g.err, kErrTimeoutDrain);
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = make_idesc(2, 1, 0, 0, kBM, BN);
    int s = 0, n = 0;
    uint32_t phase = 0;
    for (int t = first_tile; t < tiles && ok; t += tile_step, ++n) {
      const int acc = n & 1;
      if (!mbar_wait_spin(&acc_empty[acc], ((n >> 1) & 1) ^ 1, g.err, kErrTimeoutOFree)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + acc * BN;
      for (int k = k0; k < k1; ++k) {
        if (!mbar_wait_spin(&full[s], phase, g.err, kErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t st = smem_u32(smem + s * S::kStageBytes);
        const uint64_t da = make_sdesc(st, 16, 1024, 2), db = make_sdesc(st + kBM * kBK, 16, 1024, 2);
#pragma unroll
        for (int i = 0; i < kBK / 32; ++i)
          mma_i8_ss_e(d, da + 2 * i, db + 2 * i, idesc, (k > k0 || i > 0) ? 1u : 0u);
        tc_commit_e(&empty[s]);
        if (++s == S::kStages) s = 0, phase ^= 1;
      }
      if (ok) tc_commit_e(&acc_full[acc]);
    }
    if (!ok) {  // products in flight end before TMEM is given up: a barrier of this warp's own
      __shared__ __align__(8) uint64_t drain;
      if (lane == 0) {
        mbar_init(&drain, 1);
        fence_mbarrier_init();
      }
      __syncwarp();
      tc_commit_e(&drain);
      mbar_wait(&drain, 0, g.err, kErrTimeoutDrain);
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, et = threadIdx.x - 128;
    float* cols = reinterpret_cast<float*>(smem + S::kOffCols);  // [2][scales BN, biases BN]
    uint8_t* piece = smem + S::kOffPieces + quad * 4096;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // the tokens' scales
    int n = 0;
    for (int t = first_tile; t < tiles; t += tile_step, ++n) {
      const int acc = n & 1;
      int ta, tb;
      tile_at(t, &ta, &tb);
      const int a = ta * kBM + quad * 32 + lane;
      // Scales and biases under the products: the columns' in shared memory (of two tiles in turn: the barrier
      // below keeps the four warps within one tile of another), the lane's row's in registers.
      float* col_scale = cols + acc * 2 * BN;
      float* col_bias = col_scale + BN;
      for (int c = et; c < BN; c += 128) {
        const int b = tb * BN + c;
        const bool in = b < g.rows_b;
        col_scale[c] = in ? g.scale_b[b] : 0.f;
        col_bias[c] = kTokenLanes && in && g.bias != nullptr ? load_one(static_cast<const OutT*>(g.bias) + b) : 0.f;
      }
      row_scale = a < g.rows_a ? g.scale_a[a] : 0.f;
      row_bias =
          !kTokenLanes && a < g.rows_a && g.bias != nullptr ? load_one(static_cast<const OutT*>(g.bias) + a) : 0.f;
      asm volatile("bar.sync 1, 128;" ::: "memory");
      // After a wait that ran out a warp only keeps the barrier's count.
      if (ok && !mbar_wait_spin(&acc_full[acc], (n >> 1) & 1, g.err, kErrTimeoutScores)) ok = false;
      if (!ok) continue;
      tc_fence_after();
      const uint32_t d = tmem + acc * BN + (static_cast<uint32_t>(quad * 32) << 16);
      if (!S::kSplits || g.split == 1) {
        if constexpr (kTokenLanes) {
          constexpr int kCols = 128 / sizeof(OutT);
#pragma unroll 1
          for (int c = 0; c < BN; c += kCols)
            emit_rows<OutT, 128>(FromTmem{d + c}, piece, g, ta * kBM + quad * 32, tb * BN + c, row_scale, col_scale + c, col_bias + c);
        } else {
#pragma unroll 1
          for (int c = 0; c < BN; c += 16) {
            uint32_t r[16];
            tmem_ld16(d + c, r);
            tmem_wait_ld();
            emit<16, kTokenLanes, OutT>(r, g, a, tb * BN + c, row_scale, row_bias, col_scale + c, col_bias + c);
          }
        }
      } else if constexpr (S::kSplits) {
        // this part's partial tile, column by column (a warp's 32 lanes are 128 consecutive bytes); every
        // copy has landed and every product has read its stage, so the ring is free
        int32_t* red = reinterpret_cast<int32_t*>(smem) + quad * 32 + lane;
#pragma unroll 1
        for (int c = 0; c < BN; c += 16) {
          uint32_t r[16];
          tmem_ld16(d + c, r);
          tmem_wait_ld();
#pragma unroll
          for (int i = 0; i < 16; ++i) red[(c + i) * kBM] = static_cast<int32_t>(r[i]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    }
  }

  if constexpr (S::kSplits) {
    if (g.split > 1) {  // a cluster has one tile; the barriers are reached whatever happened above
      __syncwarp();
      cluster_sync();
      if (warp >= 4 && ok) {
        int ta, tb;
        tile_at(first_tile, &ta, &tb);
        const int row = (warp & 3) * 32 + lane;
        const uint32_t red = smem_u32(smem) + row * 4;
        const float* col_scale = reinterpret_cast<const float*>(smem + S::kOffCols);
        auto reduce = [&](auto parts) {
          reduce_split<decltype(parts)::value, BN, kTokenLanes, OutT>(
              red, smem + S::kOffPieces + (warp & 3) * 4096, g, ta * kBM + (warp & 3) * 32, tb * BN, rank, row_scale,
              row_bias, col_scale, col_scale + BN);
        };
        if (g.split == 2)
          reduce(std::integral_constant<int, 2>{});
        else if (g.split == 4)
          reduce(std::integral_constant<int, 4>{});
        else
          reduce(std::integral_constant<int, 8>{});
      }
      __syncwarp();
      cluster_sync();  // nobody leaves while its partial tile is read
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 2) tmem_dealloc(tmem, S::kTmemCols);
}

// ----------------------------------------------------------------------------
// Two CTAs a tile
// ----------------------------------------------------------------------------
// 256 tokens x up to 256 channels on a pair of SMs (cta_group::2): each CTA brings its 128 tokens and half of the
// channels' rows, the first one issues the products for both, each keeps its 128 rows of the sum in its own
// TMEM. A CTA then reads 32 KB for each 128 bytes of K where it read 48 KB for the same number of products: the
// one-CTA kernel is bound by what L2 delivers. The width is a multiple of 32 from 128 on, chosen so that the last
// wave of tiles is full. 8192 x 4096 -> 14336: 282 us, 3410 TOP/s, the tensor pipe busy for 92 % of it; 310 us with one
// CTA a tile.
struct PairShape {
  static constexpr int kBN = 256;  // widest
  // The ring holds as many stages as there is room for, six of the widest: a stage is on its way for about 3300
  // cycles (both CTAs' copies, the products, the word back to both), so narrow ones have to be more.
  static constexpr int kRing = 6 * (kBM + kBN / 2) * kBK;
  static constexpr int kMaxStages = 8;
  static __host__ __device__ int stage_bytes(int bn) { return (kBM + bn / 2) * kBK; }
  static __host__ __device__ int stages(int bn) {
    return kRing / stage_bytes(bn) < kMaxStages ? kRing / stage_bytes(bn) : kMaxStages;
  }
  // Eight epilogue warps, two for each quarter of the rows, half of the columns each: with one tile a CTA nothing
  // hides behind the epilogue.
  static constexpr int kEpilogueWarps = 8;
  static constexpr int kRowBytes = 64;  // of output a row and warp at a time: what room six stages leave
  static constexpr int kThreads = 128 + 32 * kEpilogueWarps;
  static constexpr int kOffCols = kRing;
  static constexpr int kOffPieces = kOffCols + 2 * 2 * kBN * 4;
  static constexpr int kSmem = kOffPieces + kEpilogueWarps * 32 * kRowBytes + 1024;
};

// The barrier of the pair's first CTA at the offset of `bar` (bit 24 of a shared::cluster address tells the two apart).
__device__ __forceinline__ uint32_t first_cta(const uint64_t* bar) { return smem_u32(bar) & 0xFEFFFFFFu; }

__device__ __forceinline__ void tma_load_pair_e(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];\n\t}" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}

__device__ __forceinline__ void mma_i8_pair_e(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "@e tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive at `bar` in both CTAs once the products issued so far are done.
__device__ __forceinline__ void commit_pair_e(const uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\t"
      "elect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t}" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}

template <typename OutT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PairShape::kThreads, 1)
    gemm_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                     const GemmArgs g) {
  using S = PairShape;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ __align__(8) uint64_t full[S::kMaxStages], empty[S::kMaxStages], acc_full[2], acc_empty[2], drain;
  __shared__ uint32_t tmem_base;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x & 1, first_tile = blockIdx.x >> 1, tile_step = gridDim.x >> 1;
  const int tiles = g.tiles_a * g.tiles_b, bn = g.bn;
  const int stage_bytes = S::stage_bytes(bn), stages = S::stages(bn);
  const uint32_t bytes = 2u * stage_bytes;  // of a stage in both CTAs

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kMaxStages; ++s) {
      mbar_init(&full[s], 1);   // the first CTA's: its own arrival and the bytes of both
      mbar_init(&empty[s], 1);  // each CTA's: the products that read the stage are done
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&acc_full[i], 1);
      mbar_init(&acc_empty[i], 2 * S::kEpilogueWarps);  // the first CTA's: the epilogue warps of both
    }
    mbar_init(&drain, 1);
    fence_mbarrier_init();
    prefetch_tmap(&map_a);
    prefetch_tmap(&map_b);
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base)), "r"(512)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();  // barriers and TMEM of both are there
  tc_fence_after();
  const uint32_t tmem = tmem_base;

  auto tile_at = [&](int t, int* ta, int* tb) {  // groups of 8 A tiles (2048 tokens), A fastest
    const int group = t / (8 * g.tiles_b), first = group * 8;
    const int wide = min(8, g.tiles_a - first), r = t - group * 8 * g.tiles_b;
    *ta = first + r % wide;
    *tb = r / wide;
  };

  bool ok = true;
  if (warp == 0) {
    int s = 0, used = 0, early = 0;
    uint32_t phase = 0;
    // as in the one-CTA kernel: the first stages' weights before the quantiser's end
    if (first_tile < tiles) {
      int ta, tb;
      tile_at(first_tile, &ta, &tb);
      early = min(stages, g.k_tiles);
      for (int i = 0; i < early; ++i) {
        if (rank == 0) mbar_arrive_expect_tx_e(&full[i], bytes);
        tma_load_pair_e(smem + i * stage_bytes + kBM * kBK, &map_b, first_cta(&full[i]), i * kBK,
                        tb * bn + rank * (bn / 2));
      }
    }
    asm volatile("griddepcontrol.wait;" ::: "memory");
    for (int t = first_tile; t < tiles && ok; t += tile_step) {
      int ta, tb;
      tile_at(t, &ta, &tb);
      for (int k = 0; k < g.k_tiles; ++k) {
        uint8_t* st = smem + s * stage_bytes;
        const bool half = used < early;
        if (!half) {
          if (!mbar_wait_spin(&empty[s], phase ^ 1, g.err, kErrTimeoutEmpty)) {
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx_e(&full[s], bytes);
          tma_load_pair_e(st + kBM * kBK, &map_b, first_cta(&full[s]), k * kBK, tb * bn + rank * (bn / 2));
        }
        tma_load_pair_e(st, &map_a, first_cta(&full[s]), k * kBK, (2 * ta + rank) * kBM);
        ++used;
        if (++s == stages) s = 0, phase ^= 1;
      }
    }
    if (!ok && rank == 0) {
      for (int i = 0; i < stages && used > i; ++i)
        mbar_wait(&full[i], ((used - 1 - i) / stages) & 1, g.err, kErrTimeoutDrain);
    }
  } else if (warp == 1 && rank == 0) {
    const uint32_t idesc = make_idesc(2, 1, 0, 0, 2 * kBM, bn);
    int s = 0, n = 0;
    uint32_t phase = 0;
    for (int t = first_tile; t < tiles && ok; t += tile_step, ++n) {
      const int acc = n & 1;
      if (!mbar_wait_spin(&acc_empty[acc], ((n >> 1) & 1) ^ 1, g.err, kErrTimeoutOFree)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const uint32_t d = tmem + acc * S::kBN;
      for (int k = 0; k < g.k_tiles; ++k) {
        if (!mbar_wait_spin(&full[s], phase, g.err, kErrTimeoutFull)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t st = smem_u32(smem + s * stage_bytes);
        const uint64_t da = make_sdesc(st, 16, 1024, 2), db = make_sdesc(st + kBM * kBK, 16, 1024, 2);
#pragma unroll
        for (int i = 0; i < kBK / 32; ++i)
          mma_i8_pair_e(d, da + 2 * i, db + 2 * i, idesc, (k > 0 || i > 0) ? 1u : 0u);
        commit_pair_e(&empty[s]);
        if (++s == stages) s = 0, phase ^= 1;
      }
      if (ok) commit_pair_e(&acc_full[acc]);
    }
    if (!ok) {  // products in flight end before TMEM is given up
      commit_pair_e(&drain);
      mbar_wait(&drain, 0, g.err, kErrTimeoutDrain);
    }
  } else if (warp >= 4) {
    const int quad = warp & 3, side = (warp - 4) >> 2, et = threadIdx.x - 128;
    float* cols = reinterpret_cast<float*>(smem + S::kOffCols);
    uint8_t* piece = smem + S::kOffPieces + (warp - 4) * 32 * S::kRowBytes;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    int n = 0;
    for (int t = first_tile; t < tiles; t += tile_step, ++n) {
      const int acc = n & 1;
      int ta, tb;
      tile_at(t, &ta, &tb);
      const int a0 = (2 * ta + rank) * kBM + quad * 32;
      float* col_scale = cols + acc * 2 * S::kBN;
      float* col_bias = col_scale + S::kBN;
      for (int c = et; c < bn; c += 32 * S::kEpilogueWarps) {
        const int b = tb * bn + c;
        const bool in = b < g.rows_b;
        col_scale[c] = in ? g.scale_b[b] : 0.f;
        col_bias[c] = in && g.bias != nullptr ? load_one(static_cast<const OutT*>(g.bias) + b) : 0.f;
      }
      const float row_scale = a0 + lane < g.rows_a ? g.scale_a[a0 + lane] : 0.f;
      asm volatile("bar.sync 1, 256;" ::: "memory");
      // After a wait that ran out a warp only keeps the barrier's count.
      if (ok && !mbar_wait_spin(&acc_full[acc], (n >> 1) & 1, g.err, kErrTimeoutScores)) ok = false;
      if (!ok) continue;
      tc_fence_after();
      const uint32_t d = tmem + acc * S::kBN + (static_cast<uint32_t>(quad * 32) << 16);
      constexpr int kCols = S::kRowBytes / sizeof(OutT);
#pragma unroll 1
      for (int c = side * kCols; c < bn; c += 2 * kCols)
        emit_rows<OutT, S::kRowBytes>(FromTmem{d + c}, piece, g, a0, tb * bn + c, row_scale, col_scale + c, col_bias + c);
      tc_fence_before();
      __syncwarp();
      if (lane == 0)
        asm volatile(
            "{\n\t.reg .b32 a;\n\t"
            "mapa.shared::cluster.u32 a, %0, 0;\n\t"
            "mbarrier.arrive.release.cluster.shared::cluster.b64 _, [a];\n\t}" ::"r"(smem_u32(&acc_empty[acc]))
            : "memory");
    }
  }
  tc_fence_before();
  __syncwarp();
  cluster_sync();  // neither CTA leaves, or gives up its TMEM, while the other's products may reach it
  if (warp == 2)
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

struct Plan {
  bool token_lanes, pair;
  int bn, split;
};

// Which kernel, how wide a tile and into how many parts K is cut, by sizes alone: the least of an estimate in SM
// cycles. A step of 128 bytes of K costs the most of three: two cycles a column in the tensor core; what L2 has to
// deliver, 64 bytes a cycle and SM when all of them ask (18 TB/s); the time a stage is on its way (2050 cycles, 3300
// in a pair) over the stages of the ring. A wave of CTAs costs its steps; the epilogue 8 cycles a column of whole
// lines, 60 of single values (tokens on the columns), and a split's two meetings 2500 and 20 a column of its share.
// Against rules by the number of tiles alone: linear of 256 x 18944 -> 3584 37 us, 29 so; 1536 tokens 135, 102 so;
// 128 x 512 -> 1000 12.8, 6.1 so.
static Plan plan_of(int64_t m, int n, int k_tiles) {
  auto ceil_div = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  auto most = [](double a, double b, double c) { return a > b ? (a > c ? a : c) : (b > c ? b : c); };
  Plan best{};
  double least = 1e300;
  auto offer = [&](bool token_lanes, bool pair, int bn, int split, double cost) {
    if (cost < least) {
      least = cost;
      best = Plan{token_lanes, pair, bn, split};
    }
  };
  auto busy = [](int64_t ctas) { return ctas >= kSms ? 1. : static_cast<double>(ctas) / kSms; };
  auto one_cta = [&](bool token_lanes, int bn, int stages) {
    const int64_t tiles = ceil_div(token_lanes ? m : n, kBM) * ceil_div(token_lanes ? n : m, bn);
    for (int split = 1; split <= kMaxSplit; split *= 2) {
      // A part has work, and all clusters are resident at once: a GPC has room for whole ones only, so clusters of
      // four and eight do not reach every SM (36 tiles of 4 parts took two waves, 21 us instead of 11).
      if (split > 1 && (k_tiles / split < 4 || tiles * split > (split == 2 ? kSms : 128) || bn > kMaxSplitBN ||
                        bn < 2 * split))
        break;
      const double step = most(2 * bn, 2050. / stages, 2 * (kBM + bn) * busy(tiles * split));
      const double out = (!token_lanes ? 60. : split == 1 ? 8. : 20.) * bn / split + (split > 1 ? 2500 : 0);
      offer(token_lanes, false, bn, split, ceil_div(tiles * split, kSms) * (step * ceil_div(k_tiles, split)) + out);
    }
  };
  if (m <= 16)
    one_cta(false, 16, GemmShape<16>::kStages);
  else if (m <= 32)
    one_cta(false, 32, GemmShape<32>::kStages);
  else if (m <= 64)
    one_cta(false, 64, GemmShape<64>::kStages);
  if (m > 32) {
    one_cta(true, 64, GemmShape<64>::kStages);
    one_cta(true, 128, GemmShape<128>::kStages);
    one_cta(true, 256, GemmShape<256>::kStages);
  }
  if (m > 128)
    for (int bn = 256; bn >= 128; bn -= 32) {
      const int64_t pairs = ceil_div(m, 2 * kBM) * ceil_div(n, bn);
      const double step = most(2 * bn, 3300. / PairShape::stages(bn), 2 * (kBM + bn / 2) * busy(2 * pairs));
      offer(true, true, bn, 1, ceil_div(pairs, kSms / 2) * (step * k_tiles) + 8. * bn + 1000);
    }
  return best;
}

static int make_map(CUtensorMap* m, const void* base, int64_t rows, int k, int64_t stride, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return TM_ERR_LAUNCH;
  cuuint64_t dims[2] = {static_cast<cuuint64_t>(k), static_cast<cuuint64_t>(rows)};
  cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride)};
  cuuint32_t box[2] = {static_cast<cuuint32_t>(kBK), static_cast<cuuint32_t>(box_rows)};
  cuuint32_t estr[2] = {1u, 1u};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? TM_OK : TM_ERR_TMAP;
}

template <int BN, bool kTokenLanes, typename OutT>
static int launch(const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& g, cudaStream_t st) {
  using S = GemmShape<BN>;
  auto kernel = gemm_kernel<BN, kTokenLanes, OutT>;
  if (!allow_smem<gemm_kernel<BN, kTokenLanes, OutT>, S::smem(kTokenLanes)>()) return TM_ERR_LAUNCH;
  const int64_t tiles = static_cast<int64_t>(g.tiles_a) * g.tiles_b;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(g.split > 1 ? tiles * g.split : tiles < kSms ? tiles : kSms));
  cfg.blockDim = dim3(kGemmThreads);
  cfg.dynamicSmemBytes = S::smem(kTokenLanes);
  cfg.stream = st;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (g.split > 1) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = static_cast<unsigned>(g.split);
    at[n].val.clusterDim.y = 1;
    at[n].val.clusterDim.z = 1;
    ++n;
  }
  if (g.beside) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = at;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, a, b, g) == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}

template <typename OutT>
static int launch_pair(const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& g, cudaStream_t st) {
  if (!allow_smem<gemm_pair_kernel<OutT>, PairShape::kSmem>()) return TM_ERR_LAUNCH;
  const int64_t tiles = static_cast<int64_t>(g.tiles_a) * g.tiles_b;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (tiles < kSms / 2 ? tiles : kSms / 2)));
  cfg.blockDim = dim3(PairShape::kThreads);
  cfg.dynamicSmemBytes = PairShape::kSmem;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = g.beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, gemm_pair_kernel<OutT>, a, b, g) == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}

template <typename OutT>
static int dispatch(const Plan& p, const CUtensorMap& a, const CUtensorMap& b, const GemmArgs& g, cudaStream_t st) {
  if (p.pair) return launch_pair<OutT>(a, b, g, st);
  if (p.token_lanes) {
    if (p.bn == 256) return launch<256, true, OutT>(a, b, g, st);
    if (p.bn == 128) return launch<128, true, OutT>(a, b, g, st);
    return launch<64, true, OutT>(a, b, g, st);
  }
  if (p.bn == 64) return launch<64, false, OutT>(a, b, g, st);
  if (p.bn == 32) return launch<32, false, OutT>(a, b, g, st);
  return launch<16, false, OutT>(a, b, g, st);
}

}  // namespace linear
}  // namespace tilemix

extern "C" int tm_quant_per_token_int8(const void* x, int dtype, int64_t x_stride, int64_t rows, int cols, int8_t* out,
                                       int64_t out_stride, float* scale, int* error_flag, void* stream) {
  (void)error_flag;  // nothing that only the device could see
  using namespace tilemix::linear;
  if (rows < 0 || cols <= 0) return TM_ERR_SHAPE;
  if (dtype != TM_DTYPE_FP16 && dtype != TM_DTYPE_BF16) return TM_ERR_UNSUPPORTED;
  if (rows > 0x7fffffffll) return TM_ERR_SHAPE;
  if (rows == 0) return TM_OK;
  if (!x || !out || !scale) return TM_ERR_NULL;
  if (!aligned(x, 2) || !aligned(scale, 4)) return TM_ERR_ALIGN;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (dtype == TM_DTYPE_FP16)
    launch_quant<__half>(x, x_stride, rows, cols, out, out_stride, scale, st);
  else
    launch_quant<__nv_bfloat16>(x, x_stride, rows, cols, out, out_stride, scale, st);
  return cudaGetLastError() == cudaSuccess ? TM_OK : TM_ERR_LAUNCH;
}

namespace tilemix {
namespace linear {
static int matmul(const int8_t* x8, int64_t x_stride, const float* x_scale, const int8_t* w8, int64_t w_stride,
                  const float* w_scale, const void* bias, void* out, int64_t out_stride, int out_dtype, int64_t tokens,
                  int out_features, int in_features, bool beside, int* error_flag, void* stream) {
  if (tokens < 0 || out_features <= 0 || in_features <= 0) return TM_ERR_SHAPE;
  if (out_dtype < TM_DTYPE_FP16 || out_dtype > TM_DTYPE_FP32) return TM_ERR_UNSUPPORTED;
  // int32 sums of in_features products of at most 127 * 127 (128 * 128, should a caller bring -128)
  if (in_features > 131071 || tokens > 0x7fffff00ll || out_features > 0x7fffff00) return TM_ERR_UNSUPPORTED;
  if (tokens == 0) return TM_OK;
  if (!x8 || !x_scale || !w8 || !w_scale || !out) return TM_ERR_NULL;
  const int es = out_dtype == TM_DTYPE_FP32 ? 4 : 2;
  const int64_t round_k = (static_cast<int64_t>(in_features) + 15) / 16 * 16;
  if (tokens == 1) x_stride = round_k;  // one row: its stride is never used, but has to suit the tensor map
  if (out_features == 1) w_stride = round_k;
  if (!aligned(x8, 16) || !aligned(w8, 16) || x_stride % 16 || w_stride % 16) return TM_ERR_ALIGN;
  if (!aligned(out, es) || !aligned(x_scale, 4) || !aligned(w_scale, 4) || (bias && !aligned(bias, es)))
    return TM_ERR_ALIGN;
  if (x_stride < in_features || w_stride < in_features) return TM_ERR_SHAPE;
  const int k_tiles = (in_features + kBK - 1) / kBK;
  const Plan p = plan_of(tokens, out_features, k_tiles);
  GemmArgs g{};
  g.rows_a = static_cast<int>(p.token_lanes ? tokens : out_features);
  g.rows_b = static_cast<int>(p.token_lanes ? out_features : tokens);
  g.k_tiles = k_tiles;
  g.split = p.split;
  g.bn = p.bn;
  g.tiles_a = (g.rows_a + (p.pair ? 2 : 1) * kBM - 1) / ((p.pair ? 2 : 1) * kBM);
  g.tiles_b = (g.rows_b + p.bn - 1) / p.bn;
  if (static_cast<int64_t>(g.tiles_a) * g.tiles_b * p.split > 0x7fffffffll - 1024) return TM_ERR_UNSUPPORTED;
  g.scale_a = p.token_lanes ? x_scale : w_scale;
  g.scale_b = p.token_lanes ? w_scale : x_scale;
  g.bias = bias;
  g.out = out;
  g.ldo = out_stride;
  g.vec = aligned(out, 16) && out_stride * es % 16 == 0;
  g.beside = beside;
  g.err = error_flag;
  CUtensorMap mx, mw;
  int rc = make_map(&mx, x8, tokens, in_features, x_stride, p.token_lanes ? kBM : p.bn);
  if (rc != TM_OK) return rc;
  rc = make_map(&mw, w8, out_features, in_features, w_stride, p.pair ? p.bn / 2 : p.token_lanes ? p.bn : kBM);
  if (rc != TM_OK) return rc;
  const CUtensorMap& ma = p.token_lanes ? mx : mw;
  const CUtensorMap& mb = p.token_lanes ? mw : mx;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (out_dtype == TM_DTYPE_FP16) return dispatch<__half>(p, ma, mb, g, st);
  if (out_dtype == TM_DTYPE_BF16) return dispatch<__nv_bfloat16>(p, ma, mb, g, st);
  return dispatch<float>(p, ma, mb, g, st);
}
}  // namespace linear
}  // namespace tilemix

extern "C" int tm_int8_matmul(const int8_t* x8, int64_t x_stride, const float* x_scale, const int8_t* w8,
                              int64_t w_stride, const float* w_scale, const void* bias, void* out, int64_t out_stride,
                              int out_dtype, int64_t tokens, int out_features, int in_features, int* error_flag,
                              void* stream) {
  return tilemix::linear::matmul(x8, x_stride, x_scale, w8, w_stride, w_scale, bias, out, out_stride, out_dtype, tokens,
                                 out_features, in_features, false, error_flag, stream);
}

extern "C" int tm_int8_linear(const void* x, int dtype, int64_t x_stride, int8_t* x8, int64_t x8_stride, float* x_scale,
                              const int8_t* w8, int64_t w_stride, const float* w_scale, const void* bias, void* out,
                              int64_t out_stride, int64_t tokens, int out_features, int in_features, int* error_flag,
                              void* stream) {
  if (dtype != TM_DTYPE_FP16 && dtype != TM_DTYPE_BF16) return TM_ERR_UNSUPPORTED;
  const int rc = tm_quant_per_token_int8(x, dtype, x_stride, tokens, in_features, x8, x8_stride, x_scale, error_flag,
                                         stream);
  if (rc != TM_OK) return rc;
  return tilemix::linear::matmul(x8, x8_stride, x_scale, w8, w_stride, w_scale, bias, out, out_stride, dtype, tokens,
                                 out_features, in_features, true, error_flag, stream);
}
