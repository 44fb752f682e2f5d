// Layout of the paged 4-bit key/value cache (kv4_cache.cu writes and reads it
// back, kv4_attn.cu attends over it).
//
// The pool is uint8 [pages, kv_heads, page bytes]; a page holds page_size (a
// multiple of 16) tokens of one KV head as a run of 16-token blocks of 20 D
// bytes. Every group of 32 channels of one (token, head) row x has an fp16
// scale s and minimum m and 4-bit codes n: x ~ s n + m, so a value costs 5 bits.
// With G = D / 32 groups a block is
//   K codes   16 x D/2 bytes  token row: chunk t = 0..3, word j = 0..G-1 (32 bits):
//                             channels 32 j + 8 t + i at nibble i
//   K scales  16 x 4G bytes   token row: group j: s, m
//   V codes   16 x D/2 bytes  token row: chunk g = 0..7, half-word j = 0..G-1:
//                             channels 32 j + 4 g + i at nibble i
//   V scales  16 x 4G bytes   group j, t = 0..3: s of tokens t, t + 4, t + 8, t + 12,
//                             then m of the same four
// The order inside a row is the order in which the lanes of a warp hold the
// operands of mma.m16n8k16: a K chunk is one lane's whole share of a key row (the
// A operand's columns), a V chunk one lane's share of the transposed V (its
// rows), so each is one shared-memory load and needs no exchange between lanes;
// the V scales lie so that the scales of a lane's key pairs arrive as half2. K
// and V of a block are adjacent: one bulk copy moves everything a step needs.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

namespace tilemix {
namespace kv4 {

constexpr int kBlockTokens = 16;

template <int D>
struct Layout {
  static constexpr int kGroups = D / 32;
  static constexpr int kRowBytes = D / 2;           // codes of one token row
  static constexpr int kScaleBytes = 4 * kGroups;   // scales of one token row
  static constexpr int kOffKScale = kBlockTokens * kRowBytes;
  static constexpr int kOffV = kOffKScale + kBlockTokens * kScaleBytes;
  static constexpr int kOffVScale = kOffV + kBlockTokens * kRowBytes;
  static constexpr int kBlockBytes = 2 * kOffV;     // 20 D
  // Byte offset inside the V scales of token `tok`'s scale of group j (its minimum 8 bytes on).
  static __host__ __device__ constexpr int v_scale(int j, int tok) { return (j * 4 + tok % 4) * 16 + tok / 4 * 2; }
};

inline bool aligned(const void* p, int64_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

__host__ __device__ constexpr int block_bytes(int head_dim) { return 20 * head_dim; }

}  // namespace kv4

// Opt-in dynamic shared memory of a kernel: set once for each device that launches it.
template <auto kKernel, int kBytes>
inline bool allow_smem() {
  static std::atomic<uint64_t> done{0};  // bit: device
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return true;
  if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes) != cudaSuccess)
    return false;
  done.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

}  // namespace tilemix
