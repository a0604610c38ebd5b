// q8.h - the 8-bit paged cache: its pool object and record layout, shared by
// the sources that write it (rope_append.hip) and read it (q8.hip,
// q8_prefill.hip).
#pragma once
#include "pool.h"

// One block of one layer's K or V is a record of rec bytes:
//   int8 codes of every KV head, bs * hd of them, K as [bs][hd], V as [hd][bs];
//   then f32 scales [n_kv][bs]; then padding to 256 bytes.
// K rows lie as the S = K q' product reads them (16 bytes of one key's dims a
// lane), V transposed, as the V' P product reads it (16 keys of one dim a
// lane): both attentions load matrix operands straight from the record.
// Records of a tensor lie one behind the other, tensors as in the f16 pool:
// [layer][K, V][num_blocks]. A row of one token and head stands for
// code * scale, scale = f32(max |x| / 127).
struct rvkv_q8_pool {
  uint32_t n_layers, num_blocks, block_size, n_kv, head_dim;
  size_t rec;           // bytes of one block's record
  size_t tensor_bytes;  // num_blocks records
  hipStream_t stream;
  int device;
  unsigned char *base;
  bool owned;

  unsigned char *tensor(uint32_t layer, uint32_t which) const {
    return base + ((size_t)layer * 2 + which) * tensor_bytes;
  }
};

namespace rvkv_detail {
// Keys of a sequence that the attentions read at most, so that no key index
// wraps in 32 bits.
constexpr uint32_t kMaxKeys = 0xffffff00u;
// Fails unless the calling thread's current device is the pool's: a launch
// on the null stream would otherwise run on another GPU.
int q8_device(const char *op, int device);
}  // namespace rvkv_detail

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef int int4v __attribute__((ext_vector_type(4)));
typedef float float4v __attribute__((ext_vector_type(4)));
typedef float float16v __attribute__((ext_vector_type(16)));

// A value that is the wave's, as the compiler cannot tell by itself.
__device__ __forceinline__ uint32_t uniform(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_readfirstlane((int)x);
}

// Four int8 codes as f16, exactly: code ^ 0x80 = code + 128 in a byte below
// 0x64 is the f16 1024 + 128 + code; one subtraction leaves the code.
__device__ __forceinline__ void codes_to_half4(uint32_t c, half2v &lo,
                                               half2v &hi) {
  c ^= 0x80808080u;
  const half2v bias = {(_Float16)1152.f, (_Float16)1152.f};
  lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(
                                      0x64646464u, c, 0x04010400u)) - bias;
  hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(
                                      0x64646464u, c, 0x04030402u)) - bias;
}

// Eight codes (two words) as one f16 matrix operand.
__device__ __forceinline__ half8v codes_to_half8(uint32_t a, uint32_t b) {
  half2v p[4];
  codes_to_half4(a, p[0], p[1]);
  codes_to_half4(b, p[2], p[3]);
  half8v r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[2 * i] = p[i][0];
    r[2 * i + 1] = p[i][1];
  }
  return r;
}

// A power of two above top: 2^(exponent - 127), within what q can be scaled
// by.
__device__ __forceinline__ uint32_t scale_exponent(float top) {
  const uint32_t ex = (__float_as_uint(top) >> 23) + 1;
  return ex < 16 ? 16 : (ex > 252 ? 252 : ex);
}
// Where the running power of two above the V scales starts.
constexpr float kVnorm0 = 0x1p-100f;
