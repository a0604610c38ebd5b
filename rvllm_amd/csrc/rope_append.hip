// rope_append.hip - q and k rotated by their tokens' positions, k and v
// written into the paged cache: f16 or f32 cells, or the 8-bit records.
//
// Per token and pair p < rot / 2, in f64:
//   angle = position * inv_freq[p],  c = factor cos, s = factor sin,
//   (a, b) -> (a c - b s, a s + b c),
// the pairs being (p, p + rot / 2) or, interleaved, (2 p, 2 p + 1); dims from
// rot on stay. With norm weights, x / sqrt(mean x^2 + eps) * w comes first.
// An 8-bit row takes scale = f32(max |x| / 127) and code = rint(x / scale),
// ties to even. f64 keeps the angles of positions near 2^32 to 1e-7 and the
// codes equal to the definition's: values next to a code's border would
// round to either side of it in f32 (VALU f64 runs at the f32 rate here, and
// the launch is bound by HBM).
#include <type_traits>

#include "q8.h"

using rvkv_detail::fail;
using rvkv_detail::hip_fail;

namespace {

enum CellKind { kF16, kF32, kQ8 };

struct RopeArgs {
  const void *q, *k, *v;
  void *q_out;
  uint64_t q_stride, k_stride, v_stride;  // elements between rows
  const float *q_norm, *k_norm;
  const uint32_t *positions;
  const float *inv_freq;
  const uint32_t *slot_block, *slot_off;
  unsigned char *kc, *vc;
  uint64_t rec;  // bytes of a block in kc and vc
  uint32_t rows, n_heads, n_kv, hd, bs, num_blocks, rot, interleaved;
  float eps, factor;
};

// sin and cos of x >= 0 below 2^33: x less the nearest multiple of pi / 2
// (in two parts, 106 bits; the fma keeps the difference of near values
// exact), then the Taylor sums to x^17 / x^18 on |r| <= pi / 4, whose rest is
// below 1e-18.
__device__ __forceinline__ void sincos64(double x, double &s, double &c) {
  const double n = __builtin_rint(x * 0.63661977236758134308);
  double r = __builtin_fma(-n, 1.57079632679489655800, x);
  r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
  const double z = r * r;
  double ps = 1.0 / 355687428096000.0;  // 1 / 17!
  ps = __builtin_fma(ps, z, -1.0 / 1307674368000.0);
  ps = __builtin_fma(ps, z, 1.0 / 6227020800.0);
  ps = __builtin_fma(ps, z, -1.0 / 39916800.0);
  ps = __builtin_fma(ps, z, 1.0 / 362880.0);
  ps = __builtin_fma(ps, z, -1.0 / 5040.0);
  ps = __builtin_fma(ps, z, 1.0 / 120.0);
  ps = __builtin_fma(ps, z, -1.0 / 6.0);
  ps = __builtin_fma(ps * z, r, r);
  double pc = -1.0 / 6402373705728000.0;  // 1 / 18!
  pc = __builtin_fma(pc, z, 1.0 / 20922789888000.0);
  pc = __builtin_fma(pc, z, -1.0 / 87178291200.0);
  pc = __builtin_fma(pc, z, 1.0 / 479001600.0);
  pc = __builtin_fma(pc, z, -1.0 / 3628800.0);
  pc = __builtin_fma(pc, z, 1.0 / 40320.0);
  pc = __builtin_fma(pc, z, -1.0 / 720.0);
  pc = __builtin_fma(pc, z, 1.0 / 24.0);
  pc = __builtin_fma(pc, z, -0.5);
  pc = __builtin_fma(pc, z, 1.0);
  const uint32_t quad = (uint32_t)(int64_t)n & 3;
  s = quad & 1 ? pc : ps;
  c = quad & 1 ? ps : pc;
  if (quad & 2) s = -s;
  if ((quad + 1) & 2) c = -c;
}

// x rounded once (f64 to f16 by way of an f32 that is rounded to odd).
__device__ __forceinline__ void round_to(double x, float &out) {
  out = (float)x;
}
__device__ __forceinline__ void round_to(double x, _Float16 &out) {
  const float f = (float)x;
  uint32_t u = __float_as_uint(f);
  if ((double)f != x && x == x && !(u & 1))
    u += __builtin_fabs((double)f) > __builtin_fabs(x) ? -1 : 1;
  out = (_Float16)__uint_as_float(u);
}

// rint(x / s), ties to even: by the product with inv = 1 / s, and by the
// remainder where that lies within 1e-6 of a border.
__device__ __forceinline__ int quantise(double x, double s, double inv) {
  double r = __builtin_rint(x * inv);
  const double d = __builtin_fma(-r, s, x);
  const double over = __builtin_fabs(d) - 0.5 * s;
  if (over > -1e-6 * s) {
    const bool odd = (int)r & 1;
    if (over > 0.0 || (over == 0.0 && odd)) r += d > 0.0 ? 1.0 : -1.0;
  }
  return (int)__builtin_fmin(__builtin_fmax(r, -127.0), 127.0);
}

template <bool VEC, int E, typename In>
__device__ __forceinline__ void load_row(const In *p, In (&x)[E]) {
  static_assert(VEC && E == 8, "eight elements by 16-byte loads");
  constexpr int N = 16 / sizeof(In);
#pragma unroll
  for (int i = 0; i < E / N; ++i)
    *reinterpret_cast<uint4 *>(x + i * N) =
        *reinterpret_cast<const uint4 *>(p + i * N);
}

// One workgroup a token: its angles into LDS, then T lanes a head. VEC: a
// lane owns 8 consecutive dims (T = hd / 8) and, in the half layout, loads
// its partners' 8 too (they lie in the same lines). Otherwise 16 lanes a
// head, lane l owning dims l, l + 16, ... (any hd, rot, stride, alignment).
template <typename In, int CELL, int T, bool VEC>
__global__ void __launch_bounds__(256) rope_append_kernel(RopeArgs a) {
  constexpr int E = VEC ? 8 : 16;
  __shared__ double cs[128], sn[128];
  const uint32_t row = blockIdx.x;
  const uint32_t half = a.rot / 2;
  for (uint32_t p = threadIdx.x; p < half; p += 256) {
    double s, c;
    sincos64((double)a.positions[row] * (double)a.inv_freq[p], s, c);
    cs[p] = c * (double)a.factor;
    sn[p] = s * (double)a.factor;
  }
  __syncthreads();
  const uint32_t blk = a.slot_block[row], off = a.slot_off[row];
  const bool slot_ok = blk < a.num_blocks && off < a.bs;
  const uint32_t lane = threadIdx.x % T;
  const uint32_t n_slots = a.n_heads + 2 * a.n_kv;
  const uint32_t hd = a.hd;
  for (uint32_t slot = threadIdx.x / T; slot < n_slots; slot += 256 / T) {
    const bool is_q = slot < a.n_heads;
    const bool is_v = slot >= a.n_heads + a.n_kv;
    const uint32_t hh = is_q ? slot
                             : (is_v ? slot - a.n_heads - a.n_kv
                                     : slot - a.n_heads);
    if (!is_q && !slot_ok) continue;
    const In *src = is_q ? (const In *)a.q + (size_t)row * a.q_stride
                         : (is_v ? (const In *)a.v + (size_t)row * a.v_stride
                                 : (const In *)a.k + (size_t)row * a.k_stride);
    src += (size_t)hh * hd;
    const float *w = is_v ? nullptr : (is_q ? a.q_norm : a.k_norm);
    const auto dim = [&](int e) {
      return VEC ? 8 * lane + e : lane + 16 * (uint32_t)e;
    };
    double x[E];
    if constexpr (VEC) {
      alignas(16) In own[E];
      load_row<VEC, E>(src + 8 * lane, own);
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = (double)own[e];
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = dim(e) < hd ? (double)src[dim(e)] : 0.0;
    }
    double norm = 1.0;
    if (w) {  // (uniform over a head's lanes)
      double ss = 0.0;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = __builtin_fma(x[e], x[e], ss);
#pragma unroll
      for (int o = T / 2; o >= 1; o >>= 1) ss += __shfl_xor(ss, o, T);
      norm = 1.0 / sqrt(ss / (double)hd + (double)a.eps);
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (VEC || dim(e) < hd) x[e] = x[e] * norm * (double)w[dim(e)];
    }
    if (!is_v && a.rot) {
      if constexpr (VEC) {
        const uint32_t d0 = 8 * lane;
        if (d0 < a.rot) {
          if (a.interleaved) {
#pragma unroll
            for (int e = 0; e < E; e += 2) {
              const double c = cs[(d0 + e) / 2], s = sn[(d0 + e) / 2];
              const double u = x[e], v = x[e + 1];
              x[e] = u * c - v * s;
              x[e + 1] = u * s + v * c;
            }
          } else {
            const bool is_a = d0 < half;
            const uint32_t d1 = is_a ? d0 + half : d0 - half;
            const uint32_t p0 = is_a ? d0 : d1;
            alignas(16) In other[E];
            load_row<VEC, E>(src + d1, other);
#pragma unroll
            for (int e = 0; e < E; ++e) {
              double y = (double)other[e];
              if (w) y = y * norm * (double)w[d1 + e];
              const double s = is_a ? -sn[p0 + e] : sn[p0 + e];
              x[e] = x[e] * cs[p0 + e] + y * s;
            }
          }
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          const uint32_t d = dim(e);
          if (d < a.rot) {
            const bool is_a = a.interleaved ? !(d & 1) : d < half;
            const uint32_t p = a.interleaved ? d >> 1 : (is_a ? d : d - half);
            const uint32_t d1 = a.interleaved ? d ^ 1
                                              : (is_a ? d + half : d - half);
            double y = (double)src[d1];
            if (w) y = y * norm * (double)w[d1];
            x[e] = x[e] * cs[p] + y * (is_a ? -sn[p] : sn[p]);
          }
        }
      }
    }
    if (is_q || CELL != kQ8) {
      // q in its own type, or a row of f16 / f32 cells.
      const auto put = [&](auto *out) {
        using Out = typename std::remove_pointer<decltype(out)>::type;
        if constexpr (VEC) {
          alignas(16) Out y[E];
#pragma unroll
          for (int e = 0; e < E; ++e) round_to(x[e], y[e]);
          constexpr int N = 16 / sizeof(Out);
#pragma unroll
          for (int i = 0; i < E / N; ++i)
            *reinterpret_cast<uint4 *>(out + 8 * lane + i * N) =
                *reinterpret_cast<const uint4 *>(y + i * N);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (dim(e) < hd) round_to(x[e], out[dim(e)]);
        }
      };
      if (is_q) {
        put((In *)a.q_out + ((size_t)row * a.n_heads + hh) * hd);
      } else {
        unsigned char *block = (is_v ? a.vc : a.kc) + blk * a.rec;
        const size_t at = ((size_t)hh * a.bs + off) * hd;
        if (CELL == kF16) put((_Float16 *)block + at);
        else put((float *)block + at);
      }
      continue;
    }
    double top = 0.0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const double m = __builtin_fabs(x[e]);
      // (a NaN counts as infinite: the row is then not finite)
      top = m <= top ? top : (m == m ? m : __builtin_inf());
    }
#pragma unroll
    for (int o = T / 2; o >= 1; o >>= 1)
      top = __builtin_fmax(top, __shfl_xor(top, o, T));
    const float scale = top < __builtin_inf() ? (float)(top / 127.0)
                                              : __builtin_nanf("");
    const double s = (double)scale, inv = 1.0 / s;
    int code[E];
#pragma unroll
    for (int e = 0; e < E; ++e)
      code[e] = scale > 0.f ? quantise(x[e], s, inv) : 0;
    unsigned char *block = (is_v ? a.vc : a.kc) + blk * a.rec;
    unsigned char *tile = block + (size_t)hh * a.bs * hd;
    if (is_v) {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (VEC || dim(e) < hd)
          tile[(size_t)dim(e) * a.bs + off] = (unsigned char)code[e];
    } else if constexpr (VEC) {
      uint2 pack;
      pack.x = (code[0] & 255) | (code[1] & 255) << 8 | (code[2] & 255) << 16 |
               (uint32_t)code[3] << 24;
      pack.y = (code[4] & 255) | (code[5] & 255) << 8 | (code[6] & 255) << 16 |
               (uint32_t)code[7] << 24;
      *reinterpret_cast<uint2 *>(tile + (size_t)off * hd + 8 * lane) = pack;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (dim(e) < hd)
          tile[(size_t)off * hd + dim(e)] = (unsigned char)code[e];
    }
    if (lane == 0)
      *reinterpret_cast<float *>(block + (size_t)a.n_kv * a.bs * hd +
                                 ((size_t)hh * a.bs + off) * 4) = scale;
  }
}

template <typename In, int CELL>
void launch(const RopeArgs &a, bool vec, hipStream_t st) {
  const dim3 grid(a.rows), block(256);
  if (vec) {
    switch (a.hd) {
      case 32: hipLaunchKernelGGL((rope_append_kernel<In, CELL, 4, true>), grid, block, 0, st, a); return;
      case 64: hipLaunchKernelGGL((rope_append_kernel<In, CELL, 8, true>), grid, block, 0, st, a); return;
      case 128: hipLaunchKernelGGL((rope_append_kernel<In, CELL, 16, true>), grid, block, 0, st, a); return;
      case 256: hipLaunchKernelGGL((rope_append_kernel<In, CELL, 32, true>), grid, block, 0, st, a); return;
      default: break;
    }
  }
  hipLaunchKernelGGL((rope_append_kernel<In, CELL, 16, false>), grid, block, 0,
                     st, a);
}

// The checks that both pools' entry points share; fills a.
int rope_append(const char *op, int cell, hipStream_t st, RopeArgs &a,
                rvkv_dtype dtype, uint32_t interleaved) {
  if (dtype != RVKV_F16 && dtype != RVKV_F32)
    return fail(RVKV_EINVAL, op, "dtype must be F16 or F32");
  if (!a.k || !a.v || !a.slot_block || !a.slot_off)
    return fail(RVKV_EINVAL, op, "NULL k/v/block_ids/offsets");
  if (a.n_heads % a.n_kv != 0)
    return fail(RVKV_EINVAL, op, "n_heads must be a multiple of n_kv_heads");
  if (a.n_heads && (!a.q || !a.q_out))
    return fail(RVKV_EINVAL, op, "NULL q/q_out");
  if (a.rot % 2 || a.rot > a.hd)
    return fail(RVKV_EINVAL, op, "rot_dim must be even and at most head_dim");
  if (a.rot && (!a.positions || !a.inv_freq))
    return fail(RVKV_EINVAL, op, "NULL positions/inv_freq");
  if (a.hd > 256)
    return fail(RVKV_EUNSUPPORTED, op, "head_dim must be at most 256");
  if (interleaved > 1)
    return fail(RVKV_EINVAL, op, "interleaved must be 0 or 1");
  if (a.rows > 0xffffffu)  // (a launch holds fewer than 2^32 threads)
    return fail(RVKV_EUNSUPPORTED, op, "too many rows for one launch");
  const uint64_t kv_row = (uint64_t)a.n_kv * a.hd;
  if (a.rows > 1 && (a.k_stride < kv_row || a.v_stride < kv_row ||
                     (a.n_heads && a.q_stride < (uint64_t)a.n_heads * a.hd)))
    return fail(RVKV_EINVAL, op, "a stride is shorter than its row");
  const uint32_t eb = dtype == RVKV_F32 ? 4 : 2;
  if ((uintptr_t)a.q % eb || (uintptr_t)a.k % eb || (uintptr_t)a.v % eb ||
      (uintptr_t)a.q_out % eb)
    return fail(RVKV_EINVAL, op, "q/k/v/q_out must be aligned to their type");
  a.interleaved = interleaved;
  bool vec = a.hd == 32 || a.hd == 64 || a.hd == 128 || a.hd == 256;
  vec = vec && (interleaved ? a.rot % 8 == 0 : a.rot % 16 == 0);
  for (uint64_t x : {(uint64_t)(uintptr_t)a.q, (uint64_t)(uintptr_t)a.k,
                     (uint64_t)(uintptr_t)a.v, (uint64_t)(uintptr_t)a.q_out,
                     a.q_stride * eb, a.k_stride * eb, a.v_stride * eb})
    vec = vec && x % 16 == 0;
  if (dtype == RVKV_F16) {
    if (cell == kQ8) launch<_Float16, kQ8>(a, vec, st);
    else if (cell == kF16) launch<_Float16, kF16>(a, vec, st);
    else launch<_Float16, kF32>(a, vec, st);
  } else {
    if (cell == kQ8) launch<float, kQ8>(a, vec, st);
    else if (cell == kF16) launch<float, kF16>(a, vec, st);
    else launch<float, kF32>(a, vec, st);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RVKV_OK : hip_fail(op, e);
}

RopeArgs rope_args(const void *q, uint64_t q_stride, const void *k,
                   uint64_t k_stride, const void *v, uint64_t v_stride,
                   uint32_t rows, uint32_t n_heads, const float *q_norm,
                   const float *k_norm, float eps, const uint32_t *positions,
                   const float *inv_freq, uint32_t rot_dim, float attn_factor,
                   const uint32_t *slot_block, const uint32_t *slot_off,
                   void *q_out) {
  RopeArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.q_out = q_out;
  a.q_stride = q_stride;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.q_norm = q_norm;
  a.k_norm = k_norm;
  a.positions = positions;
  a.inv_freq = inv_freq;
  a.slot_block = slot_block;
  a.slot_off = slot_off;
  a.rows = rows;
  a.n_heads = n_heads;
  a.rot = rot_dim;
  a.eps = eps;
  a.factor = attn_factor;
  return a;
}

}  // namespace

extern "C" {

int rvkv_rope_append(rvkv_pool *pool, uint32_t layer, const void *q,
                     uint64_t q_stride, const void *k, uint64_t k_stride,
                     const void *v, uint64_t v_stride, rvkv_dtype dtype,
                     uint32_t rows, uint32_t n_heads, const float *q_norm,
                     const float *k_norm, float eps, const uint32_t *positions,
                     const float *inv_freq, uint32_t rot_dim,
                     uint32_t interleaved, float attn_factor,
                     const uint32_t *slot_block, const uint32_t *slot_off,
                     void *q_out) {
  const char *op = "rope_append";
  if (!pool) return fail(RVKV_EINVAL, op, "pool is NULL");
  if (layer >= pool->n_layers)
    return fail(RVKV_EINVAL, op, "layer out of range");
  if (rows == 0) return RVKV_OK;
  const int rc = rvkv_detail::q8_device(op, pool->device);
  if (rc) return rc;
  RopeArgs a = rope_args(q, q_stride, k, k_stride, v, v_stride, rows, n_heads,
                         q_norm, k_norm, eps, positions, inv_freq, rot_dim,
                         attn_factor, slot_block, slot_off, q_out);
  a.n_kv = pool->n_kv;
  a.hd = pool->head_dim;
  a.bs = pool->block_size;
  a.num_blocks = pool->num_blocks;
  a.kc = reinterpret_cast<unsigned char *>(pool->tensor(layer, 0));
  a.vc = reinterpret_cast<unsigned char *>(pool->tensor(layer, 1));
  a.rec = pool->block16 * 2;
  return rope_append(op, pool->f32() ? kF32 : kF16, pool->stream, a, dtype,
                     interleaved);
}

int rvkv_q8_rope_append(rvkv_q8_pool *pool, uint32_t layer, const void *q,
                        uint64_t q_stride, const void *k, uint64_t k_stride,
                        const void *v, uint64_t v_stride, rvkv_dtype dtype,
                        uint32_t rows, uint32_t n_heads, const float *q_norm,
                        const float *k_norm, float eps,
                        const uint32_t *positions, const float *inv_freq,
                        uint32_t rot_dim, uint32_t interleaved,
                        float attn_factor, const uint32_t *slot_block,
                        const uint32_t *slot_off, void *q_out) {
  const char *op = "rope_append";
  if (!pool) return fail(RVKV_EINVAL, op, "pool is NULL");
  if (layer >= pool->n_layers)
    return fail(RVKV_EINVAL, op, "layer out of range");
  if (rows == 0) return RVKV_OK;
  const int rc = rvkv_detail::q8_device(op, pool->device);
  if (rc) return rc;
  RopeArgs a = rope_args(q, q_stride, k, k_stride, v, v_stride, rows, n_heads,
                         q_norm, k_norm, eps, positions, inv_freq, rot_dim,
                         attn_factor, slot_block, slot_off, q_out);
  a.n_kv = pool->n_kv;
  a.hd = pool->head_dim;
  a.bs = pool->block_size;
  a.num_blocks = pool->num_blocks;
  a.kc = pool->tensor(layer, 0);
  a.vc = pool->tensor(layer, 1);
  a.rec = pool->rec;
  return rope_append(op, kQ8, pool->stream, a, dtype, interleaved);
}

}  // extern "C"
