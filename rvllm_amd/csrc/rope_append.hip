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
// round to either side of it in f32.
//
// 8191 packed rows of 16 + 8 heads of 128, normed, f16, into 8-bit cells: 64 us
// for 118 MB; 8000 rows of 32 + 8 heads of 64 without norms 34 us for 91 MB.
// The vector units are busy 55 % of the time, f64 of K and the codes' borders
// first, and the waves, four a SIMD, wait half of theirs. V codes of a block
// are written by four workgroups on four XCDs, 83 MB where 51 are needed;
// neighbouring tokens on one XCD write 50 and take 69 us.
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

// The largest, or the sum, of T lanes, in every one of them (T 4 to 32). Each
// step adds the lanes' mirror image in twice as wide a group, by DPP.
template <int CTRL>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_mov_dpp((int)u, CTRL, 0xf, 0xf, true);
  const uint32_t hi =
      __builtin_amdgcn_mov_dpp((int)(u >> 32), CTRL, 0xf, 0xf, true);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <int T, typename F>
__device__ __forceinline__ double over_lanes(double x, F f) {
  x = f(x, dpp<0xb1>(x));             // quad_perm 1 0 3 2
  x = f(x, dpp<0x4e>(x));             // quad_perm 2 3 0 1
  if (T > 4) x = f(x, dpp<0x141>(x));  // row_half_mirror
  if (T > 8) x = f(x, dpp<0x140>(x));  // row_mirror
  if (T > 16) x = f(x, __shfl_xor(x, 16));
  return x;
}

// 1 / sqrt(x) for x > 0, normal: the instruction's start, then two Newton
// steps (each doubles its more than 20 bits).
__device__ __forceinline__ double rsqrt64(double x) {
  double y = __builtin_amdgcn_rsq(x);
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double e = __builtin_fma(-x * y, y, 1.0);
    y = __builtin_fma(0.5 * y, e, y);
  }
  return y;
}

// Eight elements of a row, by 16-byte accesses.
template <typename X>
struct Vec8 {
  typedef X type __attribute__((ext_vector_type(8), aligned(16)));
};

// The code of a value x that f32 holds as xf to within 2^-23 of itself, by the
// product with inv = 1 / s to 2^-22: the quotient is off by less than 127 *
// 2^-21 < 2^-14, so a rounding further than that from a border is the exact
// one's, and the others (one in 4000 values) are made exactly. (A scale that
// is no normal number gives a quotient that is not below the border.)
__device__ __forceinline__ int code_of(float xf, double x, float s, float inv) {
  const float t = xf * inv, r = __builtin_rintf(t);
  if (__builtin_fabsf(t - r) < 0.5f - 0x1p-14f && s > 0x1p-100f)
    return (int)__builtin_fminf(__builtin_fmaxf(r, -127.f), 127.f);
  if (!(s > 0.f)) return 0;
  return quantise(x, (double)s, 1.0 / (double)s);
}

// The wide form: R tokens a workgroup, T lanes a head (T >= hd / 8, lanes
// behind the head idle), lane l owning dims 8 l .. 8 l + 7; in the half layout
// it also loads its partners' 8 (they lie in the same lines). The workgroup's
// threads share the tokens' angles out between them first. f16 q is turned in
// f32 (its angles come from f64), k in f64: codes go by it.
//
// A token's V codes lie bs bytes apart, one byte a dim. With R 4, tokens in
// consecutive slots, as prompts have them, put their four bytes of a dim into
// one store.
template <typename In, int CELL, int T, int R>
__global__ void __launch_bounds__(256) rope_append_kernel(RopeArgs a) {
  typedef typename Vec8<In>::type In8;
  __shared__ double cs[R][128], sn[R][128];
  const uint32_t row0 = blockIdx.x * R;
  const uint32_t n_rows = a.rows - row0 < R ? a.rows - row0 : R;
  const uint32_t half = a.rot / 2;
  for (uint32_t i = threadIdx.x; i < half * n_rows; i += 256) {
    const uint32_t r = i / half, p = i - r * half;
    double s, c;
    sincos64((double)a.positions[row0 + r] * (double)a.inv_freq[p], s, c);
    cs[r][p] = c * (double)a.factor;
    sn[r][p] = s * (double)a.factor;
  }
  uint32_t blk[R], off[R];
  bool ok[R], run = R > 1 && n_rows == R;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool have = (uint32_t)r < n_rows;
    blk[r] = have ? a.slot_block[row0 + r] : 0xffffffffu;
    off[r] = have ? a.slot_off[row0 + r] : 0;
    ok[r] = blk[r] < a.num_blocks && off[r] < a.bs;
    run = run && ok[r] && blk[r] == blk[0] && off[r] == off[0] + r;
  }
  __syncthreads();
  const uint32_t lane = threadIdx.x % T, hd = a.hd, d0 = 8 * lane;
  const uint32_t n_slots = a.n_heads + 2 * a.n_kv;
  const bool mine = d0 < hd;
  const uint32_t dl = mine ? d0 : 0;  // (idle lanes load what lane 0 does)
  for (uint32_t slot = threadIdx.x / T; slot < n_slots; slot += 256 / T) {
    const bool is_q = slot < a.n_heads;
    const bool is_v = slot >= a.n_heads + a.n_kv;
    const uint32_t hh = is_q ? slot
                             : (is_v ? slot - a.n_heads - a.n_kv
                                     : slot - a.n_heads);
    const uint64_t stride = is_q ? a.q_stride : (is_v ? a.v_stride : a.k_stride);
    const In *src = (const In *)(is_q ? a.q : (is_v ? a.v : a.k)) +
                    row0 * stride + (size_t)hh * hd;
    const float *w = is_v ? nullptr : (is_q ? a.q_norm : a.k_norm);
    const bool turn = !is_v && dl < a.rot;
    const bool is_a = dl < half;
    const uint32_t d1 = !turn || a.interleaved ? dl
                                               : (is_a ? dl + half : dl - half);
    const uint32_t p0 = a.interleaved ? dl / 2 : (is_a ? dl : d1);
    float wx[8], wy[8];
    if (w) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        wx[e] = w[dl + e];
        wy[e] = w[d1 + e];
      }
    }
    In8 own[R], other[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const uint32_t rr = (uint32_t)r < n_rows ? r : 0;
      own[r] = *reinterpret_cast<const In8 *>(src + rr * stride + dl);
      other[r] = own[r];
      if (turn && !a.interleaved)
        other[r] = *reinterpret_cast<const In8 *>(src + rr * stride + d1);
    }
    uint32_t vcode[8] = {};
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if ((uint32_t)r >= n_rows) break;
      double norm = 1.0;
      if (w) {
        double ss = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double x = (double)own[r][e];
          ss = __builtin_fma(x, x, ss);
        }
        ss = over_lanes<T>(mine ? ss : 0.0,
                           [](double x, double y) { return x + y; });
        norm = rsqrt64(ss / (double)hd + (double)a.eps);
      }
      if (is_q && sizeof(In) == 2) {
        float x[8];
        const float nf = (float)norm;
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = w ? (float)own[r][e] * nf * wx[e] : (float)own[r][e];
        if (turn && a.interleaved) {
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            const float c = (float)cs[r][p0 + e / 2];
            const float s = (float)sn[r][p0 + e / 2];
            const float u = x[e], v = x[e + 1];
            x[e] = u * c - v * s;
            x[e + 1] = u * s + v * c;
          }
        } else if (turn) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float y = w ? (float)other[r][e] * nf * wy[e]
                              : (float)other[r][e];
            const float s = (float)sn[r][p0 + e];
            x[e] = __builtin_fmaf(x[e], (float)cs[r][p0 + e],
                                  is_a ? -y * s : y * s);
          }
        }
        In8 y;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = (In)x[e];
        if (mine)
          *reinterpret_cast<In8 *>(
              (In *)a.q_out + ((size_t)(row0 + r) * a.n_heads + hh) * hd + d0) =
              y;
        continue;
      }
      double x[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[e] = w ? (double)own[r][e] * norm * (double)wx[e]
                 : (double)own[r][e];
      if (turn && a.interleaved) {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const double c = cs[r][p0 + e / 2], s = sn[r][p0 + e / 2];
          const double u = x[e], v = x[e + 1];
          x[e] = u * c - v * s;
          x[e + 1] = u * s + v * c;
        }
      } else if (turn) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const double y = w ? (double)other[r][e] * norm * (double)wy[e]
                             : (double)other[r][e];
          const double s = is_a ? -sn[r][p0 + e] : sn[r][p0 + e];
          x[e] = x[e] * cs[r][p0 + e] + y * s;
        }
      }
      const auto put = [&](auto *out) {
        using Out = typename std::remove_pointer<decltype(out)>::type;
        typename Vec8<Out>::type y;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          Out z;
          round_to(x[e], z);
          y[e] = z;
        }
        if (mine)
          *reinterpret_cast<typename Vec8<Out>::type *>(out + d0) = y;
      };
      if (is_q) {
        put((In *)a.q_out + ((size_t)(row0 + r) * a.n_heads + hh) * hd);
        continue;
      }
      unsigned char *block = (is_v ? a.vc : a.kc) + (ok[r] ? blk[r] : 0) * a.rec;
      const size_t row_at = (size_t)hh * a.bs + off[r];
      if (CELL != kQ8) {
        if (ok[r]) {
          if (CELL == kF16) put((_Float16 *)block + row_at * hd);
          else put((float *)block + row_at * hd);
        }
        continue;
      }
      double top = 0.0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const double m = __builtin_fabs(x[e]);
        // (a NaN counts as infinite: the row is then not finite)
        top = m <= top ? top : (m == m ? m : __builtin_inf());
      }
      top = over_lanes<T>(mine ? top : 0.0, [](double u, double v) {
        return __builtin_fmax(u, v);
      });
      const float scale = top < __builtin_inf() ? (float)(top / 127.0)
                                                : __builtin_nanf("");
      const float inv = __builtin_amdgcn_rcpf(scale);
      uint32_t code[8];
#pragma unroll
      for (int e = 0; e < 8; ++e)
        code[e] = (uint32_t)code_of((float)x[e], x[e], scale, inv) & 255;
      if (!ok[r]) continue;
      if (lane == 0)
        *reinterpret_cast<float *>(block + (size_t)a.n_kv * a.bs * hd +
                                   row_at * 4) = scale;
      if (!is_v) {
        if (mine)
          *reinterpret_cast<uint2 *>(block + row_at * hd + d0) = uint2{
              code[0] | code[1] << 8 | code[2] << 16 | code[3] << 24,
              code[4] | code[5] << 8 | code[6] << 16 | code[7] << 24};
        continue;
      }
      if (run) {
#pragma unroll
        for (int e = 0; e < 8; ++e) vcode[e] |= code[e] << (8 * (r & 3));
      } else if (mine) {
        unsigned char *v = block + ((size_t)hh * hd + d0) * a.bs + off[r];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[(size_t)e * a.bs] = (unsigned char)code[e];
      }
    }
    if (CELL == kQ8 && run && is_v && mine) {
      unsigned char *v =
          a.vc + blk[0] * a.rec + ((size_t)hh * hd + d0) * a.bs + off[0];
#pragma unroll
      for (int e = 0; e < 8; ++e)  // (any alignment)
        __builtin_memcpy(v + (size_t)e * a.bs, &vcode[e], 4);
    }
  }
}

// The plain form, for any rot, stride and alignment: one token a workgroup,
// 16 lanes a head, lane l owning dims l, l + 16, ...
template <typename In, int CELL>
__global__ void __launch_bounds__(256) rope_append_any_kernel(RopeArgs a) {
  __shared__ double cs[128], sn[128];
  const uint32_t row = blockIdx.x, hd = a.hd, half = a.rot / 2;
  for (uint32_t p = threadIdx.x; p < half; p += 256) {
    double s, c;
    sincos64((double)a.positions[row] * (double)a.inv_freq[p], s, c);
    cs[p] = c * (double)a.factor;
    sn[p] = s * (double)a.factor;
  }
  __syncthreads();
  const uint32_t blk = a.slot_block[row], off = a.slot_off[row];
  const bool ok = blk < a.num_blocks && off < a.bs;
  const uint32_t lane = threadIdx.x % 16;
  const uint32_t n_slots = a.n_heads + 2 * a.n_kv;
  for (uint32_t slot = threadIdx.x / 16; slot < n_slots; slot += 16) {
    const bool is_q = slot < a.n_heads;
    const bool is_v = slot >= a.n_heads + a.n_kv;
    const uint32_t hh = is_q ? slot
                             : (is_v ? slot - a.n_heads - a.n_kv
                                     : slot - a.n_heads);
    if (!is_q && !ok) continue;
    const In *src = is_q ? (const In *)a.q + row * a.q_stride
                         : (is_v ? (const In *)a.v + row * a.v_stride
                                 : (const In *)a.k + row * a.k_stride);
    src += (size_t)hh * hd;
    const float *w = is_v ? nullptr : (is_q ? a.q_norm : a.k_norm);
    double norm = 1.0;
    if (w) {
      double ss = 0.0;
      for (uint32_t d = lane; d < hd; d += 16) {
        const double x = (double)src[d];
        ss = __builtin_fma(x, x, ss);
      }
      ss = over_lanes<16>(ss, [](double x, double y) { return x + y; });
      norm = rsqrt64(ss / (double)hd + (double)a.eps);
    }
    double x[16], top = 0.0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t d = lane + 16 * e;
      x[e] = 0.0;
      if (d >= hd) continue;
      x[e] = w ? (double)src[d] * norm * (double)w[d] : (double)src[d];
      if (!is_v && d < a.rot) {
        const bool is_a = a.interleaved ? !(d & 1) : d < half;
        const uint32_t p = a.interleaved ? d >> 1 : (is_a ? d : d - half);
        const uint32_t d1 = a.interleaved ? d ^ 1 : (is_a ? d + half : d - half);
        const double y = w ? (double)src[d1] * norm * (double)w[d1]
                           : (double)src[d1];
        x[e] = x[e] * cs[p] + y * (is_a ? -sn[p] : sn[p]);
      }
      const double m = __builtin_fabs(x[e]);
      top = m <= top ? top : (m == m ? m : __builtin_inf());
    }
    unsigned char *block = (is_v ? a.vc : a.kc) + (ok ? blk : 0) * a.rec;
    const size_t row_at = (size_t)hh * a.bs + off;
    const auto put = [&](auto *out) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (lane + 16 * e < hd) round_to(x[e], out[lane + 16 * e]);
    };
    if (is_q) {
      put((In *)a.q_out + ((size_t)row * a.n_heads + hh) * hd);
    } else if (CELL == kF16) {
      put((_Float16 *)block + row_at * hd);
    } else if (CELL == kF32) {
      put((float *)block + row_at * hd);
    } else {
      top = over_lanes<16>(top, [](double u, double v) {
        return __builtin_fmax(u, v);
      });
      const float scale = top < __builtin_inf() ? (float)(top / 127.0)
                                                : __builtin_nanf("");
      const double s = (double)scale, inv = 1.0 / s;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t d = lane + 16 * e;
        if (d < hd)
          block[is_v ? ((size_t)hh * hd + d) * a.bs + off : row_at * hd + d] =
              (unsigned char)(scale > 0.f ? quantise(x[e], s, inv) : 0);
      }
      if (lane == 0)
        *reinterpret_cast<float *>(block + (size_t)a.n_kv * a.bs * hd +
                                   row_at * 4) = scale;
    }
  }
}

// Four tokens a workgroup from 2048 on, where they fill the chip.
template <typename In, int CELL, int T>
void launch_wide(const RopeArgs &a, hipStream_t st) {
  if (a.rows >= 2048)
    hipLaunchKernelGGL((rope_append_kernel<In, CELL, T, 4>),
                       dim3((a.rows + 3) / 4), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((rope_append_kernel<In, CELL, T, 1>), dim3(a.rows),
                       dim3(256), 0, st, a);
}

template <typename In, int CELL>
void launch(const RopeArgs &a, bool wide, hipStream_t st) {
  if (!wide)
    hipLaunchKernelGGL((rope_append_any_kernel<In, CELL>), dim3(a.rows),
                       dim3(256), 0, st, a);
  else if (a.hd <= 64)
    launch_wide<In, CELL, 8>(a, st);
  else if (a.hd <= 128)
    launch_wide<In, CELL, 16>(a, st);
  else
    launch_wide<In, CELL, 32>(a, st);
}

// The checks that both pools' entry points share; fills a.
int rope_append(const char *op, int cell, int device, hipStream_t st,
                RopeArgs &a, rvkv_dtype dtype, uint32_t interleaved) {
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
  // (a head's partners are read while others are written)
  const auto apart = [&](const void *in, uint64_t stride, uint64_t width) {
    const uintptr_t x = (uintptr_t)in, y = (uintptr_t)a.q_out;
    return !in || !y || x + ((a.rows - 1) * stride + width) * eb <= y ||
           y + (uint64_t)a.rows * a.n_heads * a.hd * eb <= x;
  };
  if (!apart(a.q, a.q_stride, (uint64_t)a.n_heads * a.hd) ||
      !apart(a.k, a.k_stride, kv_row) || !apart(a.v, a.v_stride, kv_row))
    return fail(RVKV_EINVAL, op, "q_out overlaps q, k or v");
  const int rc = rvkv_detail::q8_device(op, device);
  if (rc) return rc;
  a.interleaved = interleaved;
  bool vec = a.hd % 8 == 0 &&
             (interleaved ? a.rot % 8 == 0 : a.rot % 16 == 0);
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
  return rope_append(op, pool->f32() ? kF32 : kF16, pool->device,
                     pool->stream, a, dtype, interleaved);
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
  return rope_append(op, kQ8, pool->device, pool->stream, a, dtype,
                     interleaved);
}

}  // extern "C"
