// q8.hip - the 8-bit paged cache's pool, its block copy and gather, and decode
// attention over it.
#include <new>
#include <type_traits>

#include "q8.h"

using rvkv_detail::fail;
using rvkv_detail::hip_fail;

namespace rvkv_detail {
int q8_device(const char *op, int device) {
  int cur = -1;
  const hipError_t e = hipGetDevice(&cur);
  if (e != hipSuccess) return hip_fail(op, e);
  if (cur != device)
    return fail(RVKV_EINVAL, op, "the current device is not the pool's");
  return RVKV_OK;
}
}  // namespace rvkv_detail

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// Bytes of the records of a pool; 0 when the shape is refused (reason set).
size_t q8_bytes(const char *op, uint32_t n_layers, uint32_t num_blocks,
                uint32_t block_size, uint32_t n_kv, uint32_t hd, size_t *rec) {
  if (n_layers == 0 || num_blocks == 0 || block_size == 0 || n_kv == 0 ||
      hd == 0) {
    fail(RVKV_EINVAL, op,
         "n_layers/num_blocks/block_size/n_kv_heads/head_dim must be positive");
    return 0;
  }
  if (hd % 16 || hd > 256) {
    fail(RVKV_EUNSUPPORTED, op,
         "head_dim must be a multiple of 16 and at most 256");
    return 0;
  }
  if (block_size % 16 || block_size > 4096 || n_kv > 4096) {
    fail(RVKV_EUNSUPPORTED, op,
         "block_size must be a multiple of 16; block_size and n_kv_heads at "
         "most 4096");
    return 0;
  }
  if ((uint64_t)n_kv * block_size * (hd + 4) >> 31) {
    fail(RVKV_EUNSUPPORTED, op, "a block's record must be below 2 GiB");
    return 0;
  }
  *rec = ((size_t)n_kv * block_size * (hd + 4) + 255) & ~(size_t)255;
  const unsigned __int128 all =
      (unsigned __int128)*rec * num_blocks * 2 * n_layers;
  if (all >> 48) {
    fail(RVKV_EINVAL, op, "the pool is too large");
    return 0;
  }
  return (size_t)all;
}

// ---------------------------------------------------------------------------
// Gather: the cells' values, [batch, n_kv, ctx_len, hd]. One thread 16 dims of
// a row; a block id out of range reads zeros.
// ---------------------------------------------------------------------------
template <typename Out>
__global__ void __launch_bounds__(256)
    q8_gather_kernel(const unsigned char *kc, const unsigned char *vc,
                     size_t rec, const uint32_t *tables, Out *out_k, Out *out_v,
                     uint64_t n, uint32_t max_blocks, uint32_t ctx_len,
                     uint32_t n_kv, uint32_t hd, uint32_t bs,
                     uint32_t num_blocks) {
  const uint32_t chunks = hd / 16;
  const uint64_t i = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const uint64_t row = i / chunks;
  const uint32_t d0 = (uint32_t)(i - row * chunks) * 16;
  const uint32_t tok = (uint32_t)(row % ctx_len);
  const uint64_t bh = row / ctx_len;
  const uint32_t head = (uint32_t)(bh % n_kv);
  const uint32_t blk = tables[bh / n_kv * max_blocks + tok / bs];
  const uint32_t off = tok % bs;
  const bool is_v = blockIdx.y;
  Out *out = (is_v ? out_v : out_k) + row * hd + d0;
  if (blk >= num_blocks) {
    for (int e = 0; e < 16; ++e) out[e] = (Out)0.f;
    return;
  }
  const unsigned char *block = (is_v ? vc : kc) + blk * rec;
  const float scale = *reinterpret_cast<const float *>(
      block + (size_t)n_kv * bs * hd + ((size_t)head * bs + off) * 4);
  const signed char *tile =
      reinterpret_cast<const signed char *>(block) + (size_t)head * bs * hd;
  for (int e = 0; e < 16; ++e)
    out[e] = (Out)((float)(is_v ? tile[(size_t)(d0 + e) * bs + off]
                                : tile[(size_t)off * hd + d0 + e]) *
                   scale);
}

__global__ void __launch_bounds__(256)
    q8_copy_kernel(unsigned char *base, size_t tensor_bytes, size_t rec,
                   const uint32_t *src, const uint32_t *dst,
                   uint32_t num_blocks) {
  const uint32_t s = src[blockIdx.y], d = dst[blockIdx.y];
  if (s >= num_blocks || d >= num_blocks) return;
  unsigned char *t = base + (size_t)blockIdx.z * tensor_bytes;
  const uint4 *from = reinterpret_cast<const uint4 *>(t + s * rec);
  uint4 *to = reinterpret_cast<uint4 *>(t + d * rec);
  for (size_t w = (size_t)blockIdx.x * 256 + threadIdx.x; w < rec / 16;
       w += (size_t)gridDim.x * 256)
    to[w] = from[w];
}

// ---------------------------------------------------------------------------
// Decode attention.
//
//   s_j = scale ks_j (q . kcode_j),   out = sum_j p_j vs_j vcode_j / sum_j p_j,
//   p_j = exp(s_j - max s), all keys j < ctx (and >= ctx - window).
//
// S = K q' on v_mfma_i32_16x16x64_i8: the codes as they lie in the cache, q as
// a 24-bit fixed-point number relative to its head's largest value, in three
// signed digits of base 256, each an operand of its own; integer sums are
// exact. O = V' P on v_mfma_f32_16x16x32_f16: codes are exact in f16, the
// weights two f16 parts. The 16 matrix rows are keys, or dims; the 16 columns
// are the heads of a KV group, up to 8, twice: columns 0-7 the upper digit or
// part, 8-15 the middle digit or lower part (the lowest digit takes a second
// product). So an f32-accurate result costs no conversion of K and no product
// more than a rounded one. Larger groups take n_sub workgroups.
//
// A wave takes 64 keys at a time; a workgroup's four waves take turns, or a
// wave has a partition of its own (see cut). Row 4g + i of S tile t is key
// 16g + 4t + i, so lane group g of the result holds keys 16g .. 16g+15: the
// order in which the V' P product takes its weights from the same registers,
// and 16 keys of one dim are 16 bytes of a
// V record. No operand passes through LDS, only the scales do.
//
// Bound by the reads of the cache at two waves a SIMD (199 registers at hd 128;
// three would spill, 1.9 times slower): 256 x 4096 tokens of 8 heads of 128,
// 2.2 GB, in 380 us, 5.8 TB/s; with f16 conversions of K 475 us. Contexts of 32
// to 8192 tokens and small launches are bound by each wave's start, ~5 us of
// dependent reads: length, table, cells.
// ---------------------------------------------------------------------------
struct DecodeArgs {
  const void *q;
  void *out;
  const unsigned char *kc, *vc;
  const uint32_t *tables, *ctx_lens;
  float *ws_acc, *ws_ml;
  size_t rec;
  uint32_t n_heads, n_kv, group, n_sub, hd, bs, max_blocks, num_blocks;
  uint32_t ctx_cap, part_tokens, n_parts, batch;
  float qscale;  // scale * log2(e)
  uint32_t window;
};

// A sequence's visible keys [lo, ctx); its partitions start at base, lo
// rounded down to whole records' granules of 16 keys.
struct Range {
  uint32_t ctx, lo, base;
};
__device__ __forceinline__ Range visible(const DecodeArgs &a, uint32_t b) {
  Range r;
  r.ctx = a.ctx_lens[b];
  if (r.ctx > a.ctx_cap) r.ctx = a.ctx_cap;
  r.lo = a.window && r.ctx > a.window ? r.ctx - a.window : 0;
  r.base = r.lo & ~15u;
  return r;
}

__device__ __forceinline__ float ror8(float x) {
  return __uint_as_float(__builtin_amdgcn_mov_dpp(__float_as_uint(x), 0x128,
                                                  0xf, 0xf, true));
}
// The largest of the four lanes of a column.
__device__ __forceinline__ float max_groups(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                                  __float_as_uint(x), false,
                                                  false);
  x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  const auto t = __builtin_amdgcn_permlane16_swap(__float_as_uint(x),
                                                  __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(t[0]), __uint_as_float(t[1]));
}
// The largest of a wave.
__device__ __forceinline__ float max_wave(float x) {
  const auto dpp = [](float v, auto ctrl) {
    return __uint_as_float(__builtin_amdgcn_mov_dpp(
        __float_as_uint(v), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x121>()));  // row_ror 1
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x122>()));  // 2
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x124>()));  // 4
  x = fmaxf(x, dpp(x, std::integral_constant<int, 0x128>()));  // 8
  return max_groups(x);
}
__device__ __forceinline__ half2v pk(float a, float b) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(a, b));
}
__device__ __forceinline__ int4v load_nt(const unsigned char *p) {
  return __builtin_nontemporal_load(reinterpret_cast<const int4v *>(p));
}

template <typename T, int HD, int W>
__global__ void __launch_bounds__(64 * W, HD == 256 ? 1 : 2)
    q8_decode_kernel(DecodeArgs a) {
  constexpr int NK = HD / 64, NV = HD / 16;
  constexpr float kNone = -__builtin_inff();
  __shared__ float sh_acc[W][8][HD];
  __shared__ float sh_m[W][8], sh_l[W][8];
  // A tile's scales, from one key a lane to the 16 of a lane group.
  __shared__ __align__(16) float sh_ks[W][64], sh_vs[W][64];
  // Workgroups: partitions outermost, so that those behind most sequences'
  // ends do not share an XCD (workgroup id mod 8); the n_sub workgroups of a
  // head, which read the same keys, eight apart, so that they do.
  uint32_t unit, sub = 0;
  if (a.n_sub == 1) {
    unit = blockIdx.x;
  } else {
    const uint32_t eight = blockIdx.x / (8 * a.n_sub);
    const uint32_t in = blockIdx.x - eight * 8 * a.n_sub;
    sub = in / 8;
    unit = eight * 8 + in % 8;
  }
  const uint32_t kvh = unit % a.n_kv, pb = unit / a.n_kv;
  const uint32_t part = pb / a.batch, b = pb - part * a.batch;
  if (part >= a.n_parts) return;  // (the last eight units may not be whole)
  const Range rg = visible(a, b);
  const uint64_t start64 = (uint64_t)rg.base + (uint64_t)part * a.part_tokens;
  if (a.n_parts > 1 && start64 >= rg.ctx) return;
  const uint32_t start = (uint32_t)start64;
  const uint32_t end = rg.ctx - start < a.part_tokens ? rg.ctx
                                                      : start + a.part_tokens;
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const uint32_t col = lane & 15, g = lane >> 4;
  const uint32_t h_in = sub * 8 + (col & 7);
  const bool has_head = h_in < a.group;
  const uint32_t head = kvh * a.group + (has_head ? h_in : 0);
  const uint32_t hd = a.hd, bs = a.bs, bsg = bs / 16;

  const uint32_t n_tiles = end > start ? (end - start + 63) / 64 : 0;
  const uint32_t last_granule = rg.ctx ? (rg.ctx - 1) / 16 : 0;
  const uint32_t *table = a.tables + (size_t)b * a.max_blocks;
  // Block id and granule within the block of key granule gr (clamped to the
  // sequence's last: keys behind it are masked).
  struct Place {
    uint32_t blk, in;
  };
  const auto place = [&](uint32_t tile, uint32_t gr) {
    uint32_t x = (start + tile * 64) / 16 + gr;
    x = x < last_granule ? x : last_granule;
    Place p;
    const uint32_t bi = bsg == 1 ? x : x / bsg;
    p.in = x - bi * bsg;
    p.blk = table[bi];
    return p;
  };
  int4v kr[4 * NK], vr[NV];
  float ks1, vs1;     // of key lane of the tile
  bool seen = false;  // this lane group's keys lie in a readable block
  const uint32_t gk = col >> 2;
  const uint32_t k_at = kvh * bs * hd + (col & 3) * hd + g * 16;
  const uint32_t v_at = kvh * bs * hd + col * bs;
  const uint32_t s_at = a.n_kv * hd * bs + kvh * bs * 4;
  const auto load_k = [&](Place p) {
    const uint32_t blk = p.blk < a.num_blocks ? p.blk : 0;
    const unsigned char *kp = a.kc + blk * a.rec + (k_at + p.in * 16 * hd);
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int c = 0; c < NK; ++c)
        kr[t * NK + c] = load_nt(
            kp + t * 4 * hd + ((uint32_t)c * 64 + g * 16 < hd ? c * 64 : 0));
  };
  const auto load_scales = [&](Place p) {
    seen = p.blk < a.num_blocks;
    const size_t at = (seen ? p.blk : 0) * a.rec + (s_at + p.in * 64 + col * 4);
    ks1 = *reinterpret_cast<const float *>(a.kc + at);
    vs1 = *reinterpret_cast<const float *>(a.vc + at);
  };
  const auto load_v = [&](Place p) {
    const uint32_t blk = p.blk < a.num_blocks ? p.blk : 0;
    const unsigned char *vp = a.vc + blk * a.rec + (v_at + p.in * 16);
#pragma unroll
    for (int d = 0; d < NV; ++d)  // (rows from hd on: any codes, not stored)
      vr[d] = load_nt(vp + ((uint32_t)d * 16 < hd ? d * 16 * bs : 0));
  };

  float m = kNone, l = 0.f;
  // Weights are held as 2^shift p, l with them: times vs, they stay below 2^15,
  // and their lower parts in f16's normal numbers.
  int shift = 95;
  float4v acc[NV];
#pragma unroll
  for (int d = 0; d < NV; ++d) acc[d] = float4v{0.f, 0.f, 0.f, 0.f};
  const float lower = col >= 8 ? 1.f : 0.f;

  if (wave < n_tiles) {
    Place pk0 = place(wave, gk), pv0 = place(wave, g);
    Place pk1 = place(wave + W, gk), pv1 = place(wave + W, g);
    load_k(pk0);
    load_scales(pv0);
    load_v(pv0);

    // q's digits: byte e of chunk c is dim 64 c + 16 g + e of this column's
    // head. A digit is in -128 .. 127, so q's largest value is brought below
    // 127/128 of 2^23.
    int4v qd[NK], q0[NK];
    // qscale: |scale| log2(e) / q's power of two; the sign goes with q.
    float qscale = fmaxf(fabsf(a.qscale), 0x1p-100f);
    {
      const T *q = (const T *)a.q + ((size_t)b * a.n_heads + head) * hd;
      float x[NK][16];
      float top = 0.f;
      bool finite = true;
#pragma unroll
      for (int c = 0; c < NK; ++c)
#pragma unroll
        for (int e = 0; e < 16; e += 16 / (int)sizeof(T)) {
          const uint32_t d = 64 * c + 16 * g + e;
          alignas(16) T y[16 / sizeof(T)];
          *reinterpret_cast<uint4 *>(y) = uint4{};
          if (has_head && 64 * c + 16 * g < hd)
            *reinterpret_cast<uint4 *>(y) =
                *reinterpret_cast<const uint4 *>(q + d);
#pragma unroll
          for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
            x[c][e + i] = (float)y[i];
            const float mag = fabsf(x[c][e + i]);
            finite = finite && mag < __builtin_inff();
            top = fmaxf(top, mag);
          }
        }
      top = max_groups(top);
      uint32_t ex = scale_exponent(top);  // top < 2^(ex - 127)
      ex = ex < 64 ? 64 : ex;
      float up = __uint_as_float((277 - ex) << 23) * (127.f / 128.f);
      if (a.qscale < 0.f) up = -up;
      qscale *= __uint_as_float((ex - 23) << 23) * (128.f / 127.f);
      // (a head whose q is not finite: every score, and so its row, is NaN)
      if (max_groups(finite ? 0.f : 1.f) > 0.f) qscale = __builtin_nanf("");
#pragma unroll
      for (int c = 0; c < NK; ++c)
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t mine = 0, low = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int v = (int)__builtin_rintf(x[c][4 * w + i] * up);
            const int d0 = (int)(signed char)v, v1 = (v - d0) >> 8;
            const int d1 = (int)(signed char)v1, d2 = (v1 - d1) >> 8;
            mine |= (uint32_t)((col < 8 ? d2 : d1) & 255) << (8 * i);
            low |= (uint32_t)((col < 8 ? d0 : 0) & 255) << (8 * i);
          }
          qd[c][w] = (int)mine;
          q0[c][w] = (int)low;
        }
    }
    const float digit = col < 8 ? 65536.f : 256.f;

    for (uint32_t tile = wave; tile < n_tiles; tile += W) {
      const bool more = tile + W < n_tiles;
      const uint32_t first = start + tile * 64;
      const bool masked = first < rg.lo || first + 64 > end || !__all(seen);
      bool ok = true;
      if (masked) {
        const uint32_t key = first + lane;
        ok = seen && key >= rg.lo && key < end;
        if (!ok) ks1 = vs1 = 0.f;
      }
      const uint64_t keep = __ballot(ok) >> (16 * g);
      sh_ks[wave][lane] = ks1;
      sh_vs[wave][lane] = vs1;
      __builtin_amdgcn_wave_barrier();
      float vtop = vs1;
      float s[16];
      float top = kNone;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        int4v st = {0, 0, 0, 0}, s0 = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < NK; ++c) {
          st = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[t * NK + c], qd[c], st,
                                                     0, 0, 0);
          s0 = __builtin_amdgcn_mfma_i32_16x16x64_i8(kr[t * NK + c], q0[c], s0,
                                                     0, 0, 0);
        }
        const float4v ks = *reinterpret_cast<const float4v *>(
            &sh_ks[wave][16 * g + 4 * t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = __builtin_fmaf((float)st[i], digit, (float)s0[i]);
          s[4 * t + i] = (x + ror8(x)) * ks[i];
        }
      }
      if (more) load_k(pk1);
      if (masked) {
        // (a branch, no selects on every tile)
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < 16; ++j) s[j] = keep >> j & 1 ? s[j] : kNone;
      }
#pragma unroll
      for (int j = 0; j < 16; j += 2) top = fmaxf(fmaxf(s[j], s[j + 1]), top);
      top *= qscale;
      top = max_groups(top);
      vtop = max_wave(vtop);
      if (__any(top > m) || vtop >= __uint_as_float((uint32_t)(142 - shift)
                                                    << 23)) {
        __builtin_amdgcn_sched_barrier(0);
        const float now = fmaxf(m, top);
        float fix = m == now ? 1.f : __builtin_amdgcn_exp2f(m - now);
        m = now;
        // vs < 2^(15 - shift)
        const int e = (int)(__float_as_uint(vtop) >> 23) - 126;
        const int to = 15 - e < shift ? 15 - e : shift;
        fix = __builtin_amdgcn_ldexpf(fix, to - shift);
        shift = to;
        l *= fix;
#pragma unroll
        for (int d = 0; d < NV; ++d) acc[d] *= fix;
      }
      const float mm = (m == kNone ? 0.f : m) - (float)shift;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const float4v vs = *reinterpret_cast<const float4v *>(
            &sh_vs[wave][16 * g + 4 * t]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float p = __builtin_amdgcn_exp2f(
              __builtin_fmaf(s[4 * t + i], qscale, -mm));
          l += p;
          s[4 * t + i] = p * vs[i];
        }
      }
      __builtin_amdgcn_wave_barrier();
      if (more) load_scales(pv1);
      half8v pf[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const float w0 = s[8 * u + j], w1 = s[8 * u + j + 1];
          const half2v up = pk(w0, w1);
          const half2v x = pk(__builtin_fmaf(-lower, (float)up[0], w0),
                              __builtin_fmaf(-lower, (float)up[1], w1));
          pf[u][j] = x[0];
          pf[u][j + 1] = x[1];
        }
#pragma unroll
      for (int d = 0; d < NV; ++d) {
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            codes_to_half8(vr[d][0], vr[d][1]), pf[0], acc[d], 0, 0, 0);
        acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
            codes_to_half8(vr[d][2], vr[d][3]), pf[1], acc[d], 0, 0, 0);
      }
      if (more) {
        load_v(pv1);
        pk1 = place(tile + 2 * W, gk);
        pv1 = place(tile + 2 * W, g);
      }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
  }

  // Merge the waves: a head's weights relative to the largest maximum.
  const float back = __builtin_amdgcn_ldexpf(1.f, -shift);
  if (lane < 8) {
    sh_m[wave][lane] = m;
    sh_l[wave][lane] = l * back;
  }
#pragma unroll
  for (int d = 0; d < NV; ++d) {
    float4v o = acc[d];
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = (o[i] + ror8(o[i])) * back;
    if (col < 8)
      *reinterpret_cast<float4v *>(&sh_acc[wave][col][d * 16 + 4 * g]) = o;
  }
  __syncthreads();
  for (uint32_t x = threadIdx.x; x < 8 * HD; x += 64 * W) {
    const uint32_t h = x / HD, d = x % HD;
    if (sub * 8 + h >= a.group || d >= hd) continue;
    float top = sh_m[0][h];
#pragma unroll
    for (int w = 1; w < W; ++w) top = fmaxf(top, sh_m[w][h]);
    float o = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = sh_m[w][h] == kNone
                          ? 0.f : __builtin_amdgcn_exp2f(sh_m[w][h] - top);
      o += sh_acc[w][h][d] * f;
      sum += sh_l[w][h] * f;
    }
    const size_t row = (size_t)b * a.n_heads + kvh * a.group + sub * 8 + h;
    if (a.n_parts == 1) {
      ((T *)a.out)[row * hd + d] = (T)(sum == 0.f ? 0.f : o / sum);
    } else {
      const size_t slot = row * a.n_parts + part;
      a.ws_acc[slot * HD + d] = o;
      if (d == 0) {
        a.ws_ml[slot * 2] = top;
        a.ws_ml[slot * 2 + 1] = sum;
      }
    }
  }
}

// Merges a head's partitions: every partition's weight into LDS, then
// 1024 / HD partitions at a time, four dims a thread.
template <typename T, int HD>
__global__ void __launch_bounds__(256) q8_reduce_kernel(DecodeArgs a) {
  constexpr uint32_t D4 = HD / 4, P = 256 / D4;
  constexpr float kNone = -__builtin_inff();
  __shared__ float weight[256], sh_top[4], sh_sum[4];
  __shared__ __align__(16) float sh_o[P][HD];
  const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const Range rg = visible(a, b);
  const uint32_t live =
      rg.ctx > rg.base
          ? (rg.ctx - rg.base + a.part_tokens - 1) / a.part_tokens : 0;
  const size_t row = (size_t)b * a.n_heads + h;
  const float2 *ml =
      reinterpret_cast<const float2 *>(a.ws_ml) + row * a.n_parts;
  const float *acc = a.ws_acc + row * a.n_parts * HD;
  const uint32_t d = tid % D4 * 4, w = tid / D4;
  // The largest maximum (most calls have at most 256 partitions: one load).
  float2 mine = {kNone, 0.f};
  float top = kNone;
  for (uint32_t p = tid; p < live; p += 256) {
    mine = ml[p];
    top = fmaxf(top, mine.x);
  }
  top = max_wave(top);
  if ((tid & 63) == 0) sh_top[tid >> 6] = top;
  __syncthreads();
  top = fmaxf(fmaxf(sh_top[0], sh_top[1]), fmaxf(sh_top[2], sh_top[3]));
  float4v o = {0.f, 0.f, 0.f, 0.f};
  float sum = 0.f;
  for (uint32_t p0 = 0; p0 < live; p0 += 256) {
    const uint32_t n = live - p0 < 256 ? live - p0 : 256;
    if (live > 256) mine = tid < n ? ml[p0 + tid] : float2{kNone, 0.f};
    const float f =
        mine.x == kNone ? 0.f : __builtin_amdgcn_exp2f(mine.x - top);
    sum += mine.y * f;
    weight[tid] = f;
    __syncthreads();
#pragma unroll 4
    for (uint32_t p = w; p < n; p += P)
      o += *reinterpret_cast<const float4v *>(acc + (size_t)(p0 + p) * HD + d) *
           weight[p];
    __syncthreads();
  }
#pragma unroll
  for (int i = 32; i >= 1; i >>= 1) sum += __shfl_xor(sum, i);
  if ((tid & 63) == 0) sh_sum[tid >> 6] = sum;
  *reinterpret_cast<float4v *>(&sh_o[w][d]) = o;
  __syncthreads();
  sum = sh_sum[0] + sh_sum[1] + sh_sum[2] + sh_sum[3];
  if (tid < a.hd) {
    float x = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < P; ++i) x += sh_o[i][tid];
    ((T *)a.out)[row * a.hd + tid] = (T)(sum == 0.f ? 0.f : x / sum);
  }
}

// Workgroups of a decode launch.
uint64_t decode_groups(uint64_t n_parts, uint32_t batch, uint32_t n_kv,
                       uint32_t n_sub) {
  const uint64_t units = n_parts * batch * n_kv;
  return n_sub == 1 ? units : (units + 7) / 8 * 8 * n_sub;
}

uint32_t hd_up(uint32_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

// How a launch is cut. waves 4: a workgroup's waves take a partition's tiles
// in turn; partitions of 256 to 2048 keys, so that up to 512 workgroups (two
// a CU) share the keys (2 x 32749 keys of 8 heads: 1024-key partitions 31 us,
// 512 36, 256 43; 64 x 2048: 2048 34 us, 1024 39). waves 1: launches with
// 1024-key partitions for 4096 waves or more, where single waves balance
// ragged contexts better and need no merge in the workgroup (300 contexts up
// to 8192 of 8 heads: 190 us; four waves 218, at 2048 keys 206; 256 x 4096
// 370, four waves 415 and 377).
struct Cut {
  uint32_t part_tokens, waves;
};
Cut cut(const rvkv_q8_pool *p, uint32_t batch, uint32_t n_heads,
        uint32_t keys) {
  const uint32_t n_sub = (n_heads / p->n_kv + 7) / 8;
  const uint64_t rows = (uint64_t)batch * p->n_kv * n_sub;
  if (rows * (((uint64_t)keys + 1023) / 1024) >= 4096) return {1024, 1};
  const uint64_t want = ((uint64_t)keys * rows + 511) / 512;
  const uint64_t t = (want + 255) / 256 * 256;
  return {(uint32_t)(t < 256 ? 256 : t > 2048 ? 2048 : t), 4};
}

struct Layout {
  uint32_t part_tokens, n_parts, waves;
  size_t ml_off, bytes;
};
// window 0: none. A window's first partition starts up to 15 keys before it.
Layout layout(const rvkv_q8_pool *p, uint32_t batch, uint32_t n_heads,
              uint32_t max_ctx, uint32_t window) {
  Layout w{};
  uint64_t keys = max_ctx ? max_ctx : 1;
  if (window && (uint64_t)window + 15 < keys) keys = (uint64_t)window + 15;
  const Cut c = cut(p, batch, n_heads, (uint32_t)keys);
  w.part_tokens = c.part_tokens;
  w.waves = c.waves;
  w.n_parts = (uint32_t)((keys + w.part_tokens - 1) / w.part_tokens);
  if (w.n_parts <= 1) return w;
  const size_t slots = (size_t)batch * n_heads * w.n_parts;
  w.ml_off = slots * hd_up(p->head_dim) * 4;
  w.bytes = (w.ml_off + slots * 8 + 255) & ~(size_t)255;
  return w;
}

template <typename T, int HD>
int launch_decode(const char *op, const DecodeArgs &a, uint32_t batch,
                  uint32_t waves, hipStream_t st) {
  const dim3 grid((uint32_t)decode_groups(a.n_parts, batch, a.n_kv, a.n_sub));
  if (waves == 4)
    hipLaunchKernelGGL((q8_decode_kernel<T, HD, 4>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((q8_decode_kernel<T, HD, 1>), grid, dim3(64), 0, st, a);
  if (a.n_parts > 1)
    hipLaunchKernelGGL((q8_reduce_kernel<T, HD>), dim3(a.n_heads, batch),
                       dim3(256), 0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RVKV_OK : hip_fail(op, e);
}

template <typename T>
int launch_decode(const char *op, const DecodeArgs &a, uint32_t batch,
                  uint32_t waves, hipStream_t st) {
  switch (hd_up(a.hd)) {
    case 64: return launch_decode<T, 64>(op, a, batch, waves, st);
    case 128: return launch_decode<T, 128>(op, a, batch, waves, st);
    default: return launch_decode<T, 256>(op, a, batch, waves, st);
  }
}

}  // namespace

extern "C" {

size_t rvkv_q8_pool_bytes(uint32_t n_layers, uint32_t num_blocks,
                          uint32_t block_size, uint32_t n_kv_heads,
                          uint32_t head_dim) {
  size_t rec;
  return q8_bytes("q8_pool_bytes", n_layers, num_blocks, block_size,
                  n_kv_heads, head_dim, &rec);
}

int rvkv_q8_pool_create(uint32_t n_layers, uint32_t num_blocks,
                        uint32_t block_size, uint32_t n_kv_heads,
                        uint32_t head_dim, void *memory, size_t memory_bytes,
                        rvkv_stream stream, rvkv_q8_pool **out) {
  const char *op = "q8_pool_create";
  if (!out) return fail(RVKV_EINVAL, op, "out is NULL");
  *out = nullptr;
  size_t rec = 0;
  const size_t bytes = q8_bytes(op, n_layers, num_blocks, block_size,
                                n_kv_heads, head_dim, &rec);
  if (!bytes)
    return head_dim % 16 || head_dim > 256 || block_size % 16 ||
                   block_size > 4096 || n_kv_heads > 4096 ||
                   (uint64_t)n_kv_heads * block_size * (head_dim + 4) >> 31
               ? RVKV_EUNSUPPORTED : RVKV_EINVAL;
  if (memory && memory_bytes < bytes)
    return fail(RVKV_EINVAL, op, "memory smaller than the required bytes");
  if ((uintptr_t)memory % 256)
    return fail(RVKV_EINVAL, op, "memory must be 256-byte aligned");
  int device = -1;
  hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) {
    (void)hipGetLastError();
    // (the caller's memory needs no device yet; every launch asks again)
    if (!memory) return hip_fail(op, e);
    device = -1;
  } else if (memory) {
    hipPointerAttribute_t at{};
    e = hipPointerGetAttributes(&at, memory);
    if (e != hipSuccess) (void)hipGetLastError();
    if (e != hipSuccess || at.type != hipMemoryTypeDevice ||
        at.device != device)
      return fail(RVKV_EINVAL, op, "memory is not the current device's");
  }
  rvkv_q8_pool *p = new (std::nothrow) rvkv_q8_pool();
  if (!p) return fail(RVKV_ENOMEM, op, "out of host memory");
  p->n_layers = n_layers;
  p->num_blocks = num_blocks;
  p->block_size = block_size;
  p->n_kv = n_kv_heads;
  p->head_dim = head_dim;
  p->rec = rec;
  p->tensor_bytes = rec * num_blocks;
  p->stream = static_cast<hipStream_t>(stream);
  p->device = device;
  p->base = static_cast<unsigned char *>(memory);
  if (!memory) {
    e = hipMalloc(&p->base, bytes);
    if (e != hipSuccess) {
      (void)hipGetLastError();
      delete p;
      return fail(RVKV_ENOMEM, op, "hipMalloc of the pool failed");
    }
    p->owned = true;
    e = hipMemsetAsync(p->base, 0, bytes, p->stream);
    if (e != hipSuccess) {
      (void)hipFree(p->base);
      delete p;
      return hip_fail(op, e);
    }
  }
  *out = p;
  return RVKV_OK;
}

void rvkv_q8_pool_destroy(rvkv_q8_pool *pool) {
  if (!pool) return;
  if (pool->owned) {
    (void)hipStreamSynchronize(pool->stream);
    (void)hipFree(pool->base);
  }
  delete pool;
}

int rvkv_q8_pool_set_stream(rvkv_q8_pool *pool, rvkv_stream stream) {
  if (!pool) return fail(RVKV_EINVAL, "q8_pool_set_stream", "pool is NULL");
  pool->stream = static_cast<hipStream_t>(stream);
  return RVKV_OK;
}

int rvkv_q8_gather(const rvkv_q8_pool *pool, uint32_t layer,
                   const uint32_t *block_idx, uint32_t batch,
                   uint32_t max_blocks, uint32_t ctx_len, void *out_k,
                   void *out_v, rvkv_dtype out_dtype) {
  const char *op = "kv_gather";
  if (!pool) return fail(RVKV_EINVAL, op, "pool is NULL");
  if (layer >= pool->n_layers)
    return fail(RVKV_EINVAL, op, "layer out of range");
  if (batch == 0 || max_blocks == 0 || ctx_len == 0)
    return fail(RVKV_EINVAL, op,
                "batch/max_blocks/ctx_len/block_size/n_kv_heads/head_dim must "
                "be positive");
  if ((uint64_t)ctx_len > (uint64_t)max_blocks * pool->block_size)
    return fail(RVKV_EINVAL, op,
                "ctx_len must not exceed max_blocks * block_size");
  if (!block_idx || !out_k || !out_v)
    return fail(RVKV_EINVAL, op, "NULL block_idx/out_k/out_v");
  if (out_dtype != RVKV_F16 && out_dtype != RVKV_F32)
    return fail(RVKV_EINVAL, op, "out dtype must be F16 or F32");
  const uint64_t n = (uint64_t)batch * pool->n_kv * ctx_len *
                     (pool->head_dim / 16);
  if ((n + 255) / 256 > 0xffffffull)
    return fail(RVKV_EUNSUPPORTED, op, "too many rows for one launch");
  const int rc = rvkv_detail::q8_device(op, pool->device);
  if (rc) return rc;
  const dim3 grid((uint32_t)((n + 255) / 256), 2);
  if (out_dtype == RVKV_F16)
    hipLaunchKernelGGL(q8_gather_kernel<_Float16>, grid, dim3(256), 0,
                       pool->stream, pool->tensor(layer, 0),
                       pool->tensor(layer, 1), pool->rec, block_idx,
                       (_Float16 *)out_k, (_Float16 *)out_v, n, max_blocks,
                       ctx_len, pool->n_kv, pool->head_dim, pool->block_size,
                       pool->num_blocks);
  else
    hipLaunchKernelGGL(q8_gather_kernel<float>, grid, dim3(256), 0,
                       pool->stream, pool->tensor(layer, 0),
                       pool->tensor(layer, 1), pool->rec, block_idx,
                       (float *)out_k, (float *)out_v, n, max_blocks, ctx_len,
                       pool->n_kv, pool->head_dim, pool->block_size,
                       pool->num_blocks);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RVKV_OK : hip_fail(op, e);
}

int rvkv_q8_copy_blocks(rvkv_q8_pool *pool, const uint32_t *src,
                        const uint32_t *dst, uint32_t n) {
  const char *op = "copy_blocks";
  if (!pool) return fail(RVKV_EINVAL, op, "pool is NULL");
  if (n == 0) return RVKV_OK;
  if (!src || !dst) return fail(RVKV_EINVAL, op, "NULL src/dst");
  if (n > 65535)
    return fail(RVKV_EUNSUPPORTED, op, "at most 65535 pairs per call");
  if (pool->n_layers > 32767)
    return fail(RVKV_EUNSUPPORTED, op, "too many layers");
  const int rc = rvkv_detail::q8_device(op, pool->device);
  if (rc) return rc;
  size_t gx = (pool->rec / 16 + 255) / 256;
  if (gx > 64) gx = 64;
  hipLaunchKernelGGL(q8_copy_kernel, dim3((uint32_t)gx, n, 2 * pool->n_layers),
                     dim3(256), 0, pool->stream, pool->base,
                     pool->tensor_bytes, pool->rec, src, dst,
                     pool->num_blocks);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RVKV_OK : hip_fail(op, e);
}

size_t rvkv_q8_decode_workspace_bytes(const rvkv_q8_pool *pool, uint32_t batch,
                                      uint32_t n_heads, uint32_t max_ctx_len,
                                      int32_t window) {
  if (!pool || batch == 0 || n_heads == 0 || n_heads % pool->n_kv) return 0;
  return layout(pool, batch, n_heads, max_ctx_len,
                window > 0 ? (uint32_t)window : 0).bytes;
}

int rvkv_q8_paged_decode(const rvkv_q8_pool *pool, uint32_t layer,
                         const void *q, rvkv_dtype dtype,
                         const uint32_t *block_tables,
                         const uint32_t *ctx_lens, uint32_t batch,
                         uint32_t max_blocks, uint32_t n_heads,
                         uint32_t max_ctx_len, float scale, int32_t window,
                         void *out, void *ws, size_t ws_bytes) {
  const char *op = "paged_decode";
  if (!pool) return fail(RVKV_EINVAL, op, "pool is NULL");
  if (layer >= pool->n_layers)
    return fail(RVKV_EINVAL, op, "layer out of range");
  if (dtype != RVKV_F16 && dtype != RVKV_F32)
    return fail(RVKV_EINVAL, op, "dtype must be F16 or F32");
  if (batch == 0) return RVKV_OK;
  if (batch > 65535) return fail(RVKV_EUNSUPPORTED, op, "batch too large");
  if (max_blocks == 0)
    return fail(RVKV_EINVAL, op, "max_blocks must be positive");
  if (n_heads == 0 || n_heads % pool->n_kv != 0)
    return fail(RVKV_EINVAL, op,
                "n_heads must be a positive multiple of n_kv_heads");
  if (!q || !block_tables || !ctx_lens || !out)
    return fail(RVKV_EINVAL, op, "NULL q/block_tables/ctx_lens/out");
  if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
    return fail(RVKV_EINVAL, op, "q and out must be 16-byte aligned");
  const uint32_t group = n_heads / pool->n_kv, n_sub = (group + 7) / 8;
  if (n_heads > 65535)
    return fail(RVKV_EUNSUPPORTED, op, "head count too large");
  const uint64_t cap = (uint64_t)max_blocks * pool->block_size;
  if (max_ctx_len == 0) max_ctx_len = 1;
  if (max_ctx_len > rvkv_detail::kMaxKeys) max_ctx_len = rvkv_detail::kMaxKeys;
  const Layout w = layout(pool, batch, n_heads, max_ctx_len,
                          window > 0 ? (uint32_t)window : 0);
  // (a launch holds fewer than 2^32 threads)
  if (decode_groups(w.n_parts, batch, pool->n_kv, n_sub) > 0xffffffu)
    return fail(RVKV_EUNSUPPORTED, op, "too many partitions for one launch");
  if (w.bytes) {
    if (!ws) return fail(RVKV_EINVAL, op, "workspace is NULL");
    if (ws_bytes < w.bytes)
      return fail(RVKV_EINVAL, op, "workspace smaller than the required bytes");
    if ((uintptr_t)ws % 256)
      return fail(RVKV_EINVAL, op, "workspace must be 256-byte aligned");
  }
  const int rc = rvkv_detail::q8_device(op, pool->device);
  if (rc) return rc;
  DecodeArgs a{};
  a.q = q;
  a.out = out;
  a.kc = pool->tensor(layer, 0);
  a.vc = pool->tensor(layer, 1);
  a.tables = block_tables;
  a.ctx_lens = ctx_lens;
  a.ws_acc = static_cast<float *>(ws);
  a.ws_ml = reinterpret_cast<float *>(static_cast<char *>(ws) + w.ml_off);
  a.rec = pool->rec;
  a.n_heads = n_heads;
  a.n_kv = pool->n_kv;
  a.group = group;
  a.n_sub = n_sub;
  a.hd = pool->head_dim;
  a.bs = pool->block_size;
  a.max_blocks = max_blocks;
  a.num_blocks = pool->num_blocks;
  a.ctx_cap = (uint32_t)(cap < max_ctx_len ? cap : max_ctx_len);
  a.part_tokens = w.part_tokens;
  a.n_parts = w.n_parts;
  a.batch = batch;
  a.qscale = scale * kLog2e;
  a.window = window > 0 ? (uint32_t)window : 0;
  return dtype == RVKV_F16
             ? launch_decode<_Float16>(op, a, batch, w.waves, pool->stream)
             : launch_decode<float>(op, a, batch, w.waves, pool->stream);
}

}  // extern "C"
