// q8_prefill.hip - attention of packed prompts over the 8-bit paged cache.
//
// Rows row_start[b] .. row_start[b+1] of q are sequence b's; row i of them is
// at position pos_offset[b] + i and sees key j iff j < read_num[b], j <= its
// position, and, with a window, j + window > its position:
//   s_j = scale ks_j (q . kcode_j),   out = sum_j p_j vs_j vcode_j / sum_j p_j.
//
// A workgroup takes 128 rows of one (sequence, KV head): the rows of the
// group's heads token by token, so a tile of K and V serves the whole group
// and the causal bound stays near its rows. Four waves, 32 rows each, on
// v_mfma_f32_32x32x16_f16 with keys (S = K q') and dims (O = V' P) as the
// matrix rows and the q rows as its columns: a lane owns one q row, so the
// running maximum and sum need one exchange with lane ^ 32. K and V tiles of
// 64 keys are fetched as codes into registers while the tile before is
// computed, turned to f16 (exact) once a workgroup and kept in LDS, two
// buffers. K rows enter the S product in the order 16 (a >> 1) + 8 h +
// 4 (a & 1) + c of result row 8 a + 4 h + c, so that a lane's weights are the
// V' P operand as they stand.
//
// f16 rows take q as it is and round the weights p vs once to f16. f32 rows
// take q and the weights as two f16 parts each, twice the products.
#include "q8.h"

using rvkv_detail::fail;
using rvkv_detail::hip_fail;
using rvkv_detail::kMaxKeys;

namespace {

constexpr int kRows = 128, kKeys = 64;
constexpr float kLog2e = 1.4426950408889634f;

struct PackedArgs {
  const void *q;
  void *out;
  const unsigned char *kc, *vc;
  const uint32_t *tables, *row_start, *pos_offset, *read_num;
  size_t rec;
  uint32_t total_rows, batch, n_heads, n_kv, group, hd, bs, max_blocks;
  uint32_t num_blocks, window;
  int32_t bsg_log2;  // log2(bs / 16), -1 if that is no power of two
  float qscale;      // scale * log2(e)
};

__device__ __forceinline__ half2v pk(float a, float b) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(a, b));
}

template <int HD>
struct Tile {
  // (16 bytes between rows beyond their length: rows on other banks)
  _Float16 k[kKeys][HD + 8];
  _Float16 v[HD][kKeys + 8];
  float ks[kKeys], vs[kKeys];
  float vtop[2];
};

template <typename T, int HD, bool SPLIT>
__global__ void __launch_bounds__(256)
    q8_prefill_kernel(PackedArgs a) {
  constexpr int NC = HD / 16, ND = HD / 32;
  constexpr int KPT = HD / 64;  // 16-byte chunks of K, and of V, a thread
  constexpr float kNone = -__builtin_inff();
  extern __shared__ __align__(16) unsigned char smem[];
  Tile<HD> *tiles = reinterpret_cast<Tile<HD> *>(smem);
  const uint32_t tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const uint32_t col = lane & 31, h = lane >> 5;
  const uint32_t G = a.group, kvh = blockIdx.y, hd = a.hd, bs = a.bs;

  // The tile index space: sequence b owns row_start[b] * G / 128 + b onward,
  // at least as many as it has tiles. b = (sequences that start at or before
  // this index) - 1.
  const uint32_t t = gridDim.x - 1 - blockIdx.x;
  uint32_t seq, local;
  {
    __shared__ uint32_t count;
    if (tid == 0) count = 0;
    __syncthreads();
    uint32_t n = 0;
    for (uint32_t b = tid; b < a.batch; b += 256) {
      const uint32_t r = a.row_start[b] < a.total_rows ? a.row_start[b]
                                                       : a.total_rows;
      n += (uint64_t)r * G / kRows + b <= t ? 1 : 0;
    }
    if (n) atomicAdd(&count, n);  // (a whole number: any order)
    __syncthreads();
    if (count == 0) return;
    seq = count - 1;
  }
  uint32_t r0 = a.row_start[seq], r1 = a.row_start[seq + 1];
  r0 = r0 < a.total_rows ? r0 : a.total_rows;
  r1 = r1 < a.total_rows ? r1 : a.total_rows;
  local = t - (uint32_t)((uint64_t)r0 * G / kRows + seq);
  const uint64_t n_flat = r1 > r0 ? (uint64_t)(r1 - r0) * G : 0;
  const uint64_t f0 = (uint64_t)local * kRows;
  if (f0 >= n_flat) return;

  // (contexts end below 2^32 - 256, so that no key index wraps)
  const uint64_t most = (uint64_t)a.max_blocks * bs;
  const uint64_t cap = most < kMaxKeys ? most : kMaxKeys;
  uint64_t read = a.read_num[seq];
  read = read < cap ? read : cap;
  const uint64_t pos0 = a.pos_offset[seq];
  // This lane's q row, and the keys [key_lo, key_hi) that it sees.
  const uint64_t f = f0 + wave * 32 + col;
  const bool live = f < n_flat;
  const uint32_t tok = (uint32_t)((live ? f : f0) / G);
  const uint32_t head = kvh * G + (uint32_t)((live ? f : f0) % G);
  const size_t row = ((size_t)(r0 + tok) * a.n_heads + head) * hd;
  const uint64_t pos = pos0 + tok;
  uint32_t key_hi = (uint32_t)(pos + 1 < read ? pos + 1 : read);
  uint32_t key_lo = a.window && pos + 1 > a.window
                        ? (uint32_t)(pos + 1 - a.window < read
                                         ? pos + 1 - a.window : read) : 0;
  if (!live) key_hi = key_lo = 0;
  // The workgroup's keys: those of its first and last row.
  const uint64_t last = f0 + kRows < n_flat ? f0 + kRows - 1 : n_flat - 1;
  const uint64_t pos_last = pos0 + last / G, pos_first = pos0 + f0 / G;
  const uint32_t end = (uint32_t)(pos_last + 1 < read ? pos_last + 1 : read);
  uint32_t beg = 0;
  if (a.window && pos_first + 1 > a.window)
    beg = (uint32_t)(pos_first + 1 - a.window < read
                         ? pos_first + 1 - a.window : read);
  beg &= ~15u;
  // Keys that every row of this wave sees, and that any does.
  uint32_t all_lo = key_lo, all_hi = live ? key_hi : 0xffffffffu,
           any_hi = key_hi;
  uint32_t any_lo = live ? key_lo : 0xffffffffu;
#pragma unroll
  for (int o = 16; o >= 1; o >>= 1) {
    all_lo = max(all_lo, (uint32_t)__shfl_xor((int)all_lo, o));
    all_hi = min(all_hi, (uint32_t)__shfl_xor((int)all_hi, o));
    any_hi = max(any_hi, (uint32_t)__shfl_xor((int)any_hi, o));
    any_lo = min(any_lo, (uint32_t)__shfl_xor((int)any_lo, o));
  }

  // q: element j of chunk c is dim 16 c + 8 h + j.
  half8v qh[NC], ql[SPLIT ? NC : 1];
  float qscale = a.qscale;
  {
    const T *q = (const T *)a.q + row;
    if constexpr (!SPLIT) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
        qh[c] = live && (uint32_t)c * 16 < hd
                    ? *reinterpret_cast<const half8v *>(q + c * 16 + 8 * h)
                    : half8v{};
    } else {
      // (brought just below 2^15 by a power of two: neither part leaves f16's
      // range, the lower one not its normal numbers)
      float top = 0.f;
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (live && (uint32_t)c * 16 < hd)
            top = fmaxf(top, fabsf((float)q[c * 16 + 8 * h + j]));
      top = fmaxf(top, __shfl_xor(top, 32));
      const uint32_t ex = scale_exponent(top);
      const float down = __uint_as_float((269 - ex) << 23);
      qscale *= __uint_as_float((ex - 15) << 23);
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float y = live && (uint32_t)c * 16 < hd
                              ? (float)q[c * 16 + 8 * h + j] * down : 0.f;
          qh[c][j] = (_Float16)y;
          ql[c][j] = (_Float16)(y - (float)qh[c][j]);
        }
    }
  }

  const uint32_t *table = a.tables + (size_t)seq * a.max_blocks;
  const uint32_t last_granule = end ? (end - 1) / 16 : 0;
  // The records of a tile's four granules of 16 keys (uniform).
  struct Places {
    uint32_t blk[4], in[4];
  };
  const auto places = [&](uint32_t kt) {
    Places p;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t x = kt / 16 + i;
      x = x < last_granule ? x : last_granule;
      const uint32_t bi = a.bsg_log2 >= 0 ? x >> a.bsg_log2 : x / (bs / 16);
      p.in[i] = x - bi * (bs / 16);
      p.blk[i] = table[bi];
    }
    return p;
  };
  const auto pick = [](const uint32_t (&x)[4], uint32_t i) {
    return i & 2 ? (i & 1 ? x[3] : x[2]) : (i & 1 ? x[1] : x[0]);
  };
  uint4 kraw[KPT], vraw[KPT];
  float sraw;
  const auto fetch = [&](uint32_t kt, const Places &p) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const uint32_t x = tid + 256 * i;
      const uint32_t key = x / NC, ch = x % NC, gr = key / 16;
      uint32_t blk = pick(p.blk, gr);
      blk = blk < a.num_blocks ? blk : 0;
      kraw[i] = uint4{};
      if (ch * 16 < hd)
        kraw[i] = *reinterpret_cast<const uint4 *>(
            a.kc + blk * a.rec + (size_t)kvh * bs * hd +
            (pick(p.in, gr) * 16 + key % 16) * hd + ch * 16);
      const uint32_t d = x / 4, gv = x % 4;
      blk = pick(p.blk, gv);
      blk = blk < a.num_blocks ? blk : 0;
      vraw[i] = uint4{};
      if (d < hd)
        vraw[i] = *reinterpret_cast<const uint4 *>(
            a.vc + blk * a.rec + (size_t)kvh * bs * hd + (size_t)d * bs +
            pick(p.in, gv) * 16);
    }
    // Scales: threads 0-63 K's, 64-127 V's; 0 where the key cannot be read.
    if (tid < 128) {
      const uint32_t key = tid & 63, gr = key / 16;
      const uint32_t blk = pick(p.blk, gr);
      const bool ok = blk < a.num_blocks && kt + key < end;
      sraw = ok ? *reinterpret_cast<const float *>(
                      (tid < 64 ? a.kc : a.vc) + blk * a.rec +
                      (size_t)a.n_kv * bs * hd +
                      ((size_t)kvh * bs + pick(p.in, gr) * 16 + key % 16) * 4)
                : 0.f;
    }
  };
  const auto put = [&](Tile<HD> &s) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const uint32_t x = tid + 256 * i;
      half8v *k = reinterpret_cast<half8v *>(&s.k[x / NC][x % NC * 16]);
      k[0] = codes_to_half8(kraw[i].x, kraw[i].y);
      k[1] = codes_to_half8(kraw[i].z, kraw[i].w);
      half8v *v = reinterpret_cast<half8v *>(&s.v[x / 4][x % 4 * 16]);
      v[0] = codes_to_half8(vraw[i].x, vraw[i].y);
      v[1] = codes_to_half8(vraw[i].z, vraw[i].w);
    }
    if (tid < 64) s.ks[tid] = sraw;
    if (tid >= 64 && tid < 128) {
      s.vs[tid - 64] = sraw;
      float top = sraw;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      if (tid == 64) s.vtop[0] = top;
    }
  };

  float m = kNone, l = 0.f;
  float vnorm = kVnorm0;  // power of two above every vs
  float16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = float16v{};

  if (beg < end) {
    Places p = places(beg);
    fetch(beg, p);
    put(tiles[0]);
    uint32_t bad = 0;  // granules of the current tile that cannot be read
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= (p.blk[i] >= a.num_blocks) << i;
    p = places(beg + kKeys);
    __syncthreads();
    uint32_t buf = 0;
    for (uint32_t kt = beg; kt < end; kt += kKeys, buf ^= 1) {
      const Tile<HD> &s = tiles[buf];
      const bool more = end - kt > kKeys;
      uint32_t bad_next = 0;
      if (more) {
        fetch(kt + kKeys, p);
#pragma unroll
        for (int i = 0; i < 4; ++i) bad_next |= (p.blk[i] >= a.num_blocks) << i;
        p = places(kt + 2 * kKeys);
      }
      if (kt < any_hi && kt + kKeys > any_lo) {  // (uniform over the wave)
        float16v sc[2];
        const uint32_t key_row = 16 * (col >> 4) + 8 * ((col >> 2) & 1) +
                                 4 * ((col >> 3) & 1) + (col & 3);
#pragma unroll
        for (int kh = 0; kh < 2; ++kh) {
          sc[kh] = float16v{};
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            const half8v kf = *reinterpret_cast<const half8v *>(
                &s.k[kh * 32 + key_row][c * 16 + 8 * h]);
            sc[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qh[c], sc[kh],
                                                            0, 0, 0);
            if constexpr (SPLIT)
              sc[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, ql[c],
                                                              sc[kh], 0, 0, 0);
          }
        }
        // Result register 8 u + j of half kh: key 32 kh + 16 u + 8 h + j.
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const float4v k4 = *reinterpret_cast<const float4v *>(
                &s.ks[kh * 32 + 16 * (r >> 3) + 8 * h + (r & 7)]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              sc[kh][r + i] *= k4[i] * qscale;
          }
        if (kt < all_lo || kt + kKeys > all_hi || bad) {
#pragma unroll
          for (int kh = 0; kh < 2; ++kh)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
              const uint32_t key = kt + kh * 32 + 16 * (r >> 3) + 8 * h +
                                   (r & 7);
              const bool ok = key >= key_lo && key < key_hi &&
                              !(bad >> (2 * kh + (r >> 3)) & 1);
              sc[kh][r] = ok ? sc[kh][r] : kNone;
            }
        }
        float top = sc[0][0];
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, sc[kh][r]);
        top = fmaxf(top, __shfl_xor(top, 32));
        const float m_new = fmaxf(m, top);
        const float mm = m_new == kNone ? 0.f : m_new;
        float fix = m == m_new ? 1.f : __builtin_amdgcn_exp2f(m - mm);
        m = m_new;
        l *= fix;
        const float vtop = s.vtop[0];
        if (vtop >= vnorm) {  // (uniform)
          uint32_t e = (__float_as_uint(vtop) >> 23) + 1;
          e = e > 253 ? 253 : e;
          const float now = __uint_as_float(e << 23);
          fix *= vnorm / now;
          vnorm = now;
        }
        if (!__all(fix == 1.f)) {
#pragma unroll
          for (int d = 0; d < ND; ++d) o[d] *= fix;
        }
        // (weights up to 2^15, as q)
        const float vdown =
            __uint_as_float((269u << 23) - __float_as_uint(vnorm));
        half8v ph[4], pl[SPLIT ? 4 : 1];
#pragma unroll
        for (int kh = 0; kh < 2; ++kh)
#pragma unroll
          for (int r = 0; r < 16; r += 4) {
            const float4v v4 = *reinterpret_cast<const float4v *>(
                &s.vs[kh * 32 + 16 * (r >> 3) + 8 * h + (r & 7)]);
            float w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float x = __builtin_amdgcn_exp2f(sc[kh][r + i] - mm);
              l += x;
              // (0 for a key that is left out, whatever its scale holds)
              w[i] = rvkv_mul0(x, v4[i] * vdown);
            }
            half8v &up = ph[2 * kh + (r >> 3)];
            if constexpr (SPLIT) {
              half8v &lo = pl[2 * kh + (r >> 3)];
#pragma unroll
              for (int i = 0; i < 4; i += 2) {
                const half2v x = pk(w[i], w[i + 1]);
                const half2v y = pk(w[i] - (float)x[0],
                                    w[i + 1] - (float)x[1]);
                up[(r & 7) + i] = x[0];
                up[(r & 7) + i + 1] = x[1];
                lo[(r & 7) + i] = y[0];
                lo[(r & 7) + i + 1] = y[1];
              }
            } else {
#pragma unroll
              for (int i = 0; i < 4; ++i) up[(r & 7) + i] = (_Float16)w[i];
            }
          }
#pragma unroll
        for (int d = 0; d < ND; ++d)
          if ((uint32_t)d * 32 < hd) {
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const half8v vf = *reinterpret_cast<const half8v *>(
                  &s.v[d * 32 + col][x * 16 + 8 * h]);
              o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, ph[x], o[d], 0,
                                                            0, 0);
              if constexpr (SPLIT)
                o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf, pl[x], o[d],
                                                              0, 0, 0);
            }
          }
      }
      if (more) put(tiles[buf ^ 1]);
      bad = bad_next;
      __syncthreads();
    }
  }

  l += __shfl_xor(l, 32);
  if (!live) return;
  T *out = (T *)a.out + row;
  const float inv = l == 0.f ? 0.f : vnorm * 0x1p-15f / l;
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int r = 0; r < 16; r += 4) {
      const uint32_t dim = d * 32 + 2 * r + 4 * h;
      if (dim < hd) {
        typedef T vec4 __attribute__((ext_vector_type(4)));
        vec4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = (T)(o[d][r + i] * inv);
        *reinterpret_cast<vec4 *>(out + dim) = y;
      }
    }
}

template <typename T, int HD, bool SPLIT>
int launch(const char *op, const PackedArgs &a, hipStream_t st) {
  const size_t lds = 2 * sizeof(Tile<HD>);
  static const hipError_t set = hipFuncSetAttribute(
      reinterpret_cast<const void *>(&q8_prefill_kernel<T, HD, SPLIT>),
      hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (set != hipSuccess) return hip_fail(op, set);
  const uint64_t tiles = (uint64_t)a.total_rows * a.group / kRows + a.batch;
  if (tiles > 0x7fffffffull)
    return fail(RVKV_EUNSUPPORTED, op, "too many rows for one launch");
  hipLaunchKernelGGL((q8_prefill_kernel<T, HD, SPLIT>),
                     dim3((uint32_t)tiles, a.n_kv), dim3(256), lds, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RVKV_OK : hip_fail(op, e);
}

template <typename T, bool SPLIT>
int launch(const char *op, const PackedArgs &a, hipStream_t st) {
  if (a.hd <= 64) return launch<T, 64, SPLIT>(op, a, st);
  if (a.hd <= 128) return launch<T, 128, SPLIT>(op, a, st);
  return launch<T, 256, SPLIT>(op, a, st);
}

}  // namespace

extern "C" {

int rvkv_q8_packed_prefill(const rvkv_q8_pool *pool, uint32_t layer,
                           const void *q, rvkv_dtype dtype,
                           const uint32_t *row_start, uint32_t total_rows,
                           const uint32_t *block_tables,
                           const uint32_t *pos_offset,
                           const uint32_t *read_num_tokens, uint32_t batch,
                           uint32_t max_blocks, uint32_t n_heads, float scale,
                           int32_t window, void *out) {
  const char *op = "packed_prefill";
  if (!pool) return fail(RVKV_EINVAL, op, "pool is NULL");
  if (layer >= pool->n_layers)
    return fail(RVKV_EINVAL, op, "layer out of range");
  if (dtype != RVKV_F16 && dtype != RVKV_F32)
    return fail(RVKV_EINVAL, op, "dtype must be F16 or F32");
  if (total_rows == 0 || batch == 0) return RVKV_OK;
  if (max_blocks == 0)
    return fail(RVKV_EINVAL, op, "max_blocks must be positive");
  if (n_heads == 0 || n_heads % pool->n_kv != 0)
    return fail(RVKV_EINVAL, op,
                "n_heads must be a positive multiple of n_kv_heads");
  if (!q || !row_start || !block_tables || !pos_offset || !read_num_tokens ||
      !out)
    return fail(RVKV_EINVAL, op,
                "NULL q/row_start/block_tables/pos_offset/read_num_tokens/out");
  if ((uintptr_t)q % 16 || (uintptr_t)out % 16)
    return fail(RVKV_EINVAL, op, "q and out must be 16-byte aligned");
  const uint32_t bsg = pool->block_size / 16;
  const int rc = rvkv_detail::q8_device(op, pool->device);
  if (rc) return rc;
  PackedArgs a{};
  a.q = q;
  a.out = out;
  a.kc = pool->tensor(layer, 0);
  a.vc = pool->tensor(layer, 1);
  a.tables = block_tables;
  a.row_start = row_start;
  a.pos_offset = pos_offset;
  a.read_num = read_num_tokens;
  a.rec = pool->rec;
  a.total_rows = total_rows;
  a.batch = batch;
  a.n_heads = n_heads;
  a.n_kv = pool->n_kv;
  a.group = n_heads / pool->n_kv;
  a.hd = pool->head_dim;
  a.bs = pool->block_size;
  a.max_blocks = max_blocks;
  a.num_blocks = pool->num_blocks;
  a.window = window > 0 ? (uint32_t)window : 0;
  a.bsg_log2 = bsg & (bsg - 1) ? -1 : __builtin_ctz(bsg);
  a.qscale = scale * kLog2e;
  return dtype == RVKV_F16 ? launch<_Float16, false>(op, a, pool->stream)
                           : launch<float, true>(op, a, pool->stream);
}

}  // extern "C"
