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
//
// Bound by issue: a tile of 64 keys costs a wave its matrix cycles (1024 at hd
// 128) and then its vector cycles (softmax, conversion, staging: ~1600), which
// overlap little. Seven prompts of 571 to 4001 rows, 16 + 8 heads of 128: 187
// GFLOP in 284 us, 660 TFLOP/s; 4 prompts up to 4000 at 32 + 8 heads of 64: 555.
// With 64 rows a wave, each LDS operand feeding two products, the accumulators
// move between the register files every tile: 514 us.
#include <atomic>

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
  uint32_t n_tiles, n_pieces, piece_keys;
  int32_t bsg_log2;  // log2(bs / 16), -1 if that is no power of two
  float qscale;      // scale * log2(e)
  float *ws_acc, *ws_ml;
};

__device__ __forceinline__ half2v pk(float a, float b) {
  return __builtin_bit_cast(half2v, __builtin_amdgcn_cvt_pkrtz(a, b));
}

__device__ __forceinline__ float max_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x),
                                                  __float_as_uint(x), false,
                                                  false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

template <int HD>
struct alignas(16) Tile {
  // (16 bytes between rows beyond their length: rows on other banks)
  _Float16 k[kKeys][HD + 8];
  _Float16 v[HD][kKeys + 8];
  float ks[kKeys];  // K scale * scale * log2(e)
  float vs[kKeys];  // V scale * 2^6 / vnorm; 0 for a key that cannot be read
  float vnorm;      // a power of two above every V scale so far
  uint32_t bad;     // bit i: granule i (16 keys) lies in no block
};

// A workgroup's tile: 128 flattened rows (token * group + head) of one
// sequence from f0 on, its sequence's fields, and the keys [beg, end) that
// its rows see.
struct Work {
  uint32_t seq, r0, beg, end, f0, n_flat;  // (the host keeps rows * group
  uint64_t pos0, read;                     //  below 2^32)
};

// Sum and maximum over a wave, by DPP and swaps of rows (by LDS exchanges each
// took ~500 cycles, and a workgroup's search for its tile takes ten).
template <typename F>
__device__ __forceinline__ uint32_t over_wave(uint32_t x, F f) {
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x128, 0xf, 0xf, true));
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x124, 0xf, 0xf, true));
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x122, 0xf, 0xf, true));
  x = f(x, (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x121, 0xf, 0xf, true));
  const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = f((uint32_t)a[0], (uint32_t)a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return uniform(f((uint32_t)b[0], (uint32_t)b[1]));
}
__device__ __forceinline__ uint32_t wave_sum(uint32_t x) {
  return over_wave(x, [](uint32_t u, uint32_t v) { return u + v; });
}
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
  return over_wave(x, [](uint32_t u, uint32_t v) { return u > v ? u : v; });
}
__device__ __forceinline__ uint32_t wave_min(uint32_t x) {
  return over_wave(x, [](uint32_t u, uint32_t v) { return u < v ? u : v; });
}

// The t-th tile of the launch; false: there are no more than t. Every wave
// finds it by itself.
//
// Up to 256 sequences: the tiles level by level, those furthest into their
// sequence (which see the most keys) first: with n_b tiles in sequence b,
// C(j) = sum max(0, n_b - j) tiles lie at level j or above, so tile t is at
// the level with C(j + 1) <= t < C(j), of the (t - C(j+1))-th sequence that
// reaches it. (Sequence by sequence, a long one's tiles could start last: 519
// against 461 us at seven prompts of 571 to 4001 rows.)
//
// More sequences: one behind the other, b owning indices row_start[b] * group
// / 128 + b onward, at least as many as it has tiles; the host's n_tiles
// counts in that way.
__device__ __forceinline__ bool find_work(const PackedArgs &a, uint32_t t,
                                          Work &w) {
  const uint32_t lane = threadIdx.x & 63, G = a.group;
  uint32_t r0, r1, pos, read, local;
  const auto rows_at = [&](uint32_t b) {
    const uint32_t r = a.row_start[b];
    return r < a.total_rows ? r : a.total_rows;
  };
  if (a.batch <= 256) {
    uint32_t first[4], stop[4], p[4], rd[4], n[4];
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      first[i] = stop[i] = p[i] = rd[i] = n[i] = 0;
      if ((uint32_t)i * 64 >= a.batch) continue;  // (uniform)
      const uint32_t b = i * 64 + lane;
      if (b < a.batch) {
        first[i] = rows_at(b);
        stop[i] = rows_at(b + 1);
        p[i] = a.pos_offset[b];
        rd[i] = a.read_num[b];
      }
      if (stop[i] > first[i])
        n[i] = (uint32_t)(((uint64_t)(stop[i] - first[i]) * G + kRows - 1) /
                          kRows);
      most = max(most, n[i]);
    }
    const auto above = [&](uint32_t j) {
      uint32_t c = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) c += n[i] > j ? n[i] - j : 0;
      return wave_sum(c);
    };
    most = wave_max(most);
    if (t >= above(0)) return false;
    uint32_t lo = 0, hi = most;  // C(lo) > t >= C(hi)
    while (hi - lo > 1) {
      const uint32_t mid = (lo + hi) / 2;
      if (above(mid) > t) lo = mid;
      else hi = mid;
    }
    local = lo;
    uint32_t nth = t - above(lo + 1), seq = 0xffffffffu;
    r0 = r1 = pos = read = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if ((uint32_t)i * 64 >= a.batch || seq != 0xffffffffu) continue;
      uint64_t set = __ballot(n[i] > local);
      const uint32_t have = (uint32_t)__popcll(set);
      if (nth >= have) {
        nth -= have;
        continue;
      }
      for (; nth; --nth) set &= set - 1;
      const int at = __builtin_ctzll(set);
      seq = i * 64 + at;
      r0 = (uint32_t)__builtin_amdgcn_readlane((int)first[i], at);
      r1 = (uint32_t)__builtin_amdgcn_readlane((int)stop[i], at);
      pos = (uint32_t)__builtin_amdgcn_readlane((int)p[i], at);
      read = (uint32_t)__builtin_amdgcn_readlane((int)rd[i], at);
    }
    w.seq = seq;
  } else {
    t = a.n_tiles - 1 - t;
    uint32_t n = 0;
    for (uint32_t b0 = 0; b0 < a.batch; b0 += 64) {
      const uint32_t b = b0 + lane;
      n += (uint32_t)__popcll(__ballot(
          b < a.batch && (uint64_t)rows_at(b) * G / kRows + b <= t));
    }
    if (n == 0) return false;
    w.seq = n - 1;
    r0 = uniform(rows_at(w.seq));
    r1 = uniform(rows_at(w.seq + 1));
    pos = uniform(a.pos_offset[w.seq]);
    read = uniform(a.read_num[w.seq]);
    local = t - (uint32_t)((uint64_t)r0 * G / kRows + w.seq);
  }
  w.r0 = r0;
  w.pos0 = pos;
  w.n_flat = r1 > r0 ? (r1 - r0) * G : 0;
  w.f0 = local * kRows;
  if (w.f0 >= w.n_flat) return false;
  // (contexts end below 2^32 - 256, so that no key index wraps)
  const uint64_t most = (uint64_t)a.max_blocks * a.bs;
  const uint64_t cap = most < kMaxKeys ? most : kMaxKeys;
  w.read = read;
  w.read = w.read < cap ? w.read : cap;
  const uint32_t last = w.n_flat - w.f0 > kRows ? w.f0 + kRows - 1
                                                : w.n_flat - 1;
  const uint64_t pos_last = w.pos0 + last / G, pos_first = w.pos0 + w.f0 / G;
  w.end = (uint32_t)(pos_last + 1 < w.read ? pos_last + 1 : w.read);
  w.beg = 0;
  if (a.window && pos_first + 1 > a.window)
    w.beg = (uint32_t)(pos_first + 1 - a.window < w.read
                           ? pos_first + 1 - a.window : w.read);
  w.beg &= ~15u;
  return true;
}

template <typename T, int HD, bool SPLIT>
__global__ void __launch_bounds__(256, HD == 256 ? 1 : 2)
    q8_prefill_kernel(PackedArgs a) {
  constexpr int NC = HD / 16, ND = HD / 32;
  constexpr int KPT = HD / 64;  // 16-byte chunks of K, and of V, a thread
  constexpr float kNone = -__builtin_inff();
  extern __shared__ __align__(16) unsigned char smem[];
  Tile<HD> *tiles = reinterpret_cast<Tile<HD> *>(smem);
  const uint32_t tid = threadIdx.x, wave = uniform(tid >> 6), lane = tid & 63;
  const uint32_t col = lane & 31, h = lane >> 5;
  const uint32_t G = a.group, hd = a.hd, bs = a.bs, bsg = bs / 16;
  // KV heads innermost: the tiles of one head share an XCD's L2 where their
  // number is a multiple of eight.
  const uint32_t kvh = blockIdx.x % a.n_kv, rest = blockIdx.x / a.n_kv;
  const uint32_t piece = rest % a.n_pieces;
  const uint32_t t = rest / a.n_pieces;
  Work w;
  if (!find_work(a, t, w)) return;
  uint32_t beg = w.beg, end = w.end;
  bool whole = true;  // this workgroup sees all its rows' keys
  if (a.n_pieces > 1) {
    whole = end <= beg || end - beg <= a.piece_keys;
    if (whole) {
      if (piece) return;
    } else {
      const uint64_t from = (uint64_t)beg + (uint64_t)piece * a.piece_keys;
      if (from >= end) return;
      beg = (uint32_t)from;
      if (end - beg > a.piece_keys) end = beg + a.piece_keys;
    }
  }

  // This lane's q row, and the keys [key_lo, key_lo + span) that it sees.
  uint32_t all_lo = 0, all_hi = 0xffffffffu, any_lo = 0xffffffffu, any_hi = 0;
  const uint32_t f = w.f0 + wave * 32 + col;
  const bool live = f < w.n_flat;
  const uint32_t fl = live ? f : w.f0, tok = fl / G;
  const uint32_t head = kvh * G + (fl - tok * G);
  const size_t row = ((size_t)(w.r0 + tok) * a.n_heads + head) * hd;
  const uint64_t pos = w.pos0 + tok;
  const uint32_t key_hi = (uint32_t)(pos + 1 < w.read ? pos + 1 : w.read);
  const uint32_t key_lo =
      a.window && pos + 1 > a.window
          ? (uint32_t)(pos + 1 - a.window < w.read ? pos + 1 - a.window
                                                   : w.read) : 0;
  const uint32_t span = live && key_hi > key_lo ? key_hi - key_lo : 0;
  if (live) {
    all_lo = max(all_lo, key_lo);
    all_hi = min(all_hi, key_hi);
  }
  if (span) {
    any_lo = min(any_lo, key_lo);
    any_hi = max(any_hi, key_hi);
  }
  // Keys that every row of this wave sees, and that any does.
  all_lo = wave_max(all_lo);
  all_hi = wave_min(all_hi);
  any_lo = wave_min(any_lo);
  any_hi = wave_max(any_hi);

  const uint32_t *table = a.tables + (size_t)w.seq * a.max_blocks;
  const uint32_t last_granule = w.end ? (w.end - 1) / 16 : 0;
  // A granule's record and place in it (granules behind the last are not
  // looked up: their keys are masked).
  struct Place {
    uint32_t blk, in;
  };
  const auto place = [&](uint32_t x) {
    x = x < last_granule ? x : last_granule;
    Place p;
    const uint32_t bi = a.bsg_log2 >= 0 ? x >> a.bsg_log2 : x / bsg;
    p.in = x - bi * bsg;
    p.blk = table[bi];
    return p;
  };
  // K chunk i of a thread: key (tid + 256 i) / NC, in a granule that is the
  // wave's (its lanes' keys lie in one).
  const uint32_t k_key = tid / NC, k_ch = tid % NC;
  constexpr int kStep = 256 / NC;  // keys from one chunk to the next
  // (dims from hd on: any codes; q is 0 there, and they are not stored)
  const uint32_t k_dim = k_ch * 16 < hd ? k_ch * 16 : 0;
  const uint32_t gv = tid & 3, vd = tid >> 2;
  Place kp[KPT], vp, sp;
  const auto look_up = [&](uint32_t kt) {
#pragma unroll
    for (int i = 0; i < KPT; ++i)
      kp[i] = place(kt / 16 + uniform((k_key + kStep * i) >> 4));
    vp = place(kt / 16 + gv);
    sp = place(kt / 16 + (lane >> 4));
  };
  uint4 kraw[KPT], vraw[KPT];
  float sraw = 0.f;
  bool unread = false;
  const size_t head_at = (size_t)kvh * bs * hd;
  const unsigned char *scale_at =
      (wave == 0 ? a.kc : a.vc) + (size_t)a.n_kv * bs * hd +
      ((size_t)kvh * bs + (lane & 15)) * 4;
  const auto fetch = [&](uint32_t kt) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const uint32_t kb = kp[i].blk < a.num_blocks ? kp[i].blk : 0;
      kraw[i] = *reinterpret_cast<const uint4 *>(
          a.kc + kb * a.rec + head_at +
          (kp[i].in * 16 + ((k_key + kStep * i) & 15)) * hd + k_dim);
    }
    const uint32_t vb = vp.blk < a.num_blocks ? vp.blk : 0;
    const unsigned char *v0 = a.vc + vb * a.rec + head_at + vp.in * 16;
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      const uint32_t d = vd + 64 * i;
      vraw[i] = *reinterpret_cast<const uint4 *>(v0 + (d < hd ? d : 0) * bs);
    }
    if (wave < 2) {
      unread = sp.blk >= a.num_blocks;
      sraw = 0.f;
      if (!unread && kt + lane < end)
        sraw = *reinterpret_cast<const float *>(scale_at + sp.blk * a.rec +
                                                sp.in * 64);
    }
  };
  float v_so_far = kVnorm0;  // (wave 1's)
  const auto put = [&](Tile<HD> &s) {
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      half8v *k =
          reinterpret_cast<half8v *>(&s.k[k_key + kStep * i][k_ch * 16]);
      k[0] = codes_to_half8(kraw[i].x, kraw[i].y);
      k[1] = codes_to_half8(kraw[i].z, kraw[i].w);
    }
#pragma unroll
    for (int i = 0; i < KPT; ++i) {
      half8v *v = reinterpret_cast<half8v *>(&s.v[vd + 64 * i][gv * 16]);
      v[0] = codes_to_half8(vraw[i].x, vraw[i].y);
      v[1] = codes_to_half8(vraw[i].z, vraw[i].w);
    }
    if (wave == 0) {
      s.ks[lane] = sraw * a.qscale;
      const uint64_t b = __ballot(unread);
      if (lane == 0)
        s.bad = (uint32_t)((b & 1) | (b >> 15 & 2) | (b >> 30 & 4) |
                           (b >> 45 & 8));
    } else if (wave == 1) {
      float top = sraw;
#pragma unroll
      for (int o = 32; o >= 1; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
      if (top >= v_so_far) {
        uint32_t e = (__float_as_uint(top) >> 23) + 1;
        e = e > 253 ? 253 : e;
        v_so_far = __uint_as_float(e << 23);
      }
      s.vs[lane] =
          sraw * __uint_as_float((260u << 23) - __float_as_uint(v_so_far));
      if (lane == 0) s.vnorm = v_so_far;
    }
  };

  const bool any = beg < end;
  if (any) {
    look_up(beg);
    fetch(beg);
    look_up(beg + kKeys);
  }

  // q: element j of chunk c is dim 16 c + 8 h + j. rf: what a score is still
  // to be multiplied by.
  half8v qh[NC], ql[SPLIT ? NC : 1];
  float rf = 1.f;
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
    float x[NC][8];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        x[c][j] = live && (uint32_t)c * 16 < hd
                      ? (float)q[c * 16 + 8 * h + j] : 0.f;
        top = fmaxf(top, fabsf(x[c][j]));
      }
    top = max_halves(top);
    const uint32_t ex = scale_exponent(top);
    const float down = __uint_as_float((269 - ex) << 23);
    rf = __uint_as_float((ex - 15) << 23);
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float y = x[c][j] * down;
        qh[c][j] = (_Float16)y;
        ql[c][j] = (_Float16)(y - (float)qh[c][j]);
      }
  }

  // m: what the weights are relative to, their maximum to within 2^8 (it
  // moves, and o and l with it, only when a score passes it by more).
  float m = kNone, l = 0.f;
  float vnorm = kVnorm0;
  float16v o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = float16v{};
  const uint32_t key_row = 16 * (col >> 4) + 8 * ((col >> 2) & 1) +
                           4 * ((col >> 3) & 1) + (col & 3);

  const auto step = [&](const Tile<HD> &s, uint32_t kt) {
    float16v sc[2];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh) {
      sc[kh] = float16v{};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const half8v kf = *reinterpret_cast<const half8v *>(
            &s.k[kh * 32 + key_row][c * 16 + 8 * h]);
        sc[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            kf, qh[c], sc[kh], 0, 0, 0);
        if constexpr (SPLIT)
          sc[kh] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              kf, ql[c], sc[kh], 0, 0, 0);
      }
    }
    // Register 8 u + j of half kh: key 32 kh + 16 u + 8 h + j.
    const uint32_t bad = uniform(s.bad);
    const bool masked = kt < all_lo || kt + kKeys > all_hi || bad;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float4v k4 = *reinterpret_cast<const float4v *>(
            &s.ks[kh * 32 + 16 * (r >> 3) + 8 * h + (r & 7)]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[kh][r + i] *= k4[i];
      }
    if (masked) {  // (uniform over the wave)
      // (a branch, no selects on every tile)
      __builtin_amdgcn_sched_barrier(0);
      const uint32_t from = kt + 8 * h - key_lo;
#pragma unroll
      for (int kh = 0; kh < 2; ++kh)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const uint32_t key = from + kh * 32 + 16 * (r >> 3) + (r & 7);
          sc[kh][r] = key < span ? sc[kh][r] : kNone;
          if (bad >> (2 * kh + (r >> 3)) & 1) sc[kh][r] = kNone;
        }
    }
    float fix = 1.f;
    bool any_fix = false;
    float top = kNone;
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int r = 0; r < 16; r += 2)
        top = fmaxf(fmaxf(sc[kh][r], sc[kh][r + 1]), top);
    top = max_halves(top);
    if constexpr (SPLIT) top *= rf;
    if (__any(top > m + 8.f)) {
      const float now = fmaxf(m, top);
      // (-inf less -inf: nothing was seen, and nothing is held)
      fix = m == now ? 1.f : __builtin_amdgcn_exp2f(m - now);
      m = now;
      l *= fix;
      any_fix = true;
    }
    const float mm = m == kNone ? 0.f : m;
    if (s.vnorm != vnorm) {  // (uniform)
      fix *= vnorm / s.vnorm;
      vnorm = s.vnorm;
      any_fix = true;
    }
    if (any_fix) {
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= fix;
    }
    half8v ph[4], pl[SPLIT ? 4 : 1];
#pragma unroll
    for (int kh = 0; kh < 2; ++kh)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        const float4v v4 = *reinterpret_cast<const float4v *>(
            &s.vs[kh * 32 + 16 * (r >> 3) + 8 * h + (r & 7)]);
        const int x = 2 * kh + (r >> 3);
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
          float y[2];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float p = __builtin_amdgcn_exp2f(
                SPLIT ? __builtin_fmaf(sc[kh][r + i + e], rf, -mm)
                      : sc[kh][r + i + e] - mm);
            l += p;
            // (0 for a key that is left out, whatever its scale holds)
            y[e] = rvkv_mul0(p, v4[i + e]);
          }
          const int at = (r & 7) + i;
          if constexpr (SPLIT) {
            const half2v u = pk(y[0], y[1]);
            const half2v v = pk(y[0] - (float)u[0], y[1] - (float)u[1]);
            ph[x][at] = u[0];
            ph[x][at + 1] = u[1];
            pl[x][at] = v[0];
            pl[x][at + 1] = v[1];
          } else {
            ph[x][at] = (_Float16)y[0];
            ph[x][at + 1] = (_Float16)y[1];
          }
        }
      }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const half8v vf = *reinterpret_cast<const half8v *>(
            &s.v[d * 32 + col][x * 16 + 8 * h]);
        o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
            vf, ph[x], o[d], 0, 0, 0);
        if constexpr (SPLIT)
          o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
              vf, pl[x], o[d], 0, 0, 0);
      }
  };

  if (any) {
    put(tiles[0]);
    __syncthreads();
    uint32_t buf = 0;
    for (uint32_t kt = beg;; kt += kKeys, buf ^= 1) {
      const bool more = end - kt > kKeys;
      if (more) {
        fetch(kt + kKeys);
        look_up(kt + 2 * kKeys);
      }
      if (kt < any_hi && kt + kKeys > any_lo) step(tiles[buf], kt);
      if (!more) break;
      put(tiles[buf ^ 1]);
      __syncthreads();
    }
  }

  const float back = vnorm * 0x1p-6f;
  l += __shfl_xor(l, 32);
  if (!whole) {
    // A piece's part: o and l relative to m, for the merge.
    const size_t slot =
        ((size_t)(t * a.n_kv + kvh) * a.n_pieces + piece) * kRows +
        wave * 32 + col;
    float *to = a.ws_acc + slot * HD;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int r = 0; r < 16; r += 4) {
        float4v y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = o[d][r + i] * back;
        *reinterpret_cast<float4v *>(to + d * 32 + 2 * r + 4 * h) = y;
      }
    if (h == 0) {
      a.ws_ml[2 * slot] = m;
      a.ws_ml[2 * slot + 1] = l;
    }
  } else if (live) {
    T *out = (T *)a.out + row;
    const float inv = l == 0.f ? 0.f : back / l;
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
}

// Merges the pieces of tiles that were cut: HD / 4 threads a row, one row each.
template <typename T, int HD>
__global__ void __launch_bounds__(256) q8_prefill_reduce_kernel(PackedArgs a) {
  constexpr float kNone = -__builtin_inff();
  constexpr uint32_t TR = HD / 4;
  const uint32_t kvh = blockIdx.x % a.n_kv, t = blockIdx.x / a.n_kv;
  Work w;
  if (!find_work(a, t, w)) return;
  if (w.end <= w.beg || w.end - w.beg <= a.piece_keys) return;
  const uint32_t live = (w.end - w.beg - 1) / a.piece_keys + 1;
  const uint32_t d = threadIdx.x % TR * 4;
  {
    const uint32_t in = blockIdx.y * (256 / TR) + threadIdx.x / TR;
    const uint32_t f = w.f0 + in;
    if (f >= w.n_flat) return;
    const size_t slot0 = (size_t)(t * a.n_kv + kvh) * a.n_pieces * kRows + in;
    float top = kNone;
    for (uint32_t p = 0; p < live; ++p)
      top = fmaxf(top, a.ws_ml[2 * (slot0 + p * kRows)]);
    float4v o = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    for (uint32_t p = 0; p < live; ++p) {
      const size_t slot = slot0 + p * kRows;
      const float m = a.ws_ml[2 * slot];
      const float e = m == kNone ? 0.f : __builtin_amdgcn_exp2f(m - top);
      l += a.ws_ml[2 * slot + 1] * e;
      o += *reinterpret_cast<const float4v *>(a.ws_acc + slot * HD + d) * e;
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t tok = f / a.group;
    const uint32_t head = kvh * a.group + f % a.group;
    if (d < a.hd) {
      T *out = (T *)a.out + ((size_t)(w.r0 + tok) * a.n_heads + head) * a.hd;
      typedef T vec4 __attribute__((ext_vector_type(4)));
      vec4 y;
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = (T)(o[i] * inv);
      *reinterpret_cast<vec4 *>(out + d) = y;
    }
  }
}

uint32_t hd_up(uint32_t hd) { return hd <= 64 ? 64 : hd <= 128 ? 128 : 256; }

struct Layout {
  uint64_t n_tiles, n_pieces, piece_keys;
  size_t ml_off, bytes;
};

// How a call is cut: into the workgroups that are resident at once (256 CUs by
// two, by three at hd 64 in f16, by one above hd 128). The rows' tiles alone
// where they are at least half of that; otherwise each tile's keys as well, as
// far as the host can tell them from the width of the table and the window, in
// pieces of at least 128. 450 rows behind 7700 keys, 32 + 8 heads of 64: f32
// 109 us for 512 workgroups, 164 for 256, 137 for 768; f16 74 us for 768, 83
// for 512, 136 for 256 (before the waves' search for their tile was shortened).
Layout layout(const rvkv_q8_pool *p, uint32_t total_rows, uint32_t batch,
              uint32_t n_heads, uint32_t max_blocks, uint32_t window,
              rvkv_dtype dtype) {
  Layout w{};
  const uint32_t G = n_heads / p->n_kv;
  const uint64_t want = p->head_dim > 128 ? 256
                        : p->head_dim <= 64 && dtype == RVKV_F16 ? 768 : 512;
  w.n_tiles = (uint64_t)total_rows * G / kRows + batch;
  w.n_pieces = 1;

  uint64_t keys = (uint64_t)max_blocks * p->block_size;
  if (keys > kMaxKeys) keys = kMaxKeys;
  const uint64_t band = (uint64_t)window + kRows / G + 16;
  if (window && band < keys) keys = band;
  w.piece_keys = keys;
  const uint64_t have = w.n_tiles * p->n_kv;
  if (have == 0 || have * 2 > want) return w;
  uint64_t n = (want + have - 1) / have;
  if (n > (keys + 127) / 128) n = (keys + 127) / 128;
  if (n > 16) n = 16;
  if (n < 2) return w;
  w.piece_keys = ((keys + n - 1) / n + kKeys - 1) / kKeys * kKeys;
  w.n_pieces = (keys + w.piece_keys - 1) / w.piece_keys;
  const size_t rows = (size_t)have * w.n_pieces * kRows;
  w.ml_off = rows * hd_up(p->head_dim) * 4;
  w.bytes = (w.ml_off + rows * 8 + 255) & ~(size_t)255;
  return w;
}

template <typename T, int HD, bool SPLIT>
int launch(const char *op, const PackedArgs &a, int device, hipStream_t st) {
  const size_t lds = 2 * sizeof(Tile<HD>);
  // (once on every device: bit d of done)
  static std::atomic<uint64_t> done{0};
  const uint64_t bit = 1ull << (device & 63);
  if (device > 63 || !(done.load() & bit)) {
    const hipError_t e = hipFuncSetAttribute(
        reinterpret_cast<const void *>(&q8_prefill_kernel<T, HD, SPLIT>),
        hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return hip_fail(op, e);
    done.fetch_or(bit);
  }
  hipLaunchKernelGGL((q8_prefill_kernel<T, HD, SPLIT>),
                     dim3(a.n_tiles * a.n_kv * a.n_pieces), dim3(256), lds, st,
                     a);
  if (a.n_pieces > 1)
    hipLaunchKernelGGL((q8_prefill_reduce_kernel<T, HD>),
                       dim3(a.n_tiles * a.n_kv, kRows * HD / 1024), dim3(256),
                       0, st, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? RVKV_OK : hip_fail(op, e);
}

template <typename T, bool SPLIT>
int launch(const char *op, const PackedArgs &a, int device, hipStream_t st) {
  if (a.hd <= 64) return launch<T, 64, SPLIT>(op, a, device, st);
  if (a.hd <= 128) return launch<T, 128, SPLIT>(op, a, device, st);
  return launch<T, 256, SPLIT>(op, a, device, st);
}

}  // namespace

extern "C" {

size_t rvkv_q8_prefill_workspace_bytes(const rvkv_q8_pool *pool,
                                       uint32_t total_rows, uint32_t batch,
                                       uint32_t n_heads, uint32_t max_blocks,
                                       int32_t window) {
  if (!pool || n_heads == 0 || n_heads % pool->n_kv) return 0;
  // (f16 is cut into as many pieces as f32, or more)
  return layout(pool, total_rows, batch, n_heads, max_blocks,
                window > 0 ? (uint32_t)window : 0, RVKV_F16).bytes;
}

int rvkv_q8_packed_prefill(const rvkv_q8_pool *pool, uint32_t layer,
                           const void *q, rvkv_dtype dtype,
                           const uint32_t *row_start, uint32_t total_rows,
                           const uint32_t *block_tables,
                           const uint32_t *pos_offset,
                           const uint32_t *read_num_tokens, uint32_t batch,
                           uint32_t max_blocks, uint32_t n_heads, float scale,
                           int32_t window, void *out, void *ws,
                           size_t ws_bytes) {
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
  const uint32_t win = window > 0 ? (uint32_t)window : 0;
  Layout w = layout(pool, total_rows, batch, n_heads, max_blocks, win, dtype);
  if (!ws) w.n_pieces = 1;
  if (w.n_pieces > 1 && ws_bytes < w.bytes)
    return fail(RVKV_EINVAL, op, "workspace smaller than the required bytes");
  if ((uintptr_t)ws % 256)
    return fail(RVKV_EINVAL, op, "workspace must be 256-byte aligned");
  // (a launch holds fewer than 2^32 threads)
  if (w.n_tiles > 0xffffffu || w.n_tiles * pool->n_kv * w.n_pieces > 0xffffffu)
    return fail(RVKV_EUNSUPPORTED, op, "too many rows for one launch");
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
  a.window = win;
  a.n_tiles = (uint32_t)w.n_tiles;
  a.n_pieces = (uint32_t)w.n_pieces;
  a.piece_keys = (uint32_t)w.piece_keys;
  a.ws_acc = static_cast<float *>(ws);
  a.ws_ml = reinterpret_cast<float *>(static_cast<char *>(ws) + w.ml_off);
  a.bsg_log2 = bsg & (bsg - 1) ? -1 : __builtin_ctz(bsg);
  a.qscale = scale * kLog2e;
  return dtype == RVKV_F16
             ? launch<_Float16, false>(op, a, pool->device, pool->stream)
             : launch<float, true>(op, a, pool->device, pool->stream);
}

}  // extern "C"
