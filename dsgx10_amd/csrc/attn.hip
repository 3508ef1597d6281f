// Attention of a decode step's rows over the paged cache (include/dsgx.h): a shared prefix and every sequence's own tokens.
//
// One pass over the tokens with the running maximum and sum of the softmax (in powers of two). The G = Hq / Hkv query heads that
// share a head of keys and values are G columns of one matrix product, times the rows that attend over the same tokens: a
// sequence's rows over its own tokens, all rows over the prefix. The tokens are cut into ranges, a workgroup each; what the ranges
// leave (maximum, sum, unnormalised output in f32) k_combine joins.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kv_cache.cuh"

namespace dsgx {
namespace {

typedef __bf16 v8bf_t __attribute__((ext_vector_type(8)));
typedef float v4f_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;

struct Plan {
  int sp, cp;  // ranges of the prefix, tokens a range
  int so, co;  // ranges of a sequence's own tokens, tokens a range
};
struct AttnArgs {
  dsgx_kv_cache c;
  dsgx_kv_batch b;
  Plan p;
  const uint16_t* q;
  uint16_t* out;
  float *lse, *part;
  float2* ml;
  int64_t ldq, ldo;
  int Hq, G, page_shift;
  float scale2;              // |scale| log2 e; 1 for a scale of zero
  uint32_t q_flip, q_keep;   // the scale's sign and whether it is zero, on the queries' bits
};

// The tokens and rows of a workgroup: a range of the prefix for all rows, or of a sequence's own tokens for its rows
struct Range {
  const int32_t* tab;
  int head, split, first, rows, len, lo, hi;  // lo .. hi - 1 of len tokens
  bool any;
};
__device__ __forceinline__ Range range_of(const AttnArgs& a, int prefix) {
  Range r{a.b.prefix, (int)blockIdx.x % a.c.Hkv, (int)blockIdx.x / a.c.Hkv, 0, a.b.rows, a.b.prefix_len, 0, 0, true};
  if (!prefix) {
    const int b = blockIdx.z;
    r.first = a.b.cu_rows ? a.b.cu_rows[b] : b * a.b.max_rows;
    const int end = a.b.cu_rows ? a.b.cu_rows[b + 1] : r.first + a.b.max_rows;
    if (r.first < 0 || end <= r.first || end > a.b.rows) {
      r.any = false;
      return r;
    }
    r.rows = end - r.first;
    const int cap = a.b.table_ld << a.page_shift, len = a.b.lens[b];
    r.len = len < 0 ? 0 : len > cap ? cap : len;
    r.tab = a.b.table + (size_t)b * a.b.table_ld;
  }
  const int chunk = prefix ? a.p.cp : a.p.co, splits = prefix ? a.p.sp : a.p.so;
  r.lo = r.split * chunk, r.hi = r.split == splits - 1 ? r.len : min(r.len, r.lo + chunk);
  if (r.lo >= r.hi && r.split > 0) r.any = false;  // (range 0 is always written)
  return r;
}
__device__ __forceinline__ u32x4_t query_bits(u32x4_t w, const AttnArgs& a) {
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (w[i] ^ a.q_flip) & a.q_keep;
  return w;
}

// The base of a column's powers of two is moved only once a score is 2^8 above it: the sums stay far from f32's end, and the outputs are
// rescaled a few times a range instead of every step
constexpr float kSlack = 8.f;

// max and sum over the four groups of sixteen lanes, in every lane
__device__ __forceinline__ float groups_max(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float groups_sum(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// What some rows of the step see of a token and earlier ones do not (the causal edge) must not reach the earlier ones, and a product
// with a zero would let an infinity or a NaN through. So such values are zero for the product, and the end of the kernel adds them to
// the rows that see them, which are infinite or NaN by them whatever else they hold. What no row sees is zero.
template <bool F8>
__device__ __forceinline__ bool is_wild(uint32_t half_or_byte) {
  return F8 ? (half_or_byte & 0x7Fu) == 0x7Fu : (half_or_byte & 0x7F80u) == 0x7F80u;
}
// a lane's words of a token's V: zero if `out`; at the causal edge (`edge`) without what is infinite or NaN, and whether there was any
template <bool F8, int N>
__device__ __forceinline__ bool clean_v(uint32_t (&w)[N], bool out, bool edge) {
  constexpr uint32_t bits = F8 ? 8 : 16, mask = F8 ? 0xFFu : 0xFFFFu;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (out) w[i] = 0u;
#pragma unroll
    for (uint32_t b = 0; b < 32; b += bits)
      if (edge && is_wild<F8>(w[i] >> b)) odd = true, w[i] &= ~(mask << b);
  }
  return odd;
}
// value d of a token's V if it is infinite or NaN, else 0
template <bool F8>
__device__ __forceinline__ float wild_value(const uint8_t* v, int d) {
  if (F8) return is_wild<true>(v[d]) ? __builtin_nanf("") : 0.f;
  const uint32_t b = reinterpret_cast<const uint16_t*>(v)[d];
  return is_wild<false>(b) ? bf16_bits_to_f32(b) : 0.f;
}
// own or prefix token t of a head's pool; null if its page does not exist
template <bool F8>
__device__ __forceinline__ const uint8_t* token_at(const AttnArgs& a, const int32_t* tab, const uint8_t* pool, int t) {
  const int page = tab[t >> a.page_shift];
  if (page < 0 || page >= a.c.npages) return nullptr;
  return pool + ((int64_t)page * a.c.page_stride + (int64_t)(t & (a.c.page - 1)) * a.c.tok_stride) * (F8 ? 1 : 2);
}

// ---- one wave, sixteen query columns, thirty-two tokens a step, nothing through LDS ----------------------------------------------
// Scores are S[token][query] = K Q^T by v_mfma_f32_16x16x32_bf16: a lane brings one token's (lane % 16) sixteen bytes a step of the
// product, so K goes from memory to the matrix unit as it is stored; a lane leaves four tokens' (4 (lane / 16) ..) scores of one query
// (lane % 16). O[d][query] = V^T P: the same eight scores of a lane (two tiles of sixteen tokens) are the P operand as they are, and
// the V operand is eight tokens' values of one d, which a lane picks out of the eight rows it loaded (a whole row of V is sixteen lanes):
// one byte permutation a pair. The d that a tile's row stands for is VL (lane % 16) + tile: a lane's results are contiguous.
template <int D, bool F8>
struct Narrow {
  static constexpr int NS = D / 32;               // steps of the score product
  static constexpr int VL = D / 16;               // values of a row of V a lane
  static constexpr int KW = F8 ? D / 64 : D / 32;  // 16-byte words of a row of K a lane
  static constexpr int VW = F8 ? VL / 4 : VL / 2;  // 32-bit words of a row of V a lane

  v8bf_t q[NS];
  v4f_t o[VL];
  float m, l;
  bool odd;  // see clean_v

  struct Block {
    u32x4_t k[2][KW];
    uint32_t v[8][VW];
  };

  __device__ __forceinline__ void begin() {
    m = -__builtin_inff(), l = 0.f, odd = false;
#pragma unroll
    for (int i = 0; i < VL; ++i) o[i] = v4f_t{0.f, 0.f, 0.f, 0.f};
  }
  // row: the lane's query (lane % 16), D values; null: none
  __device__ __forceinline__ void load_q(const uint16_t* row, int g, const AttnArgs& a) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = F8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      u32x4_t w = {0, 0, 0, 0};
      if (row) w = *reinterpret_cast<const DSGX_GLOBAL u32x4_t*>((uintptr_t)(row + d));
      q[s] = __builtin_bit_cast(v8bf_t, query_bits(w, a));
    }
  }
  // kp, vp: the pools at the two tiles' first tokens (wave-uniform); ts: bytes from token to token
  __device__ __forceinline__ static void load(Block& x, const uint8_t* const (&kp)[2], const uint8_t* const (&vp)[2], uint32_t ts, int lane) {
    const uint32_t c = lane & 15, g = lane >> 4;
    const uint32_t ko = c * ts + 16 * g, vo = 4 * g * ts + c * VW * 4;
#pragma unroll
    for (int a = 0; a < 2; ++a) {
#pragma unroll
      for (int j = 0; j < KW; ++j) x.k[a][j] = ldg_stream(kp[a], ko + 64 * j);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t at = vo + j * ts;
        uint32_t(&w)[VW] = x.v[4 * a + j];
        if constexpr (VW >= 4) {
#pragma unroll
          for (int h = 0; h < VW / 4; ++h) {
            const u32x4_t t = ldg_stream(vp[a], at + 16 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * h + i] = t[i];
          }
        } else if constexpr (VW == 2) {
          const u32x2_t t = __builtin_nontemporal_load((const DSGX_GLOBAL u32x2_t*)((const DSGX_GLOBAL uint8_t*)(uintptr_t)vp[a] + at));
          w[0] = t[0], w[1] = t[1];
        } else {
          w[0] = __builtin_nontemporal_load((const DSGX_GLOBAL uint32_t*)((const DSGX_GLOBAL uint8_t*)(uintptr_t)vp[a] + at));
        }
      }
    }
  }
  __device__ __forceinline__ static v8bf_t k_operand(const u32x4_t (&k)[KW], int s) {
    if (!F8) return __builtin_bit_cast(v8bf_t, k[s]);
    uint32_t w[4];
    fp8x8_to_bf16(k[s / 2][2 * (s % 2)], k[s / 2][2 * (s % 2) + 1], w);
    return __builtin_bit_cast(v8bf_t, u32x4_t{w[0], w[1], w[2], w[3]});
  }
  // the V operands of output tiles t and t + 1 (t even)
  __device__ __forceinline__ static void v_operands(const uint32_t (&v)[8][VW], int t, v8bf_t& lo, v8bf_t& hi) {
    u32x4_t a, b;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (!F8) {
        a[k] = __builtin_amdgcn_perm(v[2 * k + 1][t / 2], v[2 * k][t / 2], 0x05040100u);
        b[k] = __builtin_amdgcn_perm(v[2 * k + 1][t / 2], v[2 * k][t / 2], 0x07060302u);
      } else {
        const uint32_t w = __builtin_amdgcn_perm(v[2 * k + 1][t / 4], v[2 * k][t / 4], t % 4 ? 0x07030602u : 0x05010400u);
        a[k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
        b[k] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
      }
    }
    lo = __builtin_bit_cast(v8bf_t, a), hi = __builtin_bit_cast(v8bf_t, b);
  }
  // Thirty-two tokens, t0 the first. lim: the lane's query sees the tokens below it. there0, there1: the tiles' pages exist. all: no lane
  // has anything masked here (wave-uniform). The rows' limits run from lim_lo to seen.
  __device__ __forceinline__ void step(Block& x, int t0, int lim, bool there0, bool there1, bool all, int lim_lo, int seen, float s2, int lane) {
    const int g = lane >> 4;
    v4f_t s[2];
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      s[a] = v4f_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i) s[a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k_operand(x.k[a], i), q[i], s[a], 0, 0, 0);
    }
    float e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = s[i / 4][i % 4];
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
        const bool there = i < 4 ? there0 : there1;
        if (!there || t >= lim) e[i] = -__builtin_inff();
        odd |= clean_v<F8, VW>(x.v[i], !there || t >= seen, t >= lim_lo);
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
    mx = __fmul_rn(groups_max(mx), s2);
    if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {  // (-inf + slack: the first scores move it)
      const float to = fmaxf(m, mx), alpha = exp2_hw(m - (to == -__builtin_inff() ? 0.f : to));
      l *= alpha, m = to;
#pragma unroll
      for (int i = 0; i < VL; ++i) o[i] *= alpha;
    }
    const float base = m == -__builtin_inff() ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = exp2_hw(fmaf(e[i], s2, -base)), sum += e[i];
    l += sum;
    const u32x4_t pw = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])};
    const v8bf_t p = __builtin_bit_cast(v8bf_t, pw);
#pragma unroll
    for (int i = 0; i < VL; i += 2) {
      v8bf_t a, b;
      v_operands(x.v, i, a, b);
      o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p, o[i], 0, 0, 0);
      o[i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, p, o[i + 1], 0, 0, 0);
    }
  }
};

template <int D, bool F8>
__global__ void __launch_bounds__(256) k_attn_narrow(AttnArgs a, int prefix) {
  using N = Narrow<D, F8>;
  constexpr int VL = N::VL, LD = D + 4;
  extern __shared__ float lds[];  // [4][16][LD] outputs, then [4][16] maxima and sums
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
  const Range rg = range_of(a, prefix);
  if (!rg.any) return;
  const int h = rg.head, split = rg.split, rows = rg.rows, len = rg.len, lo = rg.lo, hi = rg.hi, first = rg.first, G = a.G;
  const int32_t* tab = rg.tab;
  const bool direct = a.p.sp + a.p.so == 1;
  const int esz = F8 ? 1 : 2;
  const uint32_t ts = (uint32_t)(a.c.tok_stride * esz);
  const uint8_t *kh = static_cast<const uint8_t*>(a.c.k) + h * a.c.head_stride * esz, *vh = static_cast<const uint8_t*>(a.c.v) + h * a.c.head_stride * esz;
  const float s2 = F8 ? a.scale2 * a.c.ks[h] : a.scale2, vs = F8 ? a.c.vs[h] : 1.f;
  float* red = lds + 4 * 16 * LD;

  const int cols = rows * G;
  for (int tile = blockIdx.y; tile * 16 < cols; tile += gridDim.y) {
    const int x = tile * 16 + col, row = x / G, head = h * G + x % G;
    const bool live = x < cols;
    const int lim = !live ? 0 : prefix ? len : len - rows + row + 1;
    // the limits of the tile's first and last row
    const int last = min(tile * 16 + 15, cols - 1) / G;
    const int lim_lo = prefix ? len : len - rows + (tile * 16) / G + 1, lim_hi = prefix ? len : len - rows + last + 1;
    N n;
    n.begin();
    n.load_q(live ? a.q + (size_t)(first + row) * a.ldq + (size_t)head * D : nullptr, g, a);
    const int stop = min(hi, lim_hi);

    auto fetch = [&](typename N::Block& blk, int t0, bool& there0, bool& there1) {
      const uint8_t *kp[2], *vp[2];
      bool th[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int t = t0 + 16 * i;
        int page = -1;
        if (t < stop) page = uni(tab[t >> a.page_shift]);
        th[i] = page >= 0 && page < a.c.npages;
        const int64_t at = th[i] ? ((int64_t)page * a.c.page_stride + (int64_t)(t & (a.c.page - 1)) * a.c.tok_stride) * esz : 0;
        kp[i] = kh + at, vp[i] = vh + at;
      }
      there0 = th[0], there1 = th[1];
      N::load(blk, kp, vp, ts, lane);
    };
    typename N::Block cur, nxt;
    bool c0 = false, c1 = false, n0 = false, n1 = false;
    int t0 = lo + 32 * wave;
    if (t0 < stop) fetch(cur, t0, c0, c1);
    for (; t0 < stop; t0 += 128) {
      if (t0 + 128 < stop) fetch(nxt, t0 + 128, n0, n1);
      const bool all = c0 && c1 && t0 + 32 <= lim_lo && t0 + 32 <= stop;
      n.step(cur, t0, min(lim, hi), c0, c1, all, min(lim_lo, hi), stop, s2, lane);
      cur = nxt, c0 = n0, c1 = n1;
    }

    if (__builtin_amdgcn_ballot_w64(n.odd)) {
#pragma unroll 1
      for (int t = max(lo, lim_lo); t < stop; ++t) {
        if ((((t - lo) >> 5) & 3) != wave) continue;
        const uint8_t* v = token_at<F8>(a, tab, vh, t);
        if (!v || t >= min(lim, hi)) continue;
#pragma unroll
        for (int i = 0; i < VL; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) n.o[i][j] += wild_value<F8>(v, VL * (4 * g + j) + i);
      }
    }
    // the four waves' parts of the answer joined
    n.l = groups_sum(n.l);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int m4 = 0; m4 < VL; m4 += 4)
        *reinterpret_cast<v4f_t*>(lds + (wave * 16 + col) * LD + VL * (4 * g + i) + m4) = v4f_t{n.o[m4][i], n.o[m4 + 1][i], n.o[m4 + 2][i], n.o[m4 + 3][i]};
    if (g == 0) red[wave * 16 + col] = n.m, red[64 + wave * 16 + col] = n.l;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * (D / 4); i += 256) {
      const int qc = i / (D / 4), d = 4 * (i % (D / 4)), xx = tile * 16 + qc;
      if (xx >= cols) continue;
      float mm = -__builtin_inff(), w[4], l = 0.f;
#pragma unroll
      for (int k = 0; k < 4; ++k) mm = fmaxf(mm, red[k * 16 + qc]);
      const float base = mm == -__builtin_inff() ? 0.f : mm;
      v4f_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        w[k] = exp2_hw(red[k * 16 + qc] - base);
        l = fmaf(w[k], red[64 + k * 16 + qc], l);
        const v4f_t v = *reinterpret_cast<const v4f_t*>(lds + (k * 16 + qc) * LD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(w[k], v[j], acc[j]);
      }
      const size_t rh = (size_t)(first + xx / G) * a.Hq + h * G + xx % G;
      if (direct) {
        const float inv = l == 0.f ? 0.f : __fdiv_rn(vs, l);
        *reinterpret_cast<uint2*>(a.out + (size_t)(first + xx / G) * a.ldo + (size_t)(h * G + xx % G) * D + d) =
            make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
        if (d == 0 && a.lse) a.lse[rh] = l == 0.f ? -__builtin_inff() : (mm + __builtin_amdgcn_logf(l)) * kLn2;
      } else {
        const size_t slot = (size_t)((prefix ? 0 : a.p.sp) + split) * a.b.rows * a.Hq + rh;
        *reinterpret_cast<v4f_t*>(a.part + slot * D + d) = acc;
        if (d == 0) a.ml[slot] = make_float2(mm, l);
      }
    }
  }
}

// ---- four waves, QW query columns each, tiles of 8192 / D tokens through LDS -------------------------------------------------------
// For many columns over the same tokens (the prefix under a batch, 64 heads over one) the matrix unit is the time, and a token's K and V
// are read by four waves. A tile is staged through registers: e4m3 becomes bf16 there, and V is transposed there (four tokens by eight
// values a thread, a byte permutation a pair), so that both operands are 16-byte reads from LDS. Layouts (chunks of 16 bytes): K as rows of
// a token, V as rows of a d whose chunks hold the eight tokens that one lane's scores belong to, so that the scores are the second
// product's operand as they stand; the chunks of a row are XORed with its number, which spreads sixteen lanes' rows over all banks.
// QW 32: v_mfma_f32_32x32x16_bf16, 128 columns a workgroup; QW 16: v_mfma_f32_16x16x32_bf16, 64 columns.
typedef float v16f_t __attribute__((ext_vector_type(16)));

template <int D, bool F8, int QW>
struct Wide {
  static constexpr int KV = 8192 / D;            // tokens a tile
  static constexpr int SR = QW / 16 * 4 * (QW / 16);  // accumulators of a tile a lane: 16 or 4
  static constexpr int LG = kWave / QW;          // lanes that share a column: 2 or 4
  static constexpr int KD = 8 * LG;              // k of one instruction: 16 or 32
  static constexpr int NS = D / KD, ST = KV / QW, OT = D / QW, NE = KV * QW / kWave, NP = NE / 8;
  static constexpr int KN = F8 ? 2 : 4, VW = F8 ? 2 : 4;
  static constexpr int kTile = 16384;            // bytes of a tile of K, of V
  using acc_t = typename std::conditional<QW == 32, v16f_t, v4f_t>::type;

  __device__ __forceinline__ static acc_t mfma(v8bf_t a, v8bf_t b, acc_t c) {
    if constexpr (QW == 32) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  // the token (in its tile) of a lane's score i, the d of its result i in output tile t
  __device__ __forceinline__ static int token_of(int i, int lg) {
    return QW == 32 ? 32 * (i / 16) + 8 * ((i % 16) / 4) + 4 * lg + i % 4 : 16 * (i / 4) + 4 * lg + i % 4;
  }
  __device__ __forceinline__ static uint32_t k_addr(uint32_t row, uint32_t c) {
    constexpr uint32_t CPR = D / 8;  // chunks a row
    if (D == 64) return row / 2 * 256 + (row & 1) * 128 + ((c ^ (row >> 1)) & 7) * 16;
    return row * (CPR * 16) + (c ^ (row & 15)) * 16;
  }
  __device__ __forceinline__ static uint32_t v_addr(uint32_t d, uint32_t c) {
    constexpr uint32_t CPR = KV / 8, RP = 16 / CPR;  // chunks a row, rows of 256 bytes
    return d * (CPR * 16) + ((c ^ (d / RP) ^ (d >> 4)) & (CPR - 1)) * 16;
  }

  // The operands' reads as the lane's address XOR a constant, plus a constant: row QW u + col, chunk LG k + lg of a tile of K ..
  __device__ __forceinline__ static uint32_t k_read(uint32_t lane_at, int u, int k) { return (lane_at ^ (uint32_t)(LG * k * 16)) + (uint32_t)(QW * u * D * 2); }
  // .. and row QW i + col, chunk LG k + lg of one of V^T (the row's share of the XOR that i makes is i's alone: no carries)
  __device__ __forceinline__ static uint32_t v_read(uint32_t lane_at, int i, int k) {
    constexpr uint32_t CPR = KV / 8, RP = 16 / CPR;
    const uint32_t x = (uint32_t)(LG * k) ^ ((uint32_t)(QW * i / RP) & (CPR - 1)) ^ ((uint32_t)(QW * i / 16) & (CPR - 1));
    return (lane_at ^ (x * 16)) + (uint32_t)(QW * i) * (CPR * 16);
  }

  struct Stage {
    u32x4_t k[KN];
    uint32_t v[4][VW];
  };
  // the sixteens of tokens that a thread's loads lie in: K's load i, V's
  __device__ __forceinline__ static uint32_t k_row(int i, uint32_t tid) { return (tid + 256 * i) / (F8 ? D / 16 : D / 8); }
  __device__ __forceinline__ static uint32_t k_chunk(int i, uint32_t tid) { return (tid + 256 * i) % (F8 ? D / 16 : D / 8); }
  __device__ __forceinline__ static uint32_t v_group(uint32_t tid) { return tid / (D / 8); }  // of four tokens

  // at: byte offsets of the tile's sixteens (lane s % 16 .. of `offs`), from the head's first value
  __device__ __forceinline__ static void load(Stage& x, const uint8_t* kh, const uint8_t* vh, uint64_t offs, uint32_t ts, uint32_t tid) {
    auto off = [&](uint32_t sixteen) {
      const uint32_t lo = __shfl((int)(uint32_t)offs, (int)sixteen), hi = __shfl((int)(offs >> 32), (int)sixteen);
      return (uint64_t)hi << 32 | lo;
    };
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const uint32_t row = k_row(i, tid);
      x.k[i] = *(const DSGX_GLOBAL u32x4_t*)(uintptr_t)(kh + off(row / 16) + (row % 16) * ts + 16 * k_chunk(i, tid));
    }
    const uint32_t grp = v_group(tid), dc = tid % (D / 8);
    const uint8_t* vb = vh + off(grp / 4) + (grp % 4) * 4 * ts + dc * VW * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (F8) {
        const u32x2_t t = *(const DSGX_GLOBAL u32x2_t*)(uintptr_t)(vb + j * ts);
        x.v[j][0] = t[0], x.v[j][1] = t[1];
      } else {
        const u32x4_t t = *(const DSGX_GLOBAL u32x4_t*)(uintptr_t)(vb + j * ts);
#pragma unroll
        for (int i = 0; i < 4; ++i) x.v[j][i] = t[i];
      }
    }
  }
  // tokens 4 grp .. + 3: their chunk of a row of V^T and the half of it
  __device__ __forceinline__ static uint32_t v_chunk(uint32_t grp) { return QW == 32 ? 2 * (grp / 4) + (grp & 1) : 4 * (grp / 8) + (grp & 3); }
  __device__ __forceinline__ static uint32_t v_half(uint32_t grp) { return QW == 32 ? (grp >> 1) & 1 : (grp >> 2) & 1; }
  __device__ __forceinline__ static void store(const Stage& x, uint8_t* kt, uint8_t* vt, uint32_t tid) {
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const uint32_t row = k_row(i, tid), c = k_chunk(i, tid);
      if constexpr (F8) {
        uint32_t w[4];
        fp8x8_to_bf16(x.k[i][0], x.k[i][1], w);
        *reinterpret_cast<u32x4_t*>(kt + k_addr(row, 2 * c)) = u32x4_t{w[0], w[1], w[2], w[3]};
        fp8x8_to_bf16(x.k[i][2], x.k[i][3], w);
        *reinterpret_cast<u32x4_t*>(kt + k_addr(row, 2 * c + 1)) = u32x4_t{w[0], w[1], w[2], w[3]};
      } else {
        *reinterpret_cast<u32x4_t*>(kt + k_addr(row, c)) = x.k[i];
      }
    }
    const uint32_t grp = v_group(tid), dc = tid % (D / 8), chunk = v_chunk(grp), half = v_half(grp);
#pragma unroll
    for (int i = 0; i < 8; i += 2) {  // d = 8 dc + i and the next
      u32x2_t a, b;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if constexpr (F8) {
          const uint32_t w = __builtin_amdgcn_perm(x.v[2 * h + 1][i / 4], x.v[2 * h][i / 4], i % 4 ? 0x07030602u : 0x05010400u);
          a[h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
          b[h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
        } else {
          a[h] = __builtin_amdgcn_perm(x.v[2 * h + 1][i / 2], x.v[2 * h][i / 2], 0x05040100u);
          b[h] = __builtin_amdgcn_perm(x.v[2 * h + 1][i / 2], x.v[2 * h][i / 2], 0x07060302u);
        }
      }
      *reinterpret_cast<u32x2_t*>(vt + v_addr(8 * dc + i, chunk) + 8 * half) = a;
      *reinterpret_cast<u32x2_t*>(vt + v_addr(8 * dc + i + 1, chunk) + 8 * half) = b;
    }
  }
};

// max and sum over the lanes that share a column
template <int QW>
__device__ __forceinline__ float column_max(float v) {
  if (QW == 16) return groups_max(v);
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
template <int QW>
__device__ __forceinline__ float column_sum(float v) {
  if (QW == 16) return groups_sum(v);
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <int D, bool F8, int QW>
__global__ void __launch_bounds__(256, D == 256 && QW == 32 ? 1 : 2) k_attn_wide(AttnArgs a, int prefix) {
  using W = Wide<D, F8, QW>;
  using acc_t = typename W::acc_t;
  constexpr int KV = W::KV, COLS = 4 * QW, NE = W::NE;
  extern __shared__ __align__(16) uint8_t tiles[];  // two tiles of K and V each
  __shared__ int any_odd;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const int wave = uni((int)tid >> 6), lg = lane / QW, col = lane % QW;
  const Range rg = range_of(a, prefix);
  if (!rg.any) return;
  const int h = rg.head, split = rg.split, rows = rg.rows, len = rg.len, lo = rg.lo, hi = rg.hi, first = rg.first, G = a.G;
  const int32_t* tab = rg.tab;
  constexpr int esz = F8 ? 1 : 2;
  const uint32_t ts = (uint32_t)(a.c.tok_stride * esz);
  const uint8_t *kh = static_cast<const uint8_t*>(a.c.k) + h * a.c.head_stride * esz, *vh = static_cast<const uint8_t*>(a.c.v) + h * a.c.head_stride * esz;
  const float s2 = F8 ? a.scale2 * a.c.ks[h] : a.scale2, vs = F8 ? a.c.vs[h] : 1.f;

  const int cols = rows * G;
  for (int tile = blockIdx.y; tile * COLS < cols; tile += gridDim.y) {
    const int x = tile * COLS + wave * QW + col, row = x / G, head = h * G + x % G;
    const bool live = x < cols;
    const int last = min(tile * COLS + COLS - 1, cols - 1) / G;
    const int lim_hi = prefix ? len : len - rows + last + 1, stop = min(hi, lim_hi);
    const int lim_lo = min(hi, prefix ? len : len - rows + tile * COLS / G + 1);
    const int lim = !live ? 0 : min(hi, prefix ? len : len - rows + row + 1);
    v8bf_t q[W::NS];
#pragma unroll
    for (int s = 0; s < W::NS; ++s) {
      u32x4_t w = {0, 0, 0, 0};
      if (live) w = *reinterpret_cast<const DSGX_GLOBAL u32x4_t*>((uintptr_t)(a.q + (size_t)(first + row) * a.ldq + (size_t)head * D + W::KD * s + 8 * lg));
      q[s] = __builtin_bit_cast(v8bf_t, query_bits(w, a));
    }
    acc_t o[W::OT];
#pragma unroll
    for (int i = 0; i < W::OT; ++i)
#pragma unroll
      for (int j = 0; j < W::SR; ++j) o[i][j] = 0.f;
    float m = -__builtin_inff(), l = 0.f;  // m: the base, in scores; l: this lane's part of the sum

    // lane s < KV / 16: the page of the sixteen s of a tile, and where it lies
    auto page_of = [&](int t0) {
      const int t = t0 + 16 * (int)lane;
      return (int)lane < KV / 16 && t < stop ? tab[t >> a.page_shift] : -1;
    };
    auto place = [&](int t0, int page, uint32_t& there) {
      const int t = t0 + 16 * (int)lane;
      const bool ok = page >= 0 && page < a.c.npages;
      there = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
      return ok ? (uint64_t)(((int64_t)page * a.c.page_stride + (int64_t)(t & (a.c.page - 1)) * a.c.tok_stride) * esz) : 0ull;
    };
    constexpr uint32_t kAll = (1u << (KV / 16)) - 1;
    bool odd = false;  // see clean_v
    auto clean = [&](typename W::Stage& st, int t0, uint32_t there) {
      const uint32_t grp = W::v_group(tid);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + 4 * (int)grp + j;
        odd |= clean_v<F8, W::VW>(st.v[j], !(there >> (grp / 4) & 1) || t >= stop, t >= lim_lo);
      }
    };

    typename W::Stage st;
    uint32_t there = 0, next_there = 0;
    int page = page_of(lo), ahead = page_of(lo + KV);
    __syncthreads();  // (the tiles of a column tile before this one have been read)
    if (lo < stop) {
      const uint64_t at = place(lo, page, there);
      W::load(st, kh, vh, at, ts, tid);
      if (there != kAll || lo + KV > lim_lo) clean(st, lo, there);
      W::store(st, tiles, tiles + W::kTile, tid);
    }
    const uint32_t k_at = W::k_addr(col, lg), v_at = W::v_addr(col, lg);
    int buf = 0;
    for (int t0 = lo; t0 < stop; t0 += KV, buf ^= 1) {
      __syncthreads();
      const bool more = t0 + KV < stop;
      if (more) {
        const uint64_t at = place(t0 + KV, ahead, next_there);
        W::load(st, kh, vh, at, ts, tid);
        ahead = page_of(t0 + 2 * KV);
      }
      const uint8_t *kt = tiles + buf * 2 * W::kTile, *vt = kt + W::kTile;
      uint32_t ka = k_at, va = v_at;
      asm volatile("" : "+v"(ka), "+v"(va));  // (else every operand's address is kept in a register of its own)
      float e[NE];
#pragma unroll
      for (int u = 0; u < W::ST; ++u) {
        acc_t s;
#pragma unroll
        for (int j = 0; j < W::SR; ++j) s[j] = 0.f;
#pragma unroll
        for (int k = 0; k < W::NS; ++k)
          s = W::mfma(__builtin_bit_cast(v8bf_t, *reinterpret_cast<const u32x4_t*>(kt + W::k_read(ka, u, k))), q[k], s);
#pragma unroll
        for (int j = 0; j < W::SR; ++j) e[u * W::SR + j] = s[j];
      }
      const bool all = there == kAll && t0 + KV <= lim_lo;
      if (!all) {
#pragma unroll
        for (int i = 0; i < NE; ++i) {
          const int tk = W::token_of(i, lg);
          if (!(there >> (tk / 16) & 1) || t0 + tk >= lim) e[i] = -__builtin_inff();
        }
      }
      float mx = e[0];
#pragma unroll
      for (int i = 1; i < NE; ++i) mx = fmaxf(mx, e[i]);
      mx = __fmul_rn(column_max<QW>(mx), s2);
      if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {  // (-inf + slack: the first scores move it)
        const float to = fmaxf(m, mx), base = to == -__builtin_inff() ? 0.f : to, alpha = exp2_hw(m - base);
        l *= alpha, m = to;
#pragma unroll
        for (int i = 0; i < W::OT; ++i)
#pragma unroll
          for (int j = 0; j < W::SR; ++j) o[i][j] *= alpha;
      }
      const float base = m == -__builtin_inff() ? 0.f : m;
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NE; ++i) e[i] = exp2_hw(fmaf(e[i], s2, -base)), sum += e[i];
      l += sum;
      v8bf_t p[W::NP];
#pragma unroll
      for (int k = 0; k < W::NP; ++k) {
        const u32x4_t pw = {pack_bf16(e[8 * k], e[8 * k + 1]), pack_bf16(e[8 * k + 2], e[8 * k + 3]), pack_bf16(e[8 * k + 4], e[8 * k + 5]), pack_bf16(e[8 * k + 6], e[8 * k + 7])};
        p[k] = __builtin_bit_cast(v8bf_t, pw);
      }
#pragma unroll
      for (int k = 0; k < W::NP; ++k)
#pragma unroll
        for (int i = 0; i < W::OT; ++i) o[i] = W::mfma(__builtin_bit_cast(v8bf_t, *reinterpret_cast<const u32x4_t*>(vt + W::v_read(va, i, k))), p[k], o[i]);
      if (more) {
        if (next_there != kAll || t0 + 2 * KV > lim_lo) clean(st, t0 + KV, next_there);
        uint8_t* nt = tiles + (buf ^ 1) * 2 * W::kTile;
        W::store(st, nt, nt + W::kTile, tid);
        there = next_there;
      }
    }

    l = column_sum<QW>(l);
    if (lim_lo < stop) {  // (wave-uniform, and the same for all waves)
      if (tid == 0) any_odd = 0;
      __syncthreads();
      if (odd) any_odd = 1;
      __syncthreads();
      if (any_odd) {
#pragma unroll 1
        for (int t = max(lo, lim_lo); t < stop; ++t) {
          const uint8_t* v = token_at<F8>(a, tab, vh, t);
          if (!v || t >= lim) continue;
#pragma unroll
          for (int i = 0; i < W::OT; ++i)
#pragma unroll
            for (int j = 0; j < W::SR; ++j) o[i][j] += wild_value<F8>(v, QW * i + W::LG * (j & ~3) + 4 * lg + (j & 3));
        }
      }
    }
    if (!live) continue;
    const size_t rh = (size_t)(first + row) * a.Hq + head;
    if (a.p.sp + a.p.so == 1) {
      const float inv = l == 0.f ? 0.f : __fdiv_rn(vs, l);
      uint16_t* dst = a.out + (size_t)(first + row) * a.ldo + (size_t)head * D;
#pragma unroll
      for (int i = 0; i < W::OT; ++i)
#pragma unroll
        for (int j = 0; j < W::SR; j += 4)
          *reinterpret_cast<uint2*>(dst + QW * i + W::LG * j + 4 * lg) = make_uint2(pack_bf16(o[i][j] * inv, o[i][j + 1] * inv), pack_bf16(o[i][j + 2] * inv, o[i][j + 3] * inv));
      if (lg == 0 && a.lse) a.lse[rh] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
    } else {
      const size_t slot = (size_t)((prefix ? 0 : a.p.sp) + split) * a.b.rows * a.Hq + rh;
      float* dst = a.part + slot * D;
#pragma unroll
      for (int i = 0; i < W::OT; ++i)
#pragma unroll
        for (int j = 0; j < W::SR; j += 4) *reinterpret_cast<v4f_t*>(dst + QW * i + W::LG * j + 4 * lg) = v4f_t{o[i][j], o[i][j + 1], o[i][j + 2], o[i][j + 3]};
      if (lg == 0) a.ml[slot] = make_float2(m, l);
    }
  }
}

// One wave a row's head: the ranges' outputs joined by their maxima
template <int D>
__global__ void __launch_bounds__(256) k_combine(AttnArgs a) {
  constexpr int PL = D / 64;
  const int lane = threadIdx.x & 63, r = blockIdx.x, head = uni((int)(blockIdx.y * 4 + (threadIdx.x >> 6)));
  if (head >= a.Hq) return;
  const RowPlace p = find_row(a.b, r, lane);
  if (p.seq < 0 || p.end > a.b.rows) return;
  const int cap = a.b.table_ld << a.page_shift, len = p.len < 0 ? 0 : p.len > cap ? cap : p.len;
  const int own = max(1, min(a.p.so, (len + a.p.co - 1) / a.p.co)), ns = a.p.sp + own;
  const size_t per = (size_t)a.b.rows * a.Hq, rh = (size_t)r * a.Hq + head;
  float mm = -__builtin_inff();
  for (int s = lane; s < ns; s += kWave) mm = fmaxf(mm, a.ml[s * per + rh].x);
  mm = wave_max_f32(mm);
  const float base = mm == -__builtin_inff() ? 0.f : mm;
  float acc[PL], l = 0.f;
#pragma unroll
  for (int j = 0; j < PL; ++j) acc[j] = 0.f;
  for (int s = 0; s < ns; ++s) {
    const float2 ml = a.ml[s * per + rh];
    const float w = exp2_hw(ml.x - base);
    l = fmaf(w, ml.y, l);
    const float* v = a.part + (s * per + rh) * D + PL * lane;
#pragma unroll
    for (int j = 0; j < PL; ++j) acc[j] = fmaf(w, v[j], acc[j]);
  }
  const float vs = a.c.fmt == DSGX_KV_E4M3 ? a.c.vs[head / a.G] : 1.f, inv = l == 0.f ? 0.f : __fdiv_rn(vs, l);
  uint16_t* o = a.out + (size_t)r * a.ldo + (size_t)head * D + PL * lane;
#pragma unroll
  for (int j = 0; j < PL; ++j) o[j] = (uint16_t)f32_to_bf16_bits(acc[j] * inv);
  if (lane == 0 && a.lse) a.lse[rh] = l == 0.f ? -__builtin_inff() : (mm + __builtin_amdgcn_logf(l)) * kLn2;
}

int round_up(int64_t v, int m) { return (int)((v + m - 1) / m * m); }

// How a set of tokens is worked on by `cols` query columns: sixteen of them a workgroup, or tiles through LDS for 64 or 128
enum Kind { kNarrow, kWide16, kWide32 };
Kind kind_of(int64_t cols) {
  return cols <= 16 ? kNarrow : cols <= 64 ? kWide16 : kWide32;
}
int cols_of(Kind k) { return k == kNarrow ? 16 : k == kWide16 ? 64 : 128; }

Plan make_plan(const dsgx_kv_cache& c, const dsgx_kv_batch& b, int Hq) {
  const int G = Hq / c.Hkv, cus = num_cus_cached();
  auto cut = [&](int64_t len, int64_t cols, int64_t sets, int& n, int& chunk) {
    const Kind k = kind_of(cols);
    const int64_t tiles = sets * c.Hkv * ((cols + cols_of(k) - 1) / cols_of(k));  // workgroups a range
    const int64_t want = std::max<int64_t>(1, (k == kNarrow ? 4 : 2) * (int64_t)cus / std::max<int64_t>(1, tiles));
    chunk = std::max(256, round_up((len + want - 1) / want, 128));
    n = (int)std::max<int64_t>(1, (len + chunk - 1) / chunk);
  };
  Plan p{0, 128, 1, 128};
  if (b.prefix_len) cut(b.prefix_len, (int64_t)b.rows * G, 1, p.sp, p.cp);
  cut(b.max_len, (int64_t)b.max_rows * G, b.B, p.so, p.co);
  return p;
}
size_t ml_bytes(const Plan& p, const dsgx_kv_batch& b, int Hq) { return align256((size_t)(p.sp + p.so) * b.rows * Hq * sizeof(float2)); }

template <int D, bool F8>
int launch_part(const AttnArgs& a, int prefix, hipStream_t st) {
  const int64_t cols = (int64_t)(prefix ? a.b.rows : a.b.max_rows) * a.G;
  const Kind k = kind_of(cols);
  const size_t lds = k == kNarrow ? (4 * 16 * (D + 4) + 128) * 4 : 4 * Wide<D, F8, 32>::kTile;
  auto kern = k == kNarrow ? k_attn_narrow<D, F8> : k == kWide16 ? k_attn_wide<D, F8, 16> : k_attn_wide<D, F8, 32>;
  if (int rc = allow_dynamic_lds((const void*)kern, lds)) return rc;
  const dim3 grid((prefix ? a.p.sp : a.p.so) * a.c.Hkv, (unsigned)std::min<int64_t>(65535, (cols + cols_of(k) - 1) / cols_of(k)), prefix ? 1 : a.b.B);
  hipLaunchKernelGGL(kern, grid, dim3(256), lds, st, a, prefix);
  DSGX_HIP(hipGetLastError());
  return DSGX_OK;
}
template <int D, bool F8>
int launch(const AttnArgs& a, hipStream_t st) {
  if (a.p.sp)
    if (int rc = launch_part<D, F8>(a, 1, st)) return rc;
  if (int rc = launch_part<D, F8>(a, 0, st)) return rc;
  if (a.p.sp + a.p.so > 1) {
    hipLaunchKernelGGL(k_combine<D>, dim3(a.b.rows, (a.Hq + 3) / 4), dim3(256), 0, st, a);
    DSGX_HIP(hipGetLastError());
  }
  return DSGX_OK;
}

int check(const dsgx_kv_cache* c, const dsgx_kv_batch* b, int Hq) {
  if (int rc = check_cache("attn", c)) return rc;
  if (int rc = check_batch("attn", c, b)) return rc;
  if (Hq < 1 || Hq % c->Hkv || Hq > 65536) return fail(DSGX_EINVAL, "attn: %d query heads over %d", Hq, c->Hkv);
  if (c->tok_stride > (1 << 24)) return fail(DSGX_EINVAL, "attn: tokens %lld values apart (2^24 at most)", (long long)c->tok_stride);
  if ((int64_t)b->rows * Hq > (1 << 30)) return fail(DSGX_EINVAL, "attn: %d rows of %d heads", b->rows, Hq);
  return DSGX_OK;
}

}  // namespace
}  // namespace dsgx

using namespace dsgx;

extern "C" size_t dsgx_attn_ws_bytes(const dsgx_kv_cache* cache, const dsgx_kv_batch* batch, int Hq) {
  if (check(cache, batch, Hq)) return 0;
  const Plan p = make_plan(*cache, *batch, Hq);
  return ml_bytes(p, *batch, Hq) + align256((size_t)(p.sp + p.so) * batch->rows * Hq * cache->D * 4) + 256;
}

extern "C" int dsgx_attn(const dsgx_kv_cache* cache, const dsgx_kv_batch* batch, const uint16_t* q, int64_t ldq, int Hq, float scale, uint16_t* out, int64_t ldo,
                         float* lse, void* ws, void* stream) {
  if (int rc = check(cache, batch, Hq)) return rc;
  if (!q || !out || !ws) return fail(DSGX_EINVAL, "attn: null queries, output or workspace");
  if (!std::isfinite(scale)) return fail(DSGX_EINVAL, "attn: a scale of %g", (double)scale);
  const int64_t vals = (int64_t)Hq * cache->D;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)ws) & 15 || ldq % 8 || ldo % 8 || ldq < vals || ldo < vals)
    return fail(DSGX_EINVAL, "attn: rows %lld, %lld apart (multiples of 8, %lld at least; 16-byte aligned)", (long long)ldq, (long long)ldo, (long long)vals);
  if (batch->rows == 0) return DSGX_OK;
  AttnArgs a{};
  a.c = *cache, a.b = *batch, a.p = make_plan(*cache, *batch, Hq);
  a.q = q, a.out = out, a.lse = lse, a.ldq = ldq, a.ldo = ldo, a.Hq = Hq, a.G = Hq / cache->Hkv, a.page_shift = __builtin_ctz((unsigned)cache->page);
  a.scale2 = scale == 0.f ? 1.f : std::fabs(scale) * kLog2e, a.q_flip = scale < 0.f ? 0x80008000u : 0u, a.q_keep = scale == 0.f ? 0u : 0xFFFFFFFFu;
  a.ml = static_cast<float2*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + ml_bytes(a.p, *batch, Hq));
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool f8 = cache->fmt == DSGX_KV_E4M3;
  switch (cache->D) {
    case 64: return f8 ? launch<64, true>(a, st) : launch<64, false>(a, st);
    case 128: return f8 ? launch<128, true>(a, st) : launch<128, false>(a, st);
    default: return f8 ? launch<256, true>(a, st) : launch<256, false>(a, st);
  }
}
