// Attention of a decode step's rows over the paged cache (include/dsgx.h): a shared prefix and every sequence's own tokens.
//
// One pass over the tokens with the running maximum and sum of the softmax (in powers of two). The G = Hq / Hkv query heads that
// share a head of keys and values are G columns of one matrix product, times the rows that attend over the same tokens: a
// sequence's rows over its own tokens, all rows over the prefix. The tokens are cut into ranges, a workgroup each; what the ranges
// leave (maximum, sum, unnormalised output in f32) k_combine joins.
#include <algorithm>

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
  float scale2;  // scale * log2 e
};

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

  struct Block {
    u32x4_t k[2][KW];
    uint32_t v[8][VW];
  };

  __device__ __forceinline__ void begin() {
    m = -__builtin_inff(), l = 0.f;
#pragma unroll
    for (int i = 0; i < VL; ++i) o[i] = v4f_t{0.f, 0.f, 0.f, 0.f};
  }
  // row: the lane's query (lane % 16), D values; null: none
  __device__ __forceinline__ void load_q(const uint16_t* row, int g) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = F8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      u32x4_t w = {0, 0, 0, 0};
      if (row) w = *reinterpret_cast<const DSGX_GLOBAL u32x4_t*>((uintptr_t)(row + d));
      q[s] = __builtin_bit_cast(v8bf_t, w);
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
  // Whether a V word holds an infinity or a NaN
  __device__ __forceinline__ static bool wild(uint32_t w) {
    if (F8) {
      const uint32_t n = w & 0x7F7F7F7Fu;
      return ((n + 0x01010101u) & 0x80808080u) != 0;  // a byte of 0x7F
    }
    return (w & 0x7F80u) == 0x7F80u || (w & 0x7F800000u) == 0x7F800000u;
  }

  // Thirty-two tokens, t0 the first. lim: the lane's query sees the tokens below it. there[a]: tile a's page exists. all: no lane has
  // anything masked here (wave-uniform). seen: some query's tokens end at `seen` at most; step rows' limits run from lim_lo to seen.
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
    for (int i = 0; i < 8; ++i) e[i] = __fmul_rn(s[i / 4][i % 4], s2);
    bool odd = false;
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
        const bool there = i < 4 ? there0 : there1;
        if (!there || t >= lim) e[i] = -__builtin_inff();
        // what no query sees is zero for the product (0 * NaN); what some do and some do not is looked at below
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if (!there || t >= seen) x.v[i][w] = 0u;
          odd |= t >= lim_lo && wild(x.v[i][w]);
        }
      }
    }
    float mx = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
    mx = fmaxf(m, groups_max(mx));
    const float base = mx == -__builtin_inff() ? 0.f : mx;
    const float alpha = exp2_hw(m - base);
    m = mx;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = exp2_hw(e[i] - base), sum += e[i];
    l = fmaf(l, alpha, sum);
    const u32x4_t pw = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])};
    const v8bf_t p = __builtin_bit_cast(v8bf_t, pw);
#pragma unroll
    for (int i = 0; i < VL; ++i) o[i] *= alpha;
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) == 0, 1)) {
#pragma unroll
      for (int i = 0; i < VL; i += 2) {
        v8bf_t a, b;
        v_operands(x.v, i, a, b);
        o[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p, o[i], 0, 0, 0);
        o[i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, p, o[i + 1], 0, 0, 0);
      }
    } else {
      // A token that one row of the step sees and an earlier one does not holds an infinity or a NaN: the rows one limit at a time,
      // from the last to the first, each with the tokens past its limit zeroed
      for (int lm = seen; lm >= lim_lo; --lm) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (t0 + 16 * (i / 4) + 4 * g + i % 4 >= lm) {
#pragma unroll
            for (int w = 0; w < VW; ++w) x.v[i][w] = 0u;
          }
        const bool mine = lim == lm;
#pragma unroll
        for (int i = 0; i < VL; i += 2) {
          v8bf_t a, b;
          v_operands(x.v, i, a, b);
          const v4f_t n0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p, o[i], 0, 0, 0), n1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, p, o[i + 1], 0, 0, 0);
#pragma unroll
          for (int j = 0; j < 4; ++j) o[i][j] = mine ? n0[j] : o[i][j], o[i + 1][j] = mine ? n1[j] : o[i + 1][j];
        }
      }
    }
  }
};

// The rows that attend over one set of tokens, as query columns: column x is head h G + x % G of row first + x / G
struct Columns {
  int first, count;  // rows; columns in all
};

template <int D, bool F8>
__global__ void __launch_bounds__(256) k_attn_narrow(AttnArgs a, int prefix) {
  using N = Narrow<D, F8>;
  constexpr int VL = N::VL, LD = D + 4;
  extern __shared__ float lds[];  // [4][16][LD] outputs, then [4][16] maxima and sums
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), g = lane >> 4, col = lane & 15;
  const int h = blockIdx.x % a.c.Hkv, split = blockIdx.x / a.c.Hkv, G = a.G;
  int first = 0, rows = a.b.rows, len = a.b.prefix_len;
  const int32_t* tab = a.b.prefix;
  if (!prefix) {
    const int b = blockIdx.z;
    first = a.b.cu_rows ? a.b.cu_rows[b] : b * a.b.max_rows;
    const int end = a.b.cu_rows ? a.b.cu_rows[b + 1] : first + a.b.max_rows;
    if (first < 0 || end <= first || end > a.b.rows) return;
    rows = end - first;
    const int cap = a.b.table_ld << a.page_shift;
    len = a.b.lens[b];
    len = len < 0 ? 0 : len > cap ? cap : len;
    tab = a.b.table + (size_t)b * a.b.table_ld;
  }
  const int chunk = prefix ? a.p.cp : a.p.co, splits = prefix ? a.p.sp : a.p.so;
  const int lo = split * chunk, hi = split == splits - 1 ? len : min(len, lo + chunk);
  if (lo >= hi && split > 0) return;  // (range 0 is always written)
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
    n.load_q(live ? a.q + (size_t)(first + row) * a.ldq + (size_t)head * D : nullptr, g);
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

    // the four waves' halves of the answer joined
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

Plan make_plan(const dsgx_kv_cache& c, const dsgx_kv_batch& b, int Hq) {
  const int G = Hq / c.Hkv, cus = num_cus_cached();
  auto cut = [&](int64_t len, int64_t tiles, int& n, int& chunk) {  // tiles: workgroups a range
    const int64_t want = std::max<int64_t>(1, 4 * (int64_t)cus / std::max<int64_t>(1, tiles));
    chunk = std::max(256, round_up((len + want - 1) / want, 128));
    n = (int)std::max<int64_t>(1, (len + chunk - 1) / chunk);
  };
  Plan p{0, 128, 1, 128};
  if (b.prefix_len) cut(b.prefix_len, (int64_t)c.Hkv * (((int64_t)b.rows * G + 15) / 16), p.sp, p.cp);
  cut(b.max_len, (int64_t)c.Hkv * b.B * (((int64_t)b.max_rows * G + 15) / 16), p.so, p.co);
  return p;
}
size_t ml_bytes(const Plan& p, const dsgx_kv_batch& b, int Hq) { return align256((size_t)(p.sp + p.so) * b.rows * Hq * sizeof(float2)); }

template <int D, bool F8>
int launch(const AttnArgs& a, hipStream_t st) {
  const size_t lds = (4 * 16 * (D + 4) + 128) * 4;
  auto kern = k_attn_narrow<D, F8>;
  if (int rc = allow_dynamic_lds((const void*)kern, lds)) return rc;
  auto tiles = [&](int64_t rows) { return (unsigned)std::min<int64_t>(65535, (rows * a.G + 15) / 16); };
  if (a.p.sp) {
    hipLaunchKernelGGL(kern, dim3(a.p.sp * a.c.Hkv, tiles(a.b.rows)), dim3(256), lds, st, a, 1);
    DSGX_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(kern, dim3(a.p.so * a.c.Hkv, tiles(a.b.max_rows), a.b.B), dim3(256), lds, st, a, 0);
  DSGX_HIP(hipGetLastError());
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
  const int64_t vals = (int64_t)Hq * cache->D;
  if (((uintptr_t)q | (uintptr_t)out | (uintptr_t)ws) & 15 || ldq % 8 || ldo % 8 || ldq < vals || ldo < vals)
    return fail(DSGX_EINVAL, "attn: rows %lld, %lld apart (multiples of 8, %lld at least; 16-byte aligned)", (long long)ldq, (long long)ldo, (long long)vals);
  if (batch->rows == 0) return DSGX_OK;
  AttnArgs a{};
  a.c = *cache, a.b = *batch, a.p = make_plan(*cache, *batch, Hq);
  a.q = q, a.out = out, a.lse = lse, a.ldq = ldq, a.ldo = ldo, a.Hq = Hq, a.G = Hq / cache->Hkv, a.page_shift = __builtin_ctz((unsigned)cache->page);
  a.scale2 = scale * kLog2e;
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
