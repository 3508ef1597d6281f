// Verification of drafted tokens against the target's distribution from given random numbers (include/dsgx.h). The result is whole
// numbers that lie next to borders (a cumulative sum over the vocabulary against a random threshold), so all sums and probabilities are
// f64: with f32 exponentials about one draw in a hundred of a flat distribution over 10^5 tokens would come out one token off. (One sum that no
// draw depends on is the exception, see k_stats.)
//
// Two launches: k_stats reads every row of logits once and leaves, for each piece of it, the maximum, the sum of exp and the lowest
// id of the maximum, and for the row what its draft's target and drafter are; k_weights judges its sequence's drafts (every workgroup for
// itself: a few KB out of L2), sums the weights of its piece of the one row that the next token comes from, and the last workgroup
// of a sequence draws. Probabilities need no k_stats.
//
// A piece is as many chunks of 4096 ids as let the whole launch be on the card at once (pieces_of): the chain from a workgroup's first load to
// its last takes about 7 us in k_weights, and a second round of workgroups would wait for it again.
// Measured, both launches: 16 x 5 rows of 131072 f32 logits 27.8 us (13.3 + 14.5, 42 + 8.4 + 8.4 MB), 224 rows of 100003 in bf16 31.9 (13.7 + 18.2), 32 x 4 of 65537 probabilities 12.4, 2 rows of 32768 14.0.
#include "abi_internal.h"
#include "common.cuh"

#include <algorithm>

namespace dsgx {
namespace {

constexpr int kChunk = 4096, kThreads = 512, kWaves = kThreads / kWave, kPer = kChunk / kThreads;  // k_weights
constexpr int kStatRoom = 256 * 8, kRoom = 256;  // workgroups of either kernel on the card's 256 CUs at once; see pieces_of
constexpr int kMostPieces = 16;  // chunks a piece of k_weights
constexpr int kStatChunk = kChunk, kStatThreads = 256, kStatWaves = kStatThreads / kWave, kStatPer = kStatChunk / kStatThreads;

constexpr int kTable = 128;  // entries of 2^(k / kTable)

struct Stat {  // of one piece of one row; also of a whole row
  double sum;  // sum of exp((x - max) / T); T <= 0: 1, or NaN if the chunk holds one
  float max;
  int arg;
};
struct Judged {  // of one sequence: the row that its next token comes from
  double scale;  // p = exp((x - max) / T) * scale
  float max;
  int end, last, arg;
};
struct Sums {
  double rest, p;  // of max(p - q, 0) and of p over a chunk
};
struct Draft {  // of one row: its draft's logit and the drafter's probability of it
  float x, q;
};
struct VerifyArgs {
  dsgx_verify_in in;
  int nc;          // chunks of a row
  int ss, ns;      // k_stats: chunks a piece, pieces a row
  int sw;          // k_weights: chunks a piece
  Stat* stat;      // [rows][ns]
  Draft* drafts;   // [rows]
  Sums* sums;      // [B][nc]
  int* count;      // [B]: chunks done
  int32_t *tokens, *accepted;
};

typedef float f32x4u_t __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4u_t __attribute__((ext_vector_type(4), aligned(2)));

// U consecutive values of a row from v on (KIND 1: 8 bf16, else 4 f32; rows may begin at any value's address); `none` past V
template <int KIND>
constexpr int kUnit = KIND == 1 ? 8 : 4;
template <int KIND>
__device__ __forceinline__ void load_unit(const void* row, int v, int V, float none, float (&x)[kUnit<KIND>]) {
  constexpr int U = kUnit<KIND>;
  if (KIND == 1) {
    const uint16_t* p = static_cast<const uint16_t*>(row);
    if (v + U <= V) {
      const u32x4u_t w = *reinterpret_cast<const u32x4u_t*>(p + v);
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = v + i < V ? bf16_bits_to_f32(p[v + i]) : none;
    }
  } else {
    const float* p = static_cast<const float*>(row);
    if (v + U <= V) {
      const f32x4u_t w = *reinterpret_cast<const f32x4u_t*>(p + v);
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = w[i];
    } else {
#pragma unroll
      for (int i = 0; i < U; ++i) x[i] = v + i < V ? p[v + i] : none;
    }
  }
}
template <int KIND>
__device__ __forceinline__ const void* row_of(const void* base, int64_t ld, int r) {
  return static_cast<const uint8_t*>(base) + (KIND == 1 ? 2 : 4) * (ld * (int64_t)r);
}

// exp((x - max) / T) of f32 values in f64, for x <= max; a NaN gives NaN, an x that lies 700 T or more below the maximum e^-700 (10^-304,
// which no sum notices) or with ZERO 0. With z = 128 (x - max) / (T ln 2) = N + f, N whole (rounded by adding 1.5 * 2^52), |f| <= 1/2:
// 2^((N mod 128) / 128) out of a table in LDS, times the power series of 2^(f / 128) up to f^2, times 2^(N div 128) on the exponent's bits.
// With h = ln 2 / 256 the largest exponent, its h^3 / 6 is brought to h^3 / 24 = 8 * 10^-10, as often above as below, by giving the linear term
// the 3/4 h^2 / 6 of e^r's r^3 (r^3 is nearest 3/4 h^2 r): a draw among 10^5 ids comes out one id off once in some million. Eight
// f64 instructions a value, and the accumulation's ninth, at eight clocks a wave each, bound k_stats; with terms up to r^11 there were
// eighteen. The library's exp takes about fifty.
__constant__ double kExp2[kTable] = {
    0x1.0000000000000p+0, 0x1.0163da9fb3335p+0, 0x1.02c9a3e778061p+0, 0x1.04315e86e7f85p+0,
    0x1.059b0d3158574p+0, 0x1.0706b29ddf6dep+0, 0x1.0874518759bc8p+0, 0x1.09e3ecac6f383p+0,
    0x1.0b5586cf9890fp+0, 0x1.0cc922b7247f7p+0, 0x1.0e3ec32d3d1a2p+0, 0x1.0fb66affed31bp+0,
    0x1.11301d0125b51p+0, 0x1.12abdc06c31ccp+0, 0x1.1429aaea92de0p+0, 0x1.15a98c8a58e51p+0,
    0x1.172b83c7d517bp+0, 0x1.18af9388c8deap+0, 0x1.1a35beb6fcb75p+0, 0x1.1bbe084045cd4p+0,
    0x1.1d4873168b9aap+0, 0x1.1ed5022fcd91dp+0, 0x1.2063b88628cd6p+0, 0x1.21f49917ddc96p+0,
    0x1.2387a6e756238p+0, 0x1.251ce4fb2a63fp+0, 0x1.26b4565e27cddp+0, 0x1.284dfe1f56381p+0,
    0x1.29e9df51fdee1p+0, 0x1.2b87fd0dad990p+0, 0x1.2d285a6e4030bp+0, 0x1.2ecafa93e2f56p+0,
    0x1.306fe0a31b715p+0, 0x1.32170fc4cd831p+0, 0x1.33c08b26416ffp+0, 0x1.356c55f929ff1p+0,
    0x1.371a7373aa9cbp+0, 0x1.38cae6d05d866p+0, 0x1.3a7db34e59ff7p+0, 0x1.3c32dc313a8e5p+0,
    0x1.3dea64c123422p+0, 0x1.3fa4504ac801cp+0, 0x1.4160a21f72e2ap+0, 0x1.431f5d950a897p+0,
    0x1.44e086061892dp+0, 0x1.46a41ed1d0057p+0, 0x1.486a2b5c13cd0p+0, 0x1.4a32af0d7d3dep+0,
    0x1.4bfdad5362a27p+0, 0x1.4dcb299fddd0dp+0, 0x1.4f9b2769d2ca7p+0, 0x1.516daa2cf6642p+0,
    0x1.5342b569d4f82p+0, 0x1.551a4ca5d920fp+0, 0x1.56f4736b527dap+0, 0x1.58d12d497c7fdp+0,
    0x1.5ab07dd485429p+0, 0x1.5c9268a5946b7p+0, 0x1.5e76f15ad2148p+0, 0x1.605e1b976dc09p+0,
    0x1.6247eb03a5585p+0, 0x1.6434634ccc320p+0, 0x1.6623882552225p+0, 0x1.68155d44ca973p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6c012750bdabfp+0, 0x1.6dfb23c651a2fp+0, 0x1.6ff7df9519484p+0,
    0x1.71f75e8ec5f74p+0, 0x1.73f9a48a58174p+0, 0x1.75feb564267c9p+0, 0x1.780694fde5d3fp+0,
    0x1.7a11473eb0187p+0, 0x1.7c1ed0130c132p+0, 0x1.7e2f336cf4e62p+0, 0x1.80427543e1a12p+0,
    0x1.82589994cce13p+0, 0x1.8471a4623c7adp+0, 0x1.868d99b4492edp+0, 0x1.88ac7d98a6699p+0,
    0x1.8ace5422aa0dbp+0, 0x1.8cf3216b5448cp+0, 0x1.8f1ae99157736p+0, 0x1.9145b0b91ffc6p+0,
    0x1.93737b0cdc5e5p+0, 0x1.95a44cbc8520fp+0, 0x1.97d829fde4e50p+0, 0x1.9a0f170ca07bap+0,
    0x1.9c49182a3f090p+0, 0x1.9e86319e32323p+0, 0x1.a0c667b5de565p+0, 0x1.a309bec4a2d33p+0,
    0x1.a5503b23e255dp+0, 0x1.a799e1330b358p+0, 0x1.a9e6b5579fdbfp+0, 0x1.ac36bbfd3f37ap+0,
    0x1.ae89f995ad3adp+0, 0x1.b0e07298db666p+0, 0x1.b33a2b84f15fbp+0, 0x1.b59728de5593ap+0,
    0x1.b7f76f2fb5e47p+0, 0x1.ba5b030a1064ap+0, 0x1.bcc1e904bc1d2p+0, 0x1.bf2c25bd71e09p+0,
    0x1.c199bdd85529cp+0, 0x1.c40ab5fffd07ap+0, 0x1.c67f12e57d14bp+0, 0x1.c8f6d9406e7b5p+0,
    0x1.cb720dcef9069p+0, 0x1.cdf0b555dc3fap+0, 0x1.d072d4a07897cp+0, 0x1.d2f87080d89f2p+0,
    0x1.d5818dcfba487p+0, 0x1.d80e316c98398p+0, 0x1.da9e603db3285p+0, 0x1.dd321f301b460p+0,
    0x1.dfc97337b9b5fp+0, 0x1.e264614f5a129p+0, 0x1.e502ee78b3ff6p+0, 0x1.e7a51fbc74c83p+0,
    0x1.ea4afa2a490dap+0, 0x1.ecf482d8e67f1p+0, 0x1.efa1bee615a27p+0, 0x1.f252b376bba97p+0,
    0x1.f50765b6e4540p+0, 0x1.f7bfdad9cbe14p+0, 0x1.fa7c1819e90d8p+0, 0x1.fd3c22b8f71f1p+0,
};
struct Exp {
  double itl, max;    // kTable / (T ln 2)
  float lo, rough;    // max - 700 T; 1 / (T ln 2)
  const double* tab;  // kExp2 in LDS
};
// lo is rounded to max's bits: no further from it than the exponent reaches, and below it. Where 700 T is less than half a step of max, what
// is below max is 0 and its distance stands for 700.
__device__ __forceinline__ Exp exp_of(float max, float T, double it, const double* tab) {
  float lo = max - 700.f * T;
  const float up = __uint_as_float(__float_as_uint(lo) + (lo > 0.f ? 1u : -1u)), below = __uint_as_float(max > 0.f ? __float_as_uint(max) - 1u : __float_as_uint(max) + 1u);
  if (((double)max - (double)lo) * it > 705.0) lo = up;
  if (lo == max && max != __builtin_inff()) lo = below, it = 700.0 / ((double)max - (double)lo);
  const double l2 = it * 1.4426950408889634074;
  return Exp{l2 * kTable, (double)max, lo, l2 > 3e38 ? 3e38f : (float)l2, tab};
}
template <bool ZERO>
__device__ __forceinline__ double exp_at(const Exp& e, float x) {
  constexpr double h = 0.69314718055994530942 / (2 * kTable), a1 = 2 * h * (1.0 + h * h / 8), a2 = 2 * h * h;
  const float xc = __builtin_elementwise_maximum(x, e.lo);  // (a NaN stays)
  const double y = (double)xc - e.max, t = fma(y, e.itl, 0x1.8p52), f = fma(y, e.itl, 0x1.8p52 - t);
  const uint32_t N = (uint32_t)__builtin_bit_cast(uint64_t, t);
  const double c = e.tab[N & (kTable - 1)], s = fma(c, f * fma(f, a2, a1), c);
  // s lies in [0.99, 2), N div kTable in [-1018, 0]
  const uint64_t b = __builtin_bit_cast(uint64_t, s);
  const uint32_t hi = (uint32_t)(b >> 32) + ((N & ~(uint32_t)(kTable - 1)) << 13);
  const uint64_t v = (uint64_t)hi << 32 | (uint32_t)b;
  return __builtin_bit_cast(double, ZERO && x <= e.lo ? (uint64_t)0 : v);
}

// sums and maxima over a wave by DPP steps within the rows of sixteen lanes and half swaps, in every lane
template <int CTRL>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)dpp_mov<CTRL>((uint32_t)(b >> 32)) << 32 | dpp_mov<CTRL>((uint32_t)b));
}
__device__ __forceinline__ double wave_sum_f64(double v) {
  v += dpp_f64<0xB1>(v);
  v += dpp_f64<0x4E>(v);
  v += dpp_f64<0x141>(v);
  v += dpp_f64<0x140>(v);
  uint64_t b = __builtin_bit_cast(uint64_t, v);
  auto lo = __builtin_amdgcn_permlane16_swap((uint32_t)b, (uint32_t)b, false, false), hi = __builtin_amdgcn_permlane16_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  v = __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
  b = __builtin_bit_cast(uint64_t, v);
  lo = __builtin_amdgcn_permlane32_swap((uint32_t)b, (uint32_t)b, false, false), hi = __builtin_amdgcn_permlane32_swap((uint32_t)(b >> 32), (uint32_t)(b >> 32), false, false);
  return __builtin_bit_cast(double, (uint64_t)hi[0] << 32 | lo[0]) + __builtin_bit_cast(double, (uint64_t)hi[1] << 32 | lo[1]);
}
// inclusive sums over the lanes (shifts within the rows, the rows' last lanes handed on)
template <int CTRL, int ROWS>
__device__ __forceinline__ double scan_step_f64(double v) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)b, CTRL, ROWS, 0xF, false), hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(b >> 32), CTRL, ROWS, 0xF, false);
  return v + __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan_f64(double v) {
  v = scan_step_f64<0x111, 0xF>(v);
  v = scan_step_f64<0x112, 0xF>(v);
  v = scan_step_f64<0x114, 0xF>(v);
  v = scan_step_f64<0x118, 0xF>(v);
  v = scan_step_f64<0x142, 0xA>(v);
  return scan_step_f64<0x143, 0xC>(v);
}
__device__ __forceinline__ double readlane_f64(double v, int l) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), l) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l));
}
__device__ __forceinline__ double sum_waves(const double* red) {
  double v = red[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v += red[w];
  return v;
}
// the larger maximum, of equals the lower id
__device__ __forceinline__ void take_max(float& m, int& arg, float om, int oa) {
  const bool t = om > m || (om == m && oa < arg);
  m = t ? om : m, arg = t ? oa : arg;
}
__device__ __forceinline__ void wave_take_max(float& m, int& arg) {
  take_max(m, arg, __uint_as_float(dpp_mov<0xB1>(__float_as_uint(m))), (int)dpp_mov<0xB1>((uint32_t)arg));
  take_max(m, arg, __uint_as_float(dpp_mov<0x4E>(__float_as_uint(m))), (int)dpp_mov<0x4E>((uint32_t)arg));
  take_max(m, arg, __uint_as_float(dpp_mov<0x141>(__float_as_uint(m))), (int)dpp_mov<0x141>((uint32_t)arg));
  take_max(m, arg, __uint_as_float(dpp_mov<0x140>(__float_as_uint(m))), (int)dpp_mov<0x140>((uint32_t)arg));
  auto f = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false), i = __builtin_amdgcn_permlane16_swap((uint32_t)arg, (uint32_t)arg, false, false);
  m = __uint_as_float(f[0]), arg = (int)i[0];
  take_max(m, arg, __uint_as_float(f[1]), (int)i[1]);
  f = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false), i = __builtin_amdgcn_permlane32_swap((uint32_t)arg, (uint32_t)arg, false, false);
  m = __uint_as_float(f[0]), arg = (int)i[0];
  take_max(m, arg, __uint_as_float(f[1]), (int)i[1]);
}

// a value at an address that is the same in the whole wave, by a scalar load: waiting for it waits for no vector load
template <class T>
__device__ __forceinline__ T scalar_at(const T* p) {
  return *(const __attribute__((address_space(4))) T*)(uintptr_t)p;
}
// the sequence's rows; none if the bounds are out of order
__device__ __forceinline__ bool rows_of(const dsgx_verify_in& in, int b, int& r0, int& r1) {
  r0 = in.cu_rows ? scalar_at(in.cu_rows + b) : b * in.max_rows;
  r1 = in.cu_rows ? scalar_at(in.cu_rows + b + 1) : r0 + in.max_rows;
  return r0 >= 0 && r0 < r1 && r1 <= in.rows;
}
// the sequence of row r, and whether r is its last row; from, to: the lane's cu_rows of the first 64 sequences
__device__ __forceinline__ int seq_of(const dsgx_verify_in& in, int r, int lane, int from, int to, bool& last) {
  if (!in.cu_rows) {
    last = r % in.max_rows == in.max_rows - 1;
    return r / in.max_rows;
  }
  for (int j0 = 0; j0 < in.B; j0 += kWave) {
    const int j = j0 + lane;
    if (j0) from = in.cu_rows[j < in.B ? j : 0], to = in.cu_rows[j < in.B ? j + 1 : 0];
    const uint64_t hit = __builtin_amdgcn_ballot_w64(j < in.B && from <= r && r < to);
    if (hit) {
      last = __builtin_amdgcn_readlane(to, __builtin_ctzll(hit)) == r + 1;
      return j0 + __builtin_ctzll(hit);
    }
  }
  return -1;
}
// of T past 10^35 (infinity among them) every logit in use is the same: the range below the maximum stays finite
__device__ __forceinline__ float temp_of(const dsgx_verify_in& in, int b) {
  const float T = in.temp ? scalar_at(in.temp + b) : 1.f;
  return T > 1e35f ? 1e35f : T;
}
template <int KIND>
__device__ __forceinline__ Draft draft_of(const dsgx_verify_in& in, int r, int d) {
  const void* row = row_of<KIND>(in.target, in.ldt, r);
  return Draft{KIND == 1 ? bf16_bits_to_f32(static_cast<const uint16_t*>(row)[d]) : static_cast<const float*>(row)[d], in.q ? in.q[in.ldq * (int64_t)r + d] : 1.f};
}

// neither the compiler's passes nor its scheduler move a load across
__device__ __forceinline__ void loads_stay() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// FINE: the row's probabilities are compared with a drafter's id by id, and an error of the sum moves the borders of a draw: f64. Else the sum
// stands behind the draft's own probability alone (a draw from p itself does not need it), and exponentials in f32 do, added in f32 by
// sixteens. A term 2^-z of the largest is off by z 2^-23 (difference, scaling) and 2^-23 (the exponential), sixteen of them by 2^-22, all of
// random sign: with the sum's bulk at z <= 6, 10^-6 if every sign were the same. That decides otherwise than f64 for one draft in a million
// at most: 224 bf16 rows of 100003 take 13.7 us instead of 22.2.
template <int KIND, bool FINE>
__global__ void __launch_bounds__(kStatThreads) k_stats(VerifyArgs a) {
  constexpr int U = kUnit<KIND>, NU = kStatPer / U;
  const dsgx_verify_in& in = a.in;
  __shared__ double red[kStatWaves], tab[kTable];
  __shared__ float rm[kStatWaves];
  __shared__ int ra[kStatWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.y, c0 = blockIdx.x * a.ss, c1 = min(c0 + a.ss, a.nc);
  const void* row = row_of<KIND>(in.target, in.ldt, r);
  float x[NU][U], next[NU][U];  // (on their way before anything is waited for)
  auto load = [&](float (&to)[NU][U], int c) {
#pragma unroll
    for (int k = 0; k < NU; ++k) load_unit<KIND>(row, c * kStatChunk + (k * kStatThreads + (int)threadIdx.x) * U, in.V, -__builtin_inff(), to[k]);
  };
  // Everything is asked for before anything is waited for, what is needed first is asked for first: the launch is one round of workgroups,
  // nothing else hides a wait
  const int j0 = lane < in.B ? lane : 0, from = in.cu_rows ? in.cu_rows[j0] : 0, to = in.cu_rows ? in.cu_rows[j0 + 1] : 0;
  const double entry = kExp2[threadIdx.x & (kTable - 1)];
  loads_stay();
  load(x, c0);
  loads_stay();
  bool tail;
  const int b = seq_of(in, r, lane, from, to, tail);
  if (b < 0 || b >= in.B) return;
  const int d = tail ? -1 : scalar_at(in.draft + r);
  const float T = temp_of(in, b);
  const bool greedy = !(T > 0.f || T != T), mine = d >= 0 && d < in.V && d / kStatChunk >= c0 && d / kStatChunk < c1;
  const double it = 1.0 / (double)T;
  const Draft draft = draft_of<KIND>(in, r, mine ? d : c0 * kStatChunk);
  if (threadIdx.x < kTable) tab[threadIdx.x] = entry;
  __syncthreads();
  // the wave's maximum so far (greedy: the lane's, with its id) and the lane's sum against it
  float m = -__builtin_inff();
  int arg = 0x7FFFFFFF;
  double s = 0.0;
  Exp e{};
  auto chunk = [&](const float (&x)[NU][U], int c) {
    float mx = -__builtin_inff();
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int i = 0; i < U; ++i) mx = fmaxf(mx, x[k][i]);
    if (!greedy) {
      mx = wave_max_f32(mx);
      if (mx > m) {
        e = exp_of(mx, T, it, tab);
        s *= exp_at<true>(e, m), m = mx;
      }
    } else if (mx > m) {
      m = mx;
#pragma unroll
      for (int k = NU - 1; k >= 0; --k)
#pragma unroll
        for (int i = U - 1; i >= 0; --i) arg = x[k][i] == m ? c * kStatChunk + (k * kStatThreads + (int)threadIdx.x) * U + i : arg;
    }
    if (!greedy && m != -__builtin_inff() && !FINE) {
      float f = 0.f;
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < U; ++i) f += __builtin_amdgcn_exp2f((x[k][i] - m) * e.rough);
      s += (double)f;
    } else if (!greedy && m != -__builtin_inff()) {
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < U; ++i) s += exp_at<false>(e, x[k][i]);
    } else {  // whether there is a NaN (nothing but -inf has no maximum to subtract, and the sum 0)
      float f = 0.f;
#pragma unroll
      for (int k = 0; k < NU; ++k)
#pragma unroll
        for (int i = 0; i < U; ++i) f = x[k][i] == x[k][i] ? f : x[k][i];
      s += (double)f;
    }
  };
  for (int c = c0; c < c1; c += 2) {
    if (c + 1 < c1) load(next, c + 1);
    chunk(x, c);
    if (c + 1 >= c1) break;
    if (c + 2 < c1) load(x, c + 2);
    chunk(next, c + 1);
  }
  s = wave_sum_f64(s);
  if (greedy) wave_take_max(m, arg);
  if (lane == 0) rm[wave] = m, ra[wave] = arg, red[wave] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kStatWaves; ++w) take_max(m, arg, rm[w], ra[w]);
    e = exp_of(m, T, it, tab);
    double sum = greedy ? 1.0 : 0.0;  // (a greedy row's is 1, or NaN)
#pragma unroll
    for (int w = 0; w < kStatWaves; ++w) sum += greedy || red[w] == 0.0 ? red[w] : red[w] * exp_at<true>(e, rm[w]);
    a.stat[(size_t)r * a.ns + blockIdx.x] = Stat{sum, m, arg};
    if (mine) a.drafts[r] = draft;
  }
}

// A row's statistics out of its pieces' (the lane's own st, pieces lane, lane + 64, ..), by one wave
__device__ __forceinline__ Stat row_stat(const VerifyArgs& a, int r, float T, double it, const double* tab, int lane, Stat st) {
  float m = st.max;
  int arg = st.arg;
  const Stat* more = a.stat + (size_t)r * a.ns;
  for (int c = lane + kWave; c < a.ns; c += kWave) take_max(m, arg, more[c].max, more[c].arg);
  wave_take_max(m, arg);
  const bool greedy = !(T > 0.f || T != T);
  const Exp e = exp_of(m, T, it, tab);
  auto part = [&](const Stat& x) { return greedy ? x.sum : x.sum == 0.0 ? 0.0 : x.sum * exp_at<true>(e, x.max); };
  double s = part(st);
  for (int c = lane + kWave; c < a.ns; c += kWave) s += part(more[c]);
  return Stat{wave_sum_f64(s), m, arg};
}

// p of a value: logits x, or the probability itself
template <int KIND>
__device__ __forceinline__ double prob(float x, int v, const Judged& j, const Exp& e, bool greedy) {
  if (KIND == 2) return (double)x;
  if (greedy) return v == j.arg ? j.scale : 0.0 * j.scale;  // (a row with a NaN has a NaN scale)
  return exp_at<true>(e, x) * j.scale;
}
__device__ __forceinline__ double rest_of(double p, double q) {
  const double d = p - q;
  const uint64_t b = __builtin_bit_cast(uint64_t, d);
  return __builtin_bit_cast(double, d <= 0.0 ? (uint64_t)0 : b);  // (a NaN stays)
}

// the drafts of sequence b up to the first that is refused, by the whole workgroup, a wave a row
template <int KIND>
__device__ __forceinline__ Judged judge(const VerifyArgs& a, int r0, int r1, float T, double it, const double* tab, int lane, int wave, Judged* sh, int* stop) {
  const dsgx_verify_in& in = a.in;
  const bool greedy = !(T > 0.f || T != T);
  for (int i0 = r0;; i0 += kWaves) {
    const int r = i0 + wave;
    bool stops = false;
    Judged j{1.0, -__builtin_inff(), r, 0, -1};
    if (r < r1) {
      // everything that can be asked for now: the pieces' statistics, the draft, its values and its random number
      Stat st{0.0, -__builtin_inff(), 0x7FFFFFFF};
      if (KIND != 2 && lane < a.ns) st = a.stat[(size_t)r * a.ns + lane];
      j.last = r == r1 - 1;
      const int d = j.last ? -1 : scalar_at(in.draft + r);
      const float u = j.last ? 0.f : scalar_at(in.u + r);
      Draft v{};
      if (KIND != 2) v = Draft{scalar_at(&a.drafts[r].x), scalar_at(&a.drafts[r].q)};
      const bool known = d >= 0 && d < in.V;
      if (KIND == 2 && known) v = draft_of<KIND>(in, r, d);
      if (KIND != 2) {
        const Stat s = row_stat(a, r, T, it, tab, lane, st);
        j.max = s.max, j.arg = s.arg;
        j.scale = greedy ? s.sum * 0.0 + 1.0 : 1.0 / s.sum;
      }
      const double p = known ? prob<KIND>(v.x, d, j, exp_of(j.max, T, it, tab), greedy) : 0.0;
      stops = j.last || !((double)u * (double)v.q < p);
    }
    __syncthreads();
    if (lane == 0) sh[wave] = j, stop[wave] = stops;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w)
      if (stop[w]) return sh[w];
  }
}

// U ids from v on of the judged row: target and drafter (what the rest is less), and their weights: rest = max(p - q, 0) (the last row: p), and p
template <int KIND>
__device__ __forceinline__ void load_weights(const VerifyArgs& a, const Judged& j, int v, float (&x)[kUnit<KIND>], float (&q)[kUnit<KIND>]) {
  constexpr int U = kUnit<KIND>;
  const dsgx_verify_in& in = a.in;
  load_unit<KIND>(row_of<KIND>(in.target, in.ldt, j.end), v, in.V, KIND == 2 ? 0.f : -__builtin_inff(), x);
  if (!j.last && in.q) {
    const float* qr = in.q + in.ldq * (int64_t)j.end;
#pragma unroll
    for (int h = 0; h < U; h += 4) {
      float t[4];
      load_unit<0>(qr, v + h, in.V, 0.f, t);
#pragma unroll
      for (int i = 0; i < 4; ++i) q[h + i] = t[i];
    }
  }
}
template <int KIND>
__device__ __forceinline__ void weights(const VerifyArgs& a, const Judged& j, const Exp& e, bool greedy, int d, int v, const float (&x)[kUnit<KIND>], const float (&q)[kUnit<KIND>],
                                        double (&rest)[kUnit<KIND>], double (&p)[kUnit<KIND>]) {
  const bool drafter = !j.last && a.in.q;
#pragma unroll
  for (int i = 0; i < kUnit<KIND>; ++i) {
    p[i] = v + i < a.in.V ? prob<KIND>(x[i], v + i, j, e, greedy) : 0.0;
    rest[i] = j.last ? p[i] : rest_of(p[i], drafter ? (double)q[i] : v + i == d ? 1.0 : 0.0);
  }
}

// values that another workgroup's thread wrote and this one may read without either side's cache in between
__device__ __forceinline__ void put_f64(double* p, double v) {
  __hip_atomic_store((DSGX_GLOBAL uint64_t*)(uintptr_t)p, __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ double get_f64(const double* p) {
  return __builtin_bit_cast(double, __hip_atomic_load((const DSGX_GLOBAL uint64_t*)(uintptr_t)p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT));
}

// Judges its sequence's drafts and sums the weights of its chunks of the row that the next token comes from; the workgroup that is the
// sequence's last to be done finds the chunk and the token in it. (The sums reach memory before the count does: they are
// device-scope stores, and the count waits for their acknowledgement. The last one sets the count back for the next call.)
template <int KIND>
__global__ void __launch_bounds__(kThreads) k_weights(VerifyArgs a) {
  constexpr int U = kUnit<KIND>, NU = kPer / U;
  __shared__ double red[kMostPieces][2 * kWaves], tab[kTable];
  __shared__ Judged sh[kWaves];
  __shared__ int stop[kWaves], is_last, hits[kWaves], lasts[kWaves];
  const dsgx_verify_in& in = a.in;
  const int tid = threadIdx.x, lane = tid & 63, wave = uni(tid >> 6), b = blockIdx.y, c0 = blockIdx.x * a.sw, n = min(a.sw, a.nc - c0);
  const float T = KIND != 2 ? temp_of(in, b) : 1.f, us = scalar_at(in.us + b);
  int r0, r1;
  if (!rows_of(in, b, r0, r1)) {
    if (c0 == 0 && tid == 0) a.accepted[b] = 0;
    return;
  }
  const bool greedy = !(T > 0.f || T != T);
  const double it = 1.0 / (double)T;
  if (KIND != 2) {
    if (tid < kTable) tab[tid] = kExp2[tid];
    __syncthreads();
  }
  const Judged j = judge<KIND>(a, r0, r1, T, it, tab, lane, wave, sh, stop);
  const Exp e = exp_of(j.max, T, it, tab);
  const int d = j.last || in.q ? -1 : in.draft[j.end];
  float x[NU][U], q[NU][U], xn[NU][U], qn[NU][U];
  auto load = [&](float (&x)[NU][U], float (&q)[NU][U], int c) {
#pragma unroll
    for (int k = 0; k < NU; ++k) load_weights<KIND>(a, j, c * kChunk + (k * kThreads + tid) * U, x[k], q[k]);
  };
  load(x, q, c0);
  for (int i = 0;; ++i) {
    const bool more = i + 1 < n;
    if (more) load(xn, qn, c0 + i + 1);
    double sr = 0.0, sp = 0.0;
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      double rest[U], p[U];
      weights<KIND>(a, j, e, greedy, d, (c0 + i) * kChunk + (k * kThreads + tid) * U, x[k], q[k], rest, p);
#pragma unroll
      for (int o = 0; o < U; ++o) sr += rest[o], sp += p[o];
    }
    sr = wave_sum_f64(sr), sp = wave_sum_f64(sp);
    if (lane == 0) red[i][wave] = sr, red[i][kWaves + wave] = sp;
    if (!more) break;
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int o = 0; o < U; ++o) x[k][o] = xn[k][o], q[k][o] = qn[k][o];
  }
  __syncthreads();
  Sums* sums = a.sums + (size_t)b * a.nc;
  if (wave == 0) {
    if (lane < n) put_f64(&sums[c0 + lane].rest, sum_waves(red[lane])), put_f64(&sums[c0 + lane].p, sum_waves(red[lane] + kWaves));
    __builtin_amdgcn_s_waitcnt(0);
  }
  if (tid == 0) {
    const int before = __hip_atomic_fetch_add((DSGX_GLOBAL int*)(uintptr_t)(a.count + b), 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    is_last = before == (int)gridDim.x - 1;
    if (is_last) __hip_atomic_store((DSGX_GLOBAL int*)(uintptr_t)(a.count + b), 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!is_last) return;

  // every wave alike: the chunks' sums, 64 at a time; the chunk is the first whose running sum passes the threshold
  auto sum_of = [&](int i, bool of_p) { return i < a.nc ? get_f64(of_p ? &sums[i].p : &sums[i].rest) : 0.0; };
  const double rest0 = sum_of(lane, false), p0 = sum_of(lane, true);
  auto total_of = [&](bool of_p) {
    double t = of_p ? p0 : rest0;
    for (int i = lane + kWave; i < a.nc; i += kWave) t += sum_of(i, of_p);
    return wave_sum_f64(t);
  };
  double total = total_of(false);
  const bool of_p = total <= 0.0;  // nothing left of the difference: from p
  if (of_p) total = total_of(true);
  const double t = (double)us * total;
  int token = -1;
  if (total > 0.0 && total < __builtin_inf()) {
    double run = 0.0, before = 0.0;
    int chunk = 0;
    for (int c0 = 0; c0 < a.nc; c0 += kWave) {
      const double w = c0 ? sum_of(c0 + lane, of_p) : of_p ? p0 : rest0, upto = run + wave_scan_f64(w);
      const uint64_t some = __builtin_amdgcn_ballot_w64(w > 0.0), past = __builtin_amdgcn_ballot_w64(w > 0.0 && upto > t);
      if (some) {
        const int l = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);  // (none passes: rounding; the last that has any)
        chunk = c0 + l, before = readlane_f64(upto, l) - readlane_f64(w, l);
      }
      if (past) break;
      run = readlane_f64(upto, 63);
    }
    // inside it: eight ids a thread, and what stands before a thread's in order
    const int v0 = chunk * kChunk + tid * kPer;
    double w[kPer], mine = 0.0;
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      double rest[U], p[U];
      load_weights<KIND>(a, j, v0 + k * U, x[k], q[k]);
      weights<KIND>(a, j, e, greedy, d, v0 + k * U, x[k], q[k], rest, p);
#pragma unroll
      for (int i = 0; i < U; ++i) w[k * U + i] = of_p ? p[i] : rest[i], mine += w[k * U + i];
    }
    const double upto = wave_scan_f64(mine);
    __syncthreads();  // (the sums in red have been read)
    if (lane == 63) red[0][wave] = upto;
    __syncthreads();
    double acc = before + (upto - mine);
    for (int k = 0; k < wave; ++k) acc += red[0][k];
    int first = 0x7FFFFFFF, lastw = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      acc += w[i];
      const bool any = w[i] > 0.0;
      lastw = any ? v0 + i : lastw;
      first = any && acc > t && first == 0x7FFFFFFF ? v0 + i : first;
    }
    // ids rise with the lane and the wave: the first lane that passes the threshold, the last that has a weight
    const uint64_t past = __builtin_amdgcn_ballot_w64(first != 0x7FFFFFFF), some = __builtin_amdgcn_ballot_w64(lastw >= 0);
    const int wave_first = past ? __builtin_amdgcn_readlane(first, __builtin_ctzll(past)) : 0x7FFFFFFF, wave_last = some ? __builtin_amdgcn_readlane(lastw, 63 - __builtin_clzll(some)) : -1;
    if (lane == 0) hits[wave] = wave_first, lasts[wave] = wave_last;
    __syncthreads();
    int hit = 0x7FFFFFFF, last = -1;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) hit = min(hit, hits[k]), last = max(last, lasts[k]);
    token = hit != 0x7FFFFFFF ? hit : last;  // (the sums' rounding can leave the threshold just past the chunk's end)
  }
  for (int r = r0 + tid; r < r1; r += kThreads) a.tokens[r] = r < j.end ? in.draft[r] : r == j.end ? token : -1;
  if (tid == 0) a.accepted[b] = j.end - r0;
}

template <int KIND>
int launch(const VerifyArgs& a, hipStream_t st) {
  if constexpr (KIND != 2) if (a.in.rows) {
    if (a.in.q) hipLaunchKernelGGL((k_stats<KIND, true>), dim3(a.ns, a.in.rows), dim3(kStatThreads), 0, st, a);
    else hipLaunchKernelGGL((k_stats<KIND, false>), dim3(a.ns, a.in.rows), dim3(kStatThreads), 0, st, a);
    DSGX_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(k_weights<KIND>, dim3((a.nc + a.sw - 1) / a.sw, a.in.B), dim3(kThreads), 0, st, a);
  DSGX_HIP(hipGetLastError());
  return DSGX_OK;
}

bool sizes_ok(int B, int rows, int V) { return B >= 1 && B <= 65535 && rows >= 0 && rows <= 65535 && V >= 1 && V <= (1 << 28); }
constexpr size_t kCountBytes = 65536 * sizeof(int);  // first in the workspace whatever the sizes: what a call leaves there is the next one's start
size_t stat_bytes(int rows, int nc) { return align256((size_t)rows * nc * sizeof(Stat)) + align256((size_t)rows * sizeof(Draft)); }
size_t sums_bytes(int B, int nc) { return align256((size_t)B * nc * sizeof(Sums)); }
// Chunks a piece, so that `rows` rows of nc chunks are about `room` workgroups (or pieces are `most` long).
// k_stats (in f64), 224 bf16 rows of 25 chunks: 23.5 to 24.4 us from one to five chunks a piece; 80 f32 rows of 32: 15.0 us in 2560 workgroups,
// 14.0 in 1280. k_weights, 16 sequences of 32 chunks: 17.0 us in 512 workgroups, 14.5 in 256; 48 of 25: 24.4 in 1200, 21.8 in 624,
// 19.6 in 432, 18.3 in 240.
int pieces_of(int rows, int nc, int room, int most) {
  const int per = room / (rows > 0 ? rows : 1);  // pieces a row
  return std::min(most, per < 1 ? nc : (nc + per - 1) / per);
}

}  // namespace
}  // namespace dsgx

using namespace dsgx;

extern "C" size_t dsgx_spec_verify_ws_bytes(int B, int rows, int V) {
  if (!sizes_ok(B, rows, V)) return 0;
  const int nc = (V + kChunk - 1) / kChunk;
  return kCountBytes + stat_bytes(rows, nc) + sums_bytes(B, nc);
}

extern "C" int dsgx_spec_verify(const dsgx_verify_in* in, int32_t* tokens, int32_t* accepted, void* ws, void* stream) {
  if (!in || !in->target || !in->us || !tokens || !accepted || !ws) return fail(DSGX_EINVAL, "spec_verify: null target, us, output or workspace");
  if (!sizes_ok(in->B, in->rows, in->V) || in->max_rows < 1)
    return fail(DSGX_EINVAL, "spec_verify: %d sequences, %d rows (%d each at most), %d tokens", in->B, in->rows, in->max_rows, in->V);
  if (in->kind < 0 || in->kind > 2) return fail(DSGX_EINVAL, "spec_verify: target kind %d", in->kind);
  if (!in->cu_rows && (int64_t)in->B * in->max_rows != in->rows) return fail(DSGX_EINVAL, "spec_verify: %d sequences of %d rows are not %d rows", in->B, in->max_rows, in->rows);
  if ((!in->draft || !in->u) && (in->cu_rows || in->max_rows > 1)) return fail(DSGX_EINVAL, "spec_verify: null drafts or random numbers");
  if (in->ldt < in->V || (in->q && in->ldq < in->V)) return fail(DSGX_EINVAL, "spec_verify: rows %lld, %lld apart for %d tokens", (long long)in->ldt, (long long)in->ldq, in->V);
  if (((uintptr_t)ws & 15) || ((uintptr_t)in->target & (in->kind == 1 ? 1 : 3)) || ((uintptr_t)in->q & 3))
    return fail(DSGX_EINVAL, "spec_verify: workspace, target or probabilities not aligned");
  VerifyArgs a{};
  a.in = *in, a.tokens = tokens, a.accepted = accepted;
  a.nc = (in->V + kChunk - 1) / kChunk;
  a.ss = pieces_of(in->rows, a.nc, kStatRoom, 1 << 16), a.ns = (a.nc + a.ss - 1) / a.ss;
  a.sw = pieces_of(in->B, a.nc, kRoom, kMostPieces);
  uint8_t* w = static_cast<uint8_t*>(ws);
  a.count = reinterpret_cast<int*>(w);
  a.stat = reinterpret_cast<Stat*>(w + kCountBytes);
  a.drafts = reinterpret_cast<Draft*>(w + kCountBytes + align256((size_t)in->rows * a.nc * sizeof(Stat)));
  a.sums = reinterpret_cast<Sums*>(w + kCountBytes + stat_bytes(in->rows, a.nc));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return in->kind == 0 ? launch<0>(a, st) : in->kind == 1 ? launch<1>(a, st) : launch<2>(a, st);
}
