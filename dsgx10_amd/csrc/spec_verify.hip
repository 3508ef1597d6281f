// Verification of drafted tokens against the target's distribution from given random numbers (include/dsgx.h). The result is whole
// numbers that lie next to borders (a cumulative sum over the vocabulary against a random threshold), so all sums and probabilities are
// f64: with f32 exponentials about one draw in a hundred of a flat distribution over 10^5 tokens would come out one token off.
//
// Three launches: k_stats reads every row of logits once and leaves, for each chunk of it, the maximum, the sum of exp and the lowest
// id of the maximum; k_weights judges its sequence's drafts (every workgroup for itself: a few KB out of L2), then sums the weights of
// its chunk of the one row that the next token comes from; k_pick finds the chunk and the token in it. Probabilities need no k_stats.
#include "abi_internal.h"
#include "common.cuh"

namespace dsgx {
namespace {

constexpr int kChunk = 4096, kThreads = 256, kPer = kChunk / kThreads;

struct Stat {  // of one chunk of one row; also of a whole row
  double sum;  // sum of exp((x - max) / T); T <= 0: 1, or NaN if the chunk holds one
  float max;
  int arg;
};
struct Judged {  // of one sequence
  double max, scale;  // the drawn-from row: p = exp((x - max) * 1/T) * scale
  int end, last, arg, rows0;
};
struct Sums {
  double rest, p;  // of max(p - q, 0) and of p over a chunk
};
struct VerifyArgs {
  dsgx_verify_in in;
  int nc;
  Stat* stat;      // [rows][nc]
  Sums* sums;      // [B][nc]
  Judged* judged;  // [B]
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

// e^y for y <= 0 (a NaN stays one): y = n ln 2 + r with |r| <= ln 2 / 2, the Taylor sum of e^r up to r^13 (the next term is below
// 2^-57) and 2^n. Twenty instructions where the library's exp, which has to serve every argument, takes about fifty: the exponentials
// of the logits are what this operator computes most of.
__device__ __forceinline__ double exp_neg(double y) {
  y = y < -800.0 ? -800.0 : y;  // (e^-800 is 0 in f64)
  const double n = rint(y * 1.4426950408889634074);
  double r = fma(n, -0x1.62e42fefa39efp-1, y);
  r = fma(n, -0x1.abc9e3b39803fp-56, r);  // (what the double nearest ln 2 leaves of it)
  double s = 1.0 / 6227020800.0;
  s = fma(s, r, 1.0 / 479001600.0);
  s = fma(s, r, 1.0 / 39916800.0);
  s = fma(s, r, 1.0 / 3628800.0);
  s = fma(s, r, 1.0 / 362880.0);
  s = fma(s, r, 1.0 / 40320.0);
  s = fma(s, r, 1.0 / 5040.0);
  s = fma(s, r, 1.0 / 720.0);
  s = fma(s, r, 1.0 / 120.0);
  s = fma(s, r, 1.0 / 24.0);
  s = fma(s, r, 1.0 / 6.0);
  s = fma(s, r, 0.5);
  s = fma(s, r, 1.0);
  s = fma(s, r, 1.0);
  return ldexp(s, (int)n);
}

__device__ __forceinline__ double shfl_f64(double v, int src) {
  const uint64_t b = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __shfl((int)(uint32_t)b, src), hi = __shfl((int)(b >> 32), src);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_f64(double v, int lane) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += shfl_f64(v, lane ^ d);
  return v;
}
__device__ __forceinline__ double block_sum_f64(double v, double* red, int lane, int wave) {
  v = wave_sum_f64(v, lane);
  __syncthreads();
  if (lane == 0) red[wave] = v;
  __syncthreads();
  return (red[0] + red[1]) + (red[2] + red[3]);
}
// the larger maximum, of equals the lower id
__device__ __forceinline__ void take_max(float& m, int& arg, float om, int oa) {
  const bool t = om > m || (om == m && oa < arg);
  m = t ? om : m, arg = t ? oa : arg;
}

// the sequence's rows; none if the bounds are out of order
__device__ __forceinline__ bool rows_of(const dsgx_verify_in& in, int b, int& r0, int& r1) {
  r0 = in.cu_rows ? in.cu_rows[b] : b * in.max_rows;
  r1 = in.cu_rows ? in.cu_rows[b + 1] : r0 + in.max_rows;
  return r0 >= 0 && r0 < r1 && r1 <= in.rows;
}
__device__ __forceinline__ int seq_of(const dsgx_verify_in& in, int r, int lane) {
  if (!in.cu_rows) return r / in.max_rows;
  for (int j0 = 0; j0 < in.B; j0 += kWave) {
    const int j = j0 + lane;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(j < in.B && in.cu_rows[j < in.B ? j : 0] <= r && r < in.cu_rows[j < in.B ? j + 1 : 0]);
    if (hit) return j0 + __builtin_ctzll(hit);
  }
  return -1;
}

template <int KIND>
__global__ void __launch_bounds__(kThreads) k_stats(VerifyArgs a) {
  constexpr int U = kUnit<KIND>, NU = kPer / U;
  const dsgx_verify_in& in = a.in;
  __shared__ double red[4];
  __shared__ float rm[4];
  __shared__ int ra[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = blockIdx.y, c = blockIdx.x;
  const int b = seq_of(in, r, lane);
  if (b < 0 || b >= in.B) return;
  const float T = in.temp ? in.temp[b] : 1.f;
  const void* row = row_of<KIND>(in.target, in.ldt, r);
  float x[NU][U];
#pragma unroll
  for (int k = 0; k < NU; ++k) load_unit<KIND>(row, c * kChunk + (k * kThreads + (int)threadIdx.x) * U, in.V, -__builtin_inff(), x[k]);
  float m = -__builtin_inff();
  int arg = 0x7FFFFFFF;
#pragma unroll
  for (int k = 0; k < NU; ++k)
#pragma unroll
    for (int i = 0; i < U; ++i) {
      const int v = c * kChunk + (k * kThreads + (int)threadIdx.x) * U + i;
      if (x[k][i] > m) m = x[k][i], arg = v;  // (ids rise within a thread: the first of equals stays)
    }
#pragma unroll
  for (int d = 32; d; d >>= 1) take_max(m, arg, __shfl_xor(m, d), __shfl_xor(arg, d));
  if (lane == 0) rm[wave] = m, ra[wave] = arg;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 4; ++w) take_max(m, arg, rm[w], ra[w]);
  double s = 0.0;
  if (T > 0.f || T != T) {
    const double it = 1.0 / (double)T, md = m;
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const float xv = x[k][i];
        // (a chunk of nothing but -inf has no maximum to subtract)
        s += m == -__builtin_inff() ? (xv == xv ? 0.0 : (double)xv) : exp_neg(((double)xv - md) * it);
      }
  } else {
#pragma unroll
    for (int k = 0; k < NU; ++k)
#pragma unroll
      for (int i = 0; i < U; ++i) s += x[k][i] == x[k][i] ? 0.0 : (double)x[k][i];
    if (threadIdx.x == 0) s += 1.0;
  }
  s = block_sum_f64(s, red, lane, wave);
  if (threadIdx.x == 0) a.stat[(size_t)r * a.nc + c] = Stat{s, m, arg};
}

// A row's statistics out of its chunks', by one wave; wave-uniform
__device__ __forceinline__ Stat row_stat(const VerifyArgs& a, int r, float T, int lane) {
  float m = -__builtin_inff();
  int arg = 0x7FFFFFFF;
  const Stat* st = a.stat + (size_t)r * a.nc;
  for (int c = lane; c < a.nc; c += kWave) take_max(m, arg, st[c].max, st[c].arg);
#pragma unroll
  for (int d = 32; d; d >>= 1) take_max(m, arg, __shfl_xor(m, d), __shfl_xor(arg, d));
  double s = 0.0;
  const double it = 1.0 / (double)T;
  for (int c = lane; c < a.nc; c += kWave) {
    const double cs = st[c].sum;
    if (!(T > 0.f || T != T)) s += cs;
    else s += cs == 0.0 ? 0.0 : cs * exp_neg(((double)st[c].max - (double)m) * it);
  }
  return Stat{wave_sum_f64(s, lane), m, arg};
}

// p of a value: logits x, or the probability itself
template <int KIND>
__device__ __forceinline__ double prob(float x, int v, const Judged& j, double it, bool greedy) {
  if (KIND == 2) return (double)x;
  if (greedy) return v == j.arg ? j.scale : 0.0 * j.scale;  // (a row with a NaN has a NaN scale)
  return exp_neg(((double)x - j.max) * it) * j.scale;
}
__device__ __forceinline__ double rest_of(double p, double q) {
  const double d = p - q;
  return d > 0.0 ? d : d == d ? 0.0 : d;
}

// the drafts of sequence b up to the first that is refused; by the whole workgroup
template <int KIND>
__device__ __forceinline__ Judged judge(const VerifyArgs& a, int b, int r0, int r1, float T, int lane, int wave, Judged* sh, int* stop) {
  const dsgx_verify_in& in = a.in;
  const bool greedy = !(T > 0.f || T != T);
  const double it = 1.0 / (double)T;
  for (int i0 = r0;; i0 += 4) {
    const int r = i0 + wave;
    bool stops = false;
    Judged j{0.0, 1.0, r, 0, -1, r0};
    if (r < r1) {
      if (KIND != 2) {
        const Stat s = row_stat(a, r, T, lane);
        j.max = s.max, j.arg = s.arg;
        j.scale = greedy ? s.sum * 0.0 + 1.0 : 1.0 / s.sum;
      }
      j.last = r == r1 - 1;
      stops = j.last;
      if (!j.last) {
        const int d = in.draft[r];
        double p = 0.0, q = 1.0;
        if (d >= 0 && d < in.V) {
          const void* row = row_of<KIND>(in.target, in.ldt, r);
          const float x = KIND == 1 ? bf16_bits_to_f32(static_cast<const uint16_t*>(row)[d]) : static_cast<const float*>(row)[d];
          p = prob<KIND>(x, d, j, it, greedy);
          if (in.q) q = in.q[in.ldq * (int64_t)r + d];
        }
        stops = !((double)in.u[r] * q < p);
      }
    }
    __syncthreads();
    if (lane == 0) sh[wave] = j, stop[wave] = stops;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (stop[w]) return sh[w];
  }
}

// the weights of U ids from v on of the judged row: rest = max(p - q, 0) (the last row: p), and p
template <int KIND>
__device__ __forceinline__ void weights(const VerifyArgs& a, const Judged& j, double it, bool greedy, int v, double (&rest)[kUnit<KIND>], double (&p)[kUnit<KIND>]) {
  constexpr int U = kUnit<KIND>;
  const dsgx_verify_in& in = a.in;
  float x[U];
  load_unit<KIND>(row_of<KIND>(in.target, in.ldt, j.end), v, in.V, KIND == 2 ? 0.f : -__builtin_inff(), x);
#pragma unroll
  for (int i = 0; i < U; ++i) p[i] = v + i < in.V ? prob<KIND>(x[i], v + i, j, it, greedy) : 0.0;
  if (j.last) {
#pragma unroll
    for (int i = 0; i < U; ++i) rest[i] = p[i];
  } else if (in.q) {
    const float* qr = in.q + in.ldq * (int64_t)j.end;
#pragma unroll
    for (int h = 0; h < U; h += 4) {
      float q[4];
      load_unit<0>(qr, v + h, in.V, 0.f, q);
#pragma unroll
      for (int i = 0; i < 4; ++i) rest[h + i] = rest_of(p[h + i], (double)q[i]);
    }
  } else {
    const int d = in.draft[j.end];
#pragma unroll
    for (int i = 0; i < U; ++i) rest[i] = rest_of(p[i], v + i == d ? 1.0 : 0.0);
  }
}

template <int KIND>
__global__ void __launch_bounds__(kThreads) k_weights(VerifyArgs a) {
  constexpr int U = kUnit<KIND>, NU = kPer / U;
  __shared__ double red[4];
  __shared__ Judged sh[4];
  __shared__ int stop[4];
  const dsgx_verify_in& in = a.in;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b = blockIdx.y, c = blockIdx.x;
  int r0, r1;
  if (!rows_of(in, b, r0, r1)) return;
  const float T = KIND != 2 && in.temp ? in.temp[b] : 1.f;
  const bool greedy = !(T > 0.f || T != T);
  const Judged j = judge<KIND>(a, b, r0, r1, T, lane, wave, sh, stop);
  const double it = 1.0 / (double)T;
  double sr = 0.0, sp = 0.0;
#pragma unroll
  for (int k = 0; k < NU; ++k) {
    double rest[U], p[U];
    weights<KIND>(a, j, it, greedy, c * kChunk + (k * kThreads + (int)threadIdx.x) * U, rest, p);
#pragma unroll
    for (int i = 0; i < U; ++i) sr += rest[i], sp += p[i];
  }
  sr = block_sum_f64(sr, red, lane, wave);
  sp = block_sum_f64(sp, red, lane, wave);
  if (threadIdx.x == 0) {
    a.sums[(size_t)b * a.nc + c] = Sums{sr, sp};
    if (c == 0) a.judged[b] = j;
  }
}

template <int KIND>
__global__ void __launch_bounds__(kThreads) k_pick(VerifyArgs a) {
  constexpr int U = kUnit<KIND>, NU = kPer / U;
  __shared__ double part[kThreads];
  __shared__ int hit, lastpos;
  const dsgx_verify_in& in = a.in;
  const int b = blockIdx.x, tid = threadIdx.x;
  int r0, r1;
  if (!rows_of(in, b, r0, r1)) {
    if (tid == 0) a.accepted[b] = 0;
    return;
  }
  const Judged j = a.judged[b];
  const float T = KIND != 2 && in.temp ? in.temp[b] : 1.f;
  const bool greedy = !(T > 0.f || T != T);
  const double it = 1.0 / (double)T;
  const Sums* s = a.sums + (size_t)b * a.nc;
  // the chunk sums in order, by every thread alike (tens of values out of L2)
  double total = 0.0;
  for (int c = 0; c < a.nc; ++c) total += s[c].rest;
  const bool of_p = total <= 0.0;  // nothing left of the difference: from p
  if (of_p) {
    total = 0.0;
    for (int c = 0; c < a.nc; ++c) total += s[c].p;
  }
  const double t = (double)in.us[b] * total;
  int token = -1;
  if (total > 0.0 && total < __builtin_inf()) {
    double run = 0.0, before = 0.0;
    int chunk = 0;
    for (int c = 0; c < a.nc; ++c) {
      const double w = of_p ? s[c].p : s[c].rest;
      if (w > 0.0) chunk = c, before = run;
      run += w;
      if (w > 0.0 && run > t) break;
    }
    // inside it: sixteen ids a thread, the threads' sums before a thread added in order
    const int v0 = chunk * kChunk + tid * kPer;
    double w[kPer], mine = 0.0;
#pragma unroll
    for (int k = 0; k < NU; ++k) {
      double rest[U], p[U];
      weights<KIND>(a, j, it, greedy, v0 + k * U, rest, p);
#pragma unroll
      for (int i = 0; i < U; ++i) w[k * U + i] = of_p ? p[i] : rest[i], mine += w[k * U + i];
    }
    part[tid] = mine;
    if (tid == 0) hit = 0x7FFFFFFF, lastpos = -1;
    __syncthreads();
    double acc = before;
    for (int k = 0; k < tid; ++k) acc += part[k];
    int first = 0x7FFFFFFF, lastw = -1;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      acc += w[i];
      if (w[i] > 0.0) {
        lastw = v0 + i;
        if (acc > t && first == 0x7FFFFFFF) first = v0 + i;
      }
    }
    if (first != 0x7FFFFFFF) atomicMin(&hit, first);
    if (lastw >= 0) atomicMax(&lastpos, lastw);
    __syncthreads();
    token = hit != 0x7FFFFFFF ? hit : lastpos;  // (the sums' rounding can leave the threshold just past the chunk's end)
  }
  for (int r = r0 + tid; r < r1; r += kThreads) a.tokens[r] = r < j.end ? in.draft[r] : r == j.end ? token : -1;
  if (tid == 0) a.accepted[b] = j.end - r0;
}

template <int KIND>
int launch(const VerifyArgs& a, hipStream_t st) {
  if (KIND != 2) {
    hipLaunchKernelGGL(k_stats<KIND>, dim3(a.nc, a.in.rows), dim3(kThreads), 0, st, a);
    DSGX_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(k_weights<KIND>, dim3(a.nc, a.in.B), dim3(kThreads), 0, st, a);
  DSGX_HIP(hipGetLastError());
  hipLaunchKernelGGL(k_pick<KIND>, dim3(a.in.B), dim3(kThreads), 0, st, a);
  DSGX_HIP(hipGetLastError());
  return DSGX_OK;
}

bool sizes_ok(int B, int rows, int V) { return B >= 1 && B <= 65535 && rows >= 0 && rows <= 65535 && V >= 1 && V <= (1 << 28); }
size_t stat_bytes(int rows, int nc) { return align256((size_t)rows * nc * sizeof(Stat)); }
size_t sums_bytes(int B, int nc) { return align256((size_t)B * nc * sizeof(Sums)); }

}  // namespace
}  // namespace dsgx

using namespace dsgx;

extern "C" size_t dsgx_spec_verify_ws_bytes(int B, int rows, int V) {
  if (!sizes_ok(B, rows, V)) return 0;
  const int nc = (V + kChunk - 1) / kChunk;
  return stat_bytes(rows, nc) + sums_bytes(B, nc) + align256((size_t)B * sizeof(Judged));
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
  if (in->rows == 0) return DSGX_OK;
  VerifyArgs a{*in, (in->V + kChunk - 1) / kChunk, nullptr, nullptr, nullptr, tokens, accepted};
  uint8_t* w = static_cast<uint8_t*>(ws);
  a.stat = reinterpret_cast<Stat*>(w);
  a.sums = reinterpret_cast<Sums*>(w + stat_bytes(in->rows, a.nc));
  a.judged = reinterpret_cast<Judged*>(w + stat_bytes(in->rows, a.nc) + sums_bytes(in->B, a.nc));
  hipStream_t st = static_cast<hipStream_t>(stream);
  return in->kind == 0 ? launch<0>(a, st) : in->kind == 1 ? launch<1>(a, st) : launch<2>(a, st);
}
