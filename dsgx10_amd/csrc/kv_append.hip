// The step's queries, keys and values on their way to attention: RMSNorm of every head of q and k, the position rotation, the
// rounding, and the keys and values into their tokens' places of the paged cache, in one pass.
//
// A head is D / 8 lanes of 8 values (one 16-byte load), so a wave holds 8, 4 or 2 heads at a time; sums of squares go over the
// head's lanes by DPP and half swaps, a rotation's partner comes from the lane rot / 16 away (pairs (j, j + rot / 2)) or stands in
// the lane itself (pairs (2j, 2j + 1)). Nothing passes through LDS and no wave waits for another.
// Bound by bytes, or for few rows by the launch and three loads that wait for one another (bounds, page, and beside them the row):
// 8252 rows of 64 + 2 x 8 heads of 128 values 75 us, 4.5 TB/s read and written (a large copy: 4.7 to 4.9); 107 rows of 32 + 2 x 8 heads into
// e4m3 6.5 us, one row of 64 + 2 heads of 256 4.4 (an empty launch 1.9).
#include "kv_cache.cuh"

namespace dsgx {
namespace {

struct AppendArgs {
  dsgx_kv_cache c;
  dsgx_kv_batch b;
  dsgx_kv_append_in in;
  int page_shift;
};

template <int LANES>
__device__ __forceinline__ float head_sum(float v) {
  v = dpp_add<0xB1>(v);
  v = dpp_add<0x4E>(v);
  v = dpp_add<0x141>(v);
  if (LANES >= 16) v = dpp_add<0x140>(v);
  if (LANES >= 32) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}
__device__ __forceinline__ void unpack8(const u32x4_t& w, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f[2 * i] = bf16_lo(w[i]), f[2 * i + 1] = bf16_hi(w[i]);
}
__device__ __forceinline__ float to_e4m3_range(float v) { return v > 448.f ? 448.f : v < -448.f ? -448.f : v; }  // (a NaN passes)

template <int D, bool F8>
__global__ void __launch_bounds__(256) k_kv_append(AppendArgs a) {
  constexpr int L = D / 8, HPW = kWave / L;  // lanes a head, heads a wave
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), r = blockIdx.x;
  const dsgx_kv_append_in& in = a.in;
  const RowPlace p = find_row(a.b, r, lane);
  if (p.seq < 0) return;
  const int t = p.len - (p.end - r);
  const int pos = in.pos ? in.pos[r] : a.b.prefix_len + t;
  const bool pos_ok = in.rot == 0 || (pos >= 0 && pos < in.rope_len);
  int page = -1;
  if (pos_ok && t >= 0 && (t >> a.page_shift) < a.b.table_ld) page = a.b.table[(size_t)p.seq * a.b.table_ld + (t >> a.page_shift)];
  const bool keep = page >= 0 && page < a.c.npages;
  const int64_t tok = keep ? (int64_t)page * a.c.page_stride + (int64_t)(t & (a.c.page - 1)) * a.c.tok_stride : 0;

  const int c = lane % L, d0 = 8 * c, rel = d0 - in.rot_off, half = in.rot >> 1;
  const bool turns = rel >= 0 && rel < in.rot;
  const bool second = !in.pairs && rel >= half;
  const int partner = lane + (second ? -(in.rot >> 4) : (in.rot >> 4));
  float co[8], si[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) co[i] = 1.f, si[i] = 0.f;
  if (turns) {
    if (pos_ok) {
      const float* tab = in.rope + (size_t)pos * in.rot;
      const int j0 = in.pairs ? rel >> 1 : second ? rel - half : rel;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int j = j0 + (in.pairs ? i >> 1 : i);
        co[i] = tab[j], si[i] = tab[half + j];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) co[i] = si[i] = __builtin_nanf("");
    }
  }
  float wq[8], wk[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) wq[i] = wk[i] = 1.f;
  if (in.q_norm) unpack8(*reinterpret_cast<const u32x4_t*>(in.q_norm + d0), wq);
  if (in.k_norm) unpack8(*reinterpret_cast<const u32x4_t*>(in.k_norm + d0), wk);

  const int Hkv = a.c.Hkv, total = in.Hq + 2 * Hkv;
  for (int h0 = ((int)blockIdx.y * 4 + wave) * HPW; h0 < total; h0 += (int)gridDim.y * 4 * HPW) {
    const int h = h0 + lane / L;
    const bool live = h < total, is_q = h < in.Hq, is_k = !is_q && h < in.Hq + Hkv;
    const int hk = is_q ? h : is_k ? h - in.Hq : h - in.Hq - Hkv;
    const uint16_t* src = is_q ? in.q + (size_t)r * in.ldq : is_k ? in.k + (size_t)r * in.ldk : in.v + (size_t)r * in.ldv;
    u32x4_t w = {0, 0, 0, 0};
    if (live) w = *reinterpret_cast<const DSGX_GLOBAL u32x4_t*>((uintptr_t)(src + (size_t)hk * D + d0));
    float x[8], y[8];
    unpack8(w, x);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
    ss = head_sum<L>(ss);
    const bool norm = is_q ? in.q_norm != nullptr : is_k && in.k_norm != nullptr;
    if (norm) {
      const float rstd = __fdiv_rn(1.f, sqrtf(fmaf(ss, 1.f / D, in.eps)));
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __fmul_rn(__fmul_rn(x[i], rstd), is_q ? wq[i] : wk[i]);
    }
    if (in.rot) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float o = in.pairs ? x[i ^ 1] : __shfl(x[i], partner & 63);
        const bool lower = in.pairs ? !(i & 1) : !second;  // the pair's first: a c - b s; its second: b c + a s
        y[i] = lower ? fmaf(x[i], co[i], -__fmul_rn(o, si[i])) : fmaf(x[i], co[i], __fmul_rn(o, si[i]));
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = turns && (is_q || is_k) ? y[i] : x[i];
    }
    if (!live) continue;
    if (is_q || !F8) {
      const u32x4_t o = {pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3]), pack_bf16(x[4], x[5]), pack_bf16(x[6], x[7])};
      if (is_q) *reinterpret_cast<u32x4_t*>(in.q_out + (size_t)r * in.ldqo + (size_t)hk * D + d0) = o;
      else if (keep) *reinterpret_cast<u32x4_t*>(static_cast<uint16_t*>(is_k ? a.c.k : a.c.v) + tok + hk * a.c.head_stride + d0) = o;
    } else if (keep) {
      const float s = (is_k ? a.c.ks : a.c.vs)[hk];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = to_e4m3_range(__fdiv_rn(x[i], s));
      uint2 o;
      o.x = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
      o.x = __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], o.x, true);
      o.y = __builtin_amdgcn_cvt_pk_fp8_f32(x[4], x[5], 0, false);
      o.y = __builtin_amdgcn_cvt_pk_fp8_f32(x[6], x[7], o.y, true);
      *reinterpret_cast<uint2*>(static_cast<uint8_t*>(is_k ? a.c.k : a.c.v) + tok + hk * a.c.head_stride + d0) = o;
    }
  }
}

template <int D>
void launch(const AppendArgs& a, dim3 grid, hipStream_t st) {
  if (a.c.fmt == DSGX_KV_E4M3) hipLaunchKernelGGL((k_kv_append<D, true>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_kv_append<D, false>), grid, dim3(256), 0, st, a);
}

}  // namespace
}  // namespace dsgx

using namespace dsgx;

extern "C" int dsgx_kv_append(const dsgx_kv_cache* cache, const dsgx_kv_batch* batch, const dsgx_kv_append_in* in, void* stream) {
  if (int rc = check_cache("kv_append", cache)) return rc;
  if (int rc = check_batch("kv_append", cache, batch)) return rc;
  if (!in || !in->k || !in->v) return fail(DSGX_EINVAL, "kv_append: null keys or values");
  const int D = cache->D;
  if (in->Hq < 0 || in->Hq > 65536 || (in->Hq > 0) != (in->q != nullptr) || (in->q && !in->q_out))
    return fail(DSGX_EINVAL, "kv_append: %d query heads (q and q_out with them, neither without)", in->Hq);
  if (in->rot < 0 || in->rot % 16 || in->rot_off < 0 || in->rot_off % 16 || in->rot + in->rot_off > D)
    return fail(DSGX_EINVAL, "kv_append: dims %d .. %d of %d rotated (multiples of 16)", in->rot_off, in->rot_off + in->rot, D);
  if (in->rot && (!in->rope || in->rope_len < 1)) return fail(DSGX_EINVAL, "kv_append: a rotation needs its table");
  if (((uintptr_t)in->q | (uintptr_t)in->k | (uintptr_t)in->v | (uintptr_t)in->q_out | (uintptr_t)in->q_norm | (uintptr_t)in->k_norm | (uintptr_t)in->rope) & 15)
    return fail(DSGX_EINVAL, "kv_append: rows, norms and table have to be 16-byte aligned");
  if (in->ldk % 8 || in->ldv % 8 || in->ldk < (int64_t)cache->Hkv * D || in->ldv < (int64_t)cache->Hkv * D ||
      (in->q && (in->ldq % 8 || in->ldqo % 8 || in->ldq < (int64_t)in->Hq * D || in->ldqo < (int64_t)in->Hq * D)))
    return fail(DSGX_EINVAL, "kv_append: rows %lld, %lld, %lld, %lld apart (multiples of 8, the heads' values at least)", (long long)in->ldq, (long long)in->ldk, (long long)in->ldv,
                (long long)in->ldqo);
  if (batch->rows == 0) return DSGX_OK;
  AppendArgs a{*cache, *batch, *in, __builtin_ctz((unsigned)cache->page)};
  // few rows: the heads over workgroups of their own, so that the call is one pass of loads; many: a row a workgroup
  const int units = (in->Hq + 2 * cache->Hkv + 4 * (512 / D) - 1) / (4 * (512 / D)), want = (2 * num_cus_cached() + batch->rows - 1) / batch->rows;
  const dim3 grid(batch->rows, units < want ? units : want < 1 ? 1 : want);
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (D == 64) launch<64>(a, grid, st);
  else if (D == 128) launch<128>(a, grid, st);
  else launch<256>(a, grid, st);
  DSGX_HIP(hipGetLastError());
  return DSGX_OK;
}
