// Attention of a decode step's rows over the paged cache (include/dsgx.h): a shared prefix and every sequence's own tokens.
//
// One pass over the tokens with the running maximum and sum of the softmax (in powers of two). The G = Hq / Hkv query heads that
// share a head of keys and values are G columns of one matrix product, times the rows that attend over the same tokens: a
// sequence's rows over its own tokens, all rows over the prefix. The tokens are cut into ranges, a workgroup each; what the ranges
// leave (maximum, sum, unnormalised output in f32) k_combine joins.
//
// Bound by the cache's bytes for few columns, by the matrix unit (and, with e4m3, the staging beside it) for many, and below about 20 us by the
// chain of a launch: bounds and lengths, page numbers, keys, the waves' join. Whole calls (a large read reaches 7.1 TB/s, a large product 1.4 to
// 1.6 PFLOP/s): 69 rows of 32 heads over 32 ragged e4m3 sequences, 178 MB, 51 us (44 + 8; 3.5 TB/s); 5 rows of 64 heads of 256 over one, 50001
// tokens, 49 us (44.5 + 9.5 alone; 0.33 PFLOP/s); 8011 tokens before 48 rows of 64 heads with 37 to 600 of their own, 40 us (34 + 7); 32768 before 300 rows of
// 32 heads, e4m3, 209 us (0.78 PFLOP/s); one row over 301 tokens 10 us.
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

// How the work is cut. The prefix: `splits` ranges of `chunk` tokens, `tiles` tiles of `cols` query columns of all rows. The sequences' own
// tokens: ranges of a length that the kernels find from lens when they run (own_plan), so that about `target` workgroups have the same to do
// whatever max_len announced; at most `most` of them have a place for what they leave.
// A workgroup has `heads` heads of keys and values side by side (1, 2 or 4, a divisor of Hkv; own: as many at most).
struct Part {
  int cols, tiles, splits, chunk, heads;  // the prefix
};
struct Own {
  int cols, target, least, most, heads, tiles;  // least: tokens a range at least (a multiple of 128); tiles: of a sequence of max_rows rows
};
struct AttnArgs {
  dsgx_kv_cache c;
  dsgx_kv_batch b;
  Part pre;
  Own own;
  const uint16_t* q;
  uint16_t* out;
  float *lse, *part;  // part: [places][cols][D], the prefix's first
  float2* ml;         // [places][cols]
  int pre_blocks;     // workgroups for the prefix, a multiple of 8
  int32_t* plan;      // [4 + B]: tokens a range, heads a workgroup; from 4 on every sequence's first item
  int64_t ldq, ldo;
  int Hq, G, page_shift;
  float scale2;              // |scale| log2 e; 1 for a scale of zero
  uint32_t q_flip, q_keep;   // the scale's sign and whether it is zero, on the queries' bits
};

#define DSGX_CONST __attribute__((address_space(4)))  // read-only while a kernel runs: uniform loads go to the scalar unit
typedef const DSGX_CONST int32_t* table_t;

// A lane's sequence of 64 from j0 on: its rows, its own tokens, its tiles of `cols` columns
struct Seq {
  int first, rows, len, tiles;
};
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int j) {
  Seq s{0, 0, 0, 0};
  if (j >= a.b.B) return s;
  const int lo = a.b.cu_rows ? a.b.cu_rows[j] : j * a.b.max_rows, hi = a.b.cu_rows ? a.b.cu_rows[j + 1] : lo + a.b.max_rows, len = a.b.lens[j];
  if (lo < 0 || hi <= lo || hi > a.b.rows) return s;
  const int cap = a.b.table_ld << a.page_shift;
  s.first = lo, s.rows = hi - lo, s.len = len < 0 ? 0 : len > cap ? cap : len;
  s.tiles = (s.rows * a.G + a.own.cols - 1) / a.own.cols;
  return s;
}
// inclusive sums over the lanes: DPP shifts within the rows of sixteen, then the rows' last lanes handed on
template <int CTRL, int ROWS>
__device__ __forceinline__ int scan_step(int v) { return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false); }
__device__ __forceinline__ int wave_scan(int v) {
  v = scan_step<0x111, 0xF>(v);  // row_shr 1, 2, 4, 8
  v = scan_step<0x112, 0xF>(v);
  v = scan_step<0x114, 0xF>(v);
  v = scan_step<0x118, 0xF>(v);
  v = scan_step<0x142, 0xA>(v);  // row_bcast 15 into rows 1 and 3
  return scan_step<0x143, 0xC>(v);  // row_bcast 31 into rows 2 and 3
}
__device__ __forceinline__ int ranges_of(int len, int chunk) { return len ? (len + chunk - 1) / chunk : 1; }
// Tokens a range of the sequences' own, by a whole wave; s: the lane's sequence of the first 64. The kernels that ask get the same answer.
// A workgroup does a whole number of ranges one after the other: for one to four of them, ranges just long enough that there are no more of
// them (each sequence's last one is short) than workgroups times that, and of the four the choice that is done first, a range's own
// cost (set-up, joining) being that of kRangeCost tokens.
// Heads side by side are worth their longer way through the tokens (a wave has its head's alone) while that is 96 tokens or more.
constexpr int kRangeCost = 192, kTogether = 96;
struct Cut {
  int chunk, heads;
  int share;  // items of an XCD, 0: all in order
};
__device__ __forceinline__ Cut own_plan(const AttnArgs& a, const Seq& s0, int lane) {
  if (a.own.target == 0) return Cut{1 << 30, 1, 0};  // a range a sequence
  constexpr int KEPT = 4;  // sixty-fours of sequences in registers; the rest are read again every time
  int tiles[KEPT], len[KEPT];
#pragma unroll
  for (int k = 0; k < KEPT; ++k) {
    Seq t = s0;
    if (k) t = k * kWave < a.b.B ? seq_of(a, k * kWave + lane) : Seq{0, 0, 0, 0};
    tiles[k] = t.tiles, len[k] = t.len;
  }
  auto sum = [&](auto&& f) {
    float v = f(tiles[0], len[0]);
#pragma unroll
    for (int k = 1; k < KEPT; ++k)
      if (k * kWave < a.b.B) v += f(tiles[k], len[k]);
    for (int j0 = KEPT * kWave; j0 < a.b.B; j0 += kWave) {
      const Seq t = seq_of(a, j0 + lane);
      v += f(t.tiles, t.len);
    }
    return uni(wave_sum(v));
  };
  float w = sum([](int t, int n) { return (float)t * (float)n; }) * (float)a.c.Hkv * 1.0001f;
  int heads = a.own.heads, best = 0;
  while (heads > 1 && w < (float)a.own.target * (float)(kTogether * heads)) heads >>= 1;
  const float groups = (float)(a.c.Hkv / heads);
  w /= (float)heads;
  float cost = 3e38f;
#pragma unroll 1
  for (int turns = 1; turns <= 4; ++turns) {
    const float room = (float)(a.own.target * turns), share = w / room;
    if (share + (float)kRangeCost > cost / (float)turns) break;  // (not even without a loss)
    int chunk = max(heads > 1 ? 128 : a.own.least, ((int)min(share, 1e9f) + 128) & ~127);
    float all = 0.f;
#pragma unroll 1
    for (int k = 0; k < 3; ++k) {
      all = sum([chunk](int t, int n) { return (float)(t * ranges_of(n, chunk)); }) * groups;
      if (all <= room) break;
      if (k < 2) chunk = ((int)min((float)chunk * all / room, 1e9f) + 128) & ~127;
    }
    const float c = ceilf(all / (float)a.own.target) * (float)(chunk + kRangeCost);
    if (c < cost) cost = c, best = chunk;
    if (chunk <= (heads > 1 ? 128 : a.own.least)) break;
  }
  return Cut{best, heads, 0};
}
// The cut and every sequence's first item, for the kernels that come after; by one wave
__device__ __forceinline__ void write_plan(const AttnArgs& a, const Seq& s0, Cut cut, int lane) {
  if (lane == 0) a.plan[0] = cut.chunk, a.plan[1] = cut.heads;
  int run = 0;
  for (int j0 = 0; j0 < a.b.B; j0 += kWave) {
    const Seq t = j0 ? seq_of(a, j0 + lane) : s0;
    const int mine = t.tiles * ranges_of(t.len, cut.chunk), upto = run + wave_scan(mine);
    if (j0 + lane < a.b.B) a.plan[4 + j0 + lane] = upto - mine;
    run = __builtin_amdgcn_readlane(upto, 63);
  }
}
// What a workgroup of a launch is: `block` of `blocks` for the prefix or for the sequences' own tokens
enum Mode { kOwnOnly, kPrefixOnly, kBoth };
struct Role {
  bool prefix;
  int block, blocks;
};
// kBoth: the prefix's first, which are the longer ones (in turn with the others, 32768 tokens under 300 rows of 32 heads took 367 us instead of 250)
__device__ __forceinline__ Role role_of(const AttnArgs& a, int mode) {
  const int i = blockIdx.x, pre = mode == kBoth ? a.pre_blocks : mode == kPrefixOnly ? (int)gridDim.x : 0;
  return i < pre ? Role{true, i, pre} : Role{false, i - pre, (int)gridDim.x - pre};
}
// At a kernel's start: the cut of the sequences' own tokens. Where the prefix has a launch of its own before theirs, its last workgroup has made
// it; else every workgroup makes it and the first leaves it for k_combine.
__device__ __forceinline__ bool begin_plan(const AttnArgs& a, int mode, const Role& role, int lane, int wave, Seq& s0, Cut& cut) {
  if (role.prefix) {
    if (mode == kBoth || role.block != role.blocks - 1) return true;
    if (wave == 0) s0 = seq_of(a, lane), write_plan(a, s0, own_plan(a, s0, lane), lane);
    return false;
  }
  s0 = seq_of(a, lane);
  if (a.pre.splits && mode != kBoth) {
    cut = Cut{uni(a.plan[0]), uni(a.plan[1]), 0};
  } else {
    cut = own_plan(a, s0, lane);
    if (role.block == 0 && wave == 0 && a.own.target) write_plan(a, s0, cut, lane);
  }
  // The tiles that read the same tokens on one XCD (workgroup i runs on XCD i % 8), out of its L2: every XCD has an eighth of the items, in
  // order. 64 heads of 256 over 50001 tokens: 8 rows, eight tiles, 67 us instead of 72, 5 rows 44.9 instead of 50.2 (e4m3, half the bytes, 44.4 instead of 43.0).
  if (a.own.tiles > 1) {
    int items = 0;
    for (int j0 = 0; j0 < a.b.B; j0 += kWave) {
      const Seq t = j0 ? seq_of(a, j0 + lane) : s0;
      items += __builtin_amdgcn_readlane(wave_scan(t.tiles * ranges_of(t.len, cut.chunk)), 63);
    }
    cut.share = (items * (a.c.Hkv / cut.heads) + 7) / 8;
  }
  return true;
}
// The sequence that `item` (of all sequences' ranges times tiles) falls to, and how many items precede the sequence's; false past the last
__device__ __forceinline__ bool own_find(const AttnArgs& a, const Seq& s0, int chunk, int item, int lane, Seq& s, int& b, int& before) {
  int run = 0;
  for (int j0 = 0; j0 < a.b.B; j0 += kWave) {
    const Seq t = j0 ? seq_of(a, j0 + lane) : s0;
    const int mine = t.tiles * ranges_of(t.len, chunk), upto = run + wave_scan(mine);
    const uint64_t hit = __builtin_amdgcn_ballot_w64(upto > item);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      b = j0 + l, before = __builtin_amdgcn_readlane(upto - mine, l);
      s = Seq{__builtin_amdgcn_readlane(t.first, l), __builtin_amdgcn_readlane(t.rows, l), __builtin_amdgcn_readlane(t.len, l), __builtin_amdgcn_readlane(t.tiles, l)};
      return true;
    }
    run = __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// What a workgroup works on: tile `tile` of the columns of rows first .. first + rows - 1, over tokens lo .. hi - 1 of len, with the heads
// from `head` on
struct Item {
  table_t tab;
  int head, first, rows, len, lo, hi, tile;
  int64_t place, next;  // of the first head's first column in part and ml, and from a head to the next
  bool causal, alone;   // alone: nobody else adds to these columns, so that the result is final
};
// (the compiler cannot know that what came out of a search over the lanes is the same in all of them)
__device__ __forceinline__ int64_t uni64(int64_t v) { return (int64_t)((uint64_t)uni((uint32_t)((uint64_t)v >> 32)) << 32 | uni((uint32_t)v)); }
__device__ __forceinline__ Item uniform(const Item& t) {
  return Item{(table_t)uni64((int64_t)t.tab), uni(t.head), uni(t.first), uni(t.rows), uni(t.len), uni(t.lo), uni(t.hi), uni(t.tile), uni64(t.place), uni64(t.next), uni((int)t.causal) != 0,
              uni((int)t.alone) != 0};
}
__device__ __forceinline__ Item prefix_item(const AttnArgs& a, int i, bool& any) {
  // The tiles that read the same tokens run on the same XCD (workgroup i runs on XCD i % 8) next to each other, out of its L2: an eighth of all
  // for every XCD, in order. (Whole ranges for an XCD, 20001 tokens in 3 for 4 heads of 256 and 38 tiles took 582 us instead of 437.)
  const int n = i % 8 * (a.pre_blocks / 8) + i / 8, groups = a.c.Hkv / a.pre.heads, pair = n / a.pre.tiles, split = pair / groups;
  Item t{(table_t)(uintptr_t)a.b.prefix, pair % groups * a.pre.heads, 0, a.b.rows, a.b.prefix_len, split * a.pre.chunk, 0, n % a.pre.tiles, 0, 0, false, false};
  t.hi = min(t.len, t.lo + a.pre.chunk), t.next = (int64_t)a.pre.tiles * a.pre.cols;
  t.place = (int64_t)(split * a.c.Hkv + t.head) * t.next + (int64_t)t.tile * a.pre.cols;
  any = split < a.pre.splits;
  return t;
}
__device__ __forceinline__ int64_t own_places(const AttnArgs& a) { return (int64_t)a.pre.splits * a.c.Hkv * a.pre.tiles * a.pre.cols; }
// the item that a workgroup's i-th number stands for; one past all if there is none
__device__ __forceinline__ int item_of(const Cut& cut, int i) { return !cut.share ? i : i / 8 < cut.share ? i % 8 * cut.share + i / 8 : 1 << 30; }
__device__ __forceinline__ bool own_item(const AttnArgs& a, const Seq& s0, Cut cut, int item, int lane, Item& t) {
  Seq s;
  int b, before;
  const int chunk = cut.chunk, groups = a.c.Hkv / cut.heads;
  if (!own_find(a, s0, chunk, item / groups, lane, s, b, before)) return false;
  const int n = item / groups, i = n - before, split = i / s.tiles, head = item % groups * cut.heads;
  if ((int64_t)(n + 1) * a.c.Hkv > a.own.most) return false;
  t = Item{(table_t)(uintptr_t)(a.b.table + (size_t)b * a.b.table_ld), head, s.first, s.rows, s.len, split * chunk, (int)min((int64_t)s.len, (int64_t)(split + 1) * chunk), i % s.tiles,
           own_places(a) + ((int64_t)n * a.c.Hkv + head) * a.own.cols, a.own.cols, true, a.pre.splits == 0 && ranges_of(s.len, chunk) == 1};
  return true;
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
// a lane's words of a token's V without what is infinite or NaN if the token lies at the edge, and whether there was any
template <bool F8, int N>
__device__ __forceinline__ bool clean_edge(uint32_t (&w)[N], bool edge) {
  constexpr uint32_t bits = F8 ? 8 : 16, mask = F8 ? 0xFFu : 0xFFFFu;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (uint32_t b = 0; b < 32; b += bits)
      if (edge && is_wild<F8>(w[i] >> b)) odd = true, w[i] &= ~(mask << b);
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
__device__ __forceinline__ const uint8_t* token_at(const AttnArgs& a, table_t tab, const uint8_t* pool, int t) {
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
// Bound by memory: over long contexts 5.7 TB/s BF16 of 8 heads (6.2 of one), 4.9 e4m3, whose rows are half as long. LDS only joins the four waves.

// neither the compiler's passes nor its scheduler move a load across
__device__ __forceinline__ void loads_stay() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

template <int D, bool F8, int NQ>
struct Narrow {
  static constexpr int NS = D / 32;               // steps of the score product
  static constexpr int VL = D / 16;               // values of a row of V a lane
  static constexpr int KW = F8 ? D / 64 : D / 32;  // 16-byte words of a row of K a lane
  static constexpr int VW = F8 ? VL / 4 : VL / 2;  // 32-bit words of a row of V a lane

  v8bf_t q[NQ][NS];
  v4f_t o[NQ][VL];
  float m[NQ], l[NQ];
  bool odd;  // see clean_edge

  struct Block {
    u32x4_t k[2][KW];
    uint32_t v[8][VW];
  };

  __device__ __forceinline__ void begin() {
    odd = false;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      m[n] = -__builtin_inff(), l[n] = 0.f;
#pragma unroll
      for (int i = 0; i < VL; ++i) o[n][i] = v4f_t{0.f, 0.f, 0.f, 0.f};
    }
  }
  // row: the lane's query (lane % 16) of set n, D values; null: none
  __device__ __forceinline__ void load_q(int n, const uint16_t* row, int g, const AttnArgs& a) {
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = F8 ? 64 * (s / 2) + 16 * g + 8 * (s % 2) : 32 * s + 8 * g;
      u32x4_t w = {0, 0, 0, 0};
      if (row) w = *reinterpret_cast<const DSGX_GLOBAL u32x4_t*>((uintptr_t)(row + d));
      q[n][s] = __builtin_bit_cast(v8bf_t, query_bits(w, a));
    }
  }
  // p0, p1: a pool at the two tiles' first tokens (wave-uniform); ko, vo: the lane's offsets, ts: bytes from token to token
  __device__ __forceinline__ static void load_k(Block& x, const uint8_t* p0, const uint8_t* p1, uint32_t ko) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < KW; ++j) x.k[a][j] = ldg_stream(a ? p1 : p0, ko + 64 * j);
  }
  __device__ __forceinline__ static void load_v(Block& x, const uint8_t* p0, const uint8_t* p1, uint32_t vo, uint32_t ts) {
#pragma unroll
    for (int a = 0; a < 2; ++a)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint8_t* p = a ? p1 : p0;
        const uint32_t at = vo + j * ts;
        uint32_t(&w)[VW] = x.v[4 * a + j];
        if constexpr (VW >= 4) {
#pragma unroll
          for (int h = 0; h < VW / 4; ++h) {
            const u32x4_t t = ldg_stream(p, at + 16 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[4 * h + i] = t[i];
          }
        } else if constexpr (VW == 2) {
          const u32x2_t t = __builtin_nontemporal_load((const DSGX_GLOBAL u32x2_t*)((const DSGX_GLOBAL uint8_t*)(uintptr_t)p + at));
          w[0] = t[0], w[1] = t[1];
        } else {
          w[0] = __builtin_nontemporal_load((const DSGX_GLOBAL uint32_t*)((const DSGX_GLOBAL uint8_t*)(uintptr_t)p + at));
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
  __device__ __forceinline__ void scores(const Block& x, float (&e)[NQ][8]) const {
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      v4f_t s[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) s[n] = v4f_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        const v8bf_t k = k_operand(x.k[a], i);
#pragma unroll
        for (int n = 0; n < NQ; ++n) s[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k, q[n][i], s[n], 0, 0, 0);
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) e[n][4 * a + i] = s[n][i];
    }
  }
  // Scores of thirty-two tokens from t0 on to the softmax's numerators, as the second product's operand. lim: the lane's query sees the
  // tokens below it; there0, there1: the tiles' pages exist; all: no lane has anything masked here (wave-uniform)
  __device__ __forceinline__ v8bf_t softmax(int n, float (&e)[8], int t0, int lim, bool there0, bool there1, bool all, float s2, int g) {
    if (!all) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (!(i < 4 ? there0 : there1) || t0 + 16 * (i / 4) + 4 * g + i % 4 >= lim) e[i] = -__builtin_inff();
    }
    float mx = fmaxf(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])), fmaxf(fmaxf(e[4], e[5]), fmaxf(e[6], e[7])));
    mx = __fmul_rn(groups_max(mx), s2);
    if (__builtin_amdgcn_ballot_w64(mx > m[n] + kSlack)) {  // (-inf + slack: the first scores move it)
      const float to = fmaxf(m[n], mx), alpha = exp2_hw(m[n] - (to == -__builtin_inff() ? 0.f : to));
      l[n] *= alpha, m[n] = to;
#pragma unroll
      for (int i = 0; i < VL; ++i) o[n][i] *= alpha;
    }
    const float base = m[n] == -__builtin_inff() ? 0.f : m[n];
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = exp2_hw(fmaf(e[i], s2, -base)), sum += e[i];
    l[n] += sum;
    const u32x4_t pw = {pack_bf16(e[0], e[1]), pack_bf16(e[2], e[3]), pack_bf16(e[4], e[5]), pack_bf16(e[6], e[7])};
    return __builtin_bit_cast(v8bf_t, pw);
  }
  // what no query sees is zero for the product; the rows' limits run from lim_lo to seen
  __device__ __forceinline__ void clean(Block& x, int t0, bool there0, bool there1, int lim_lo, int seen, int g) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
      const bool out = !(i < 4 ? there0 : there1) || t >= seen;
#pragma unroll
      for (int w = 0; w < VW; ++w) x.v[i][w] = out ? 0u : x.v[i][w];
      if (lim_lo < seen) odd |= clean_edge<F8, VW>(x.v[i], t >= lim_lo);
    }
  }
  __device__ __forceinline__ void add(const Block& x, const v8bf_t (&p)[NQ]) {
#pragma unroll
    for (int i = 0; i < VL; i += 2) {
      v8bf_t a, b;
      v_operands(x.v, i, a, b);
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        o[n][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, p[n], o[n][i], 0, 0, 0);
        o[n][i + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b, p[n], o[n][i + 1], 0, 0, 0);
      }
    }
  }
};

// Waves a SIMD that the registers leave room for, and blocks on their way a wave
template <int D, bool F8, int NQ>
constexpr int kNarrowWaves = D == 64 ? 3 : 2;
template <int D, bool F8, int NQ>
constexpr int kNarrowDepth = D == 64 ? (NQ == 2 ? 1 : F8 ? 3 : 2) : D == 128 ? (F8 ? (NQ == 1 ? 3 : 2) : NQ == 1 ? 2 : 1) : 1;

template <int D, bool F8, int NQ>
__device__ __forceinline__ void narrow(const AttnArgs& a, int mode, const Role& role) {
  const bool prefix = role.prefix;
  using N = Narrow<D, F8, NQ>;
  constexpr int VL = N::VL, LD = D + 4, COLS = 16 * NQ;
  extern __shared__ __align__(16) uint8_t tiles[];
  float* lds = reinterpret_cast<float*>(tiles);  // [4][COLS][LD] outputs, then [4][COLS] maxima and sums
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), g = lane >> 4, col = lane & 15, G = a.G;
  constexpr int esz = F8 ? 1 : 2;
  const uint32_t ts = (uint32_t)(a.c.tok_stride * esz), ko = col * ts + 16 * g, vo = 4 * g * ts + col * N::VW * 4;
  float *red_m = lds + 4 * COLS * LD, *red_l = red_m + 4 * COLS;
  Seq s0{};
  Cut cut{0, a.pre.heads};
  if (!begin_plan(a, mode, role, lane, wave, s0, cut)) return;
  for (int item = role.block;; item += role.blocks) {
    Item it;
    if (prefix) {
      bool any;
      it = prefix_item(a, role.block, any);
      if (!any) return;
    } else if (!own_item(a, s0, cut, item_of(cut, item), lane, it)) {
      return;
    }
    it = uniform(it);
    const int heads = uni(cut.heads), wph = 4 / heads, step = 32 * wph;  // waves a head, which share its tokens
    const int h = it.head + wave / wph, len = it.len, rows = it.rows, cols = rows * G, x0 = it.tile * COLS;
    const uint8_t *kh = static_cast<const uint8_t*>(a.c.k) + h * a.c.head_stride * esz, *vh = static_cast<const uint8_t*>(a.c.v) + h * a.c.head_stride * esz;
    const float s2 = F8 ? a.scale2 * a.c.ks[h] : a.scale2;
    // the limits of the tile's first and last row, and of the lane's
    const int lim_hi = it.causal ? len - rows + min(x0 + COLS - 1, cols - 1) / G + 1 : len, stop = min(it.hi, lim_hi);
    const int lim_lo = min(it.hi, it.causal ? len - rows + x0 / G + 1 : len);
    N n;
    n.begin();
    int lim[NQ];
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int x = x0 + 16 * k + col, row = x / G;
      const bool live = x < cols;
      lim[k] = !live ? 0 : min(it.hi, it.causal ? len - rows + row + 1 : len);
      n.load_q(k, live ? a.q + (size_t)(it.first + row) * a.ldq + (size_t)(h * G + x % G) * D : nullptr, g, a);
    }

    auto page_of = [&](int t) { return t < stop ? it.tab[t >> a.page_shift] : -1; };
    auto place = [&](int t, int page, bool& there) -> int64_t {  // bytes from a head's first value
      there = page >= 0 && page < a.c.npages;
      return there ? ((int64_t)page * a.c.page_stride + (int64_t)(t & (a.c.page - 1)) * a.c.tok_stride) * esz : 0;
    };
    // DEPTH blocks of tokens are on their way, each in registers of its own: a block's K registers are loaded again as soon as its scores are
    // there, its V registers after its product. The page numbers are read a step before
    constexpr int DEPTH = kNarrowDepth<D, F8, NQ>;
    typename N::Block blk[DEPTH];
    bool c0[DEPTH], c1[DEPTH];
    int t0 = it.lo + 32 * (wave % wph);
    if (t0 < stop) {
      int64_t at0 = 0, at1 = 0;
#pragma unroll
      for (int s = 0; s < DEPTH; ++s) {
        const int t = t0 + step * s;
        const int64_t n0 = place(t, page_of(t), c0[s]), n1 = place(t + 16, page_of(t + 16), c1[s]);
        const bool in = t < stop;  // (else one line of the block before)
        at0 = in ? n0 : at0, at1 = in ? n1 : at1;
        const uint32_t ks = in ? ko : 0u, vo_s = in ? vo : 0u, ts_s = in ? ts : 0u;
        N::load_k(blk[s], kh + at0, kh + at1, ks);
        loads_stay();  // (issued in the loop's order, or its waits are for more than they need)
        N::load_v(blk[s], vh + at0, vh + at1, vo_s, ts_s);
        loads_stay();
      }
      int ahead0 = page_of(t0 + step * DEPTH), ahead1 = page_of(t0 + step * DEPTH + 16);
      // (no way out between the blocks of a turn: it would make the waits at the turn's start those of the shortest way there)
      for (; t0 < stop; t0 += step * DEPTH) {
#pragma unroll
        for (int s = 0; s < DEPTH; ++s) {
          const int t = t0 + step * s, tn = t + step * DEPTH;
          const bool more = tn < stop, all = c0[s] && c1[s] && t + 32 <= lim_lo;
          bool n0 = false, n1 = false;
          // (after the last block the registers are loaded from one line of it: every turn issues the same loads)
          if (more) at0 = place(tn, ahead0, n0), at1 = place(tn + 16, ahead1, n1);
          const uint32_t kn = more ? ko : 0u, vn = more ? vo : 0u, tsn = more ? ts : 0u;
          float e[NQ][8];
          n.scores(blk[s], e);
          loads_stay();
          N::load_k(blk[s], kh + at0, kh + at1, kn);
          ahead0 = page_of(tn + step), ahead1 = page_of(tn + step + 16);
          loads_stay();
          if (s == 0 || t < stop) {
            v8bf_t p[NQ];
#pragma unroll
            for (int k = 0; k < NQ; ++k) p[k] = n.softmax(k, e[k], t, lim[k], c0[s], c1[s], all, s2, g);
            if (!all) n.clean(blk[s], t, c0[s], c1[s], lim_lo, stop, g);
            n.add(blk[s], p);
          }
          loads_stay();
          N::load_v(blk[s], vh + at0, vh + at1, vn, tsn);
          loads_stay();
          c0[s] = n0, c1[s] = n1;
        }
      }
    }
    if (__builtin_amdgcn_ballot_w64(n.odd)) {
#pragma unroll 1
      for (int t = max(it.lo, lim_lo); t < stop; ++t) {
        if (((t - it.lo) >> 5) % wph != wave % wph) continue;
        const uint8_t* v = token_at<F8>(a, it.tab, vh, t);
        if (!v) continue;
#pragma unroll
        for (int k = 0; k < NQ; ++k)
          if (t < lim[k]) {
#pragma unroll
            for (int i = 0; i < VL; ++i)
#pragma unroll
              for (int j = 0; j < 4; ++j) n.o[k][i][j] += wild_value<F8>(v, VL * (4 * g + j) + i);
          }
      }
    }

    // the four waves' parts of the answer joined
    __syncthreads();  // (what an item before this one left has been read)
#pragma unroll
    for (int k = 0; k < NQ; ++k) {
      const int c = wave * COLS + 16 * k + col;
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int m4 = 0; m4 < VL; m4 += 4)
          *reinterpret_cast<v4f_t*>(lds + c * LD + VL * (4 * g + i) + m4) = v4f_t{n.o[k][m4][i], n.o[k][m4 + 1][i], n.o[k][m4 + 2][i], n.o[k][m4 + 3][i]};
      const float l = groups_sum(n.l[k]);
      if (g == 0) red_m[c] = n.m[k], red_l[c] = l;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < heads * COLS * (D / 4); i += 256) {
      const int c = i / (D / 4) % COLS, hd = i / (COLS * (D / 4)), d = 4 * (i % (D / 4)), x = x0 + c, w0 = hd * wph;
      if (x >= cols) continue;
      float mm = -__builtin_inff(), l = 0.f;
      for (int k = w0; k < w0 + wph; ++k) mm = fmaxf(mm, red_m[k * COLS + c]);
      const float base = mm == -__builtin_inff() ? 0.f : mm;
      v4f_t acc = {0.f, 0.f, 0.f, 0.f};
      for (int k = w0; k < w0 + wph; ++k) {
        const float w = exp2_hw(red_m[k * COLS + c] - base);
        l = fmaf(w, red_l[k * COLS + c], l);
        const v4f_t v = *reinterpret_cast<const v4f_t*>(lds + (k * COLS + c) * LD + d);
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = fmaf(w, v[j], acc[j]);
      }
      if (it.alone) {
        const int row = it.first + x / G, head = (it.head + hd) * G + x % G;
        const float vs = F8 ? a.c.vs[it.head + hd] : 1.f, inv = l == 0.f ? 0.f : __fdiv_rn(vs, l);
        *reinterpret_cast<uint2*>(a.out + (size_t)row * a.ldo + (size_t)head * D + d) = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
        if (d == 0 && a.lse) a.lse[(size_t)row * a.Hq + head] = l == 0.f ? -__builtin_inff() : (mm + __builtin_amdgcn_logf(l)) * kLn2;
      } else {
        const int64_t at = it.place + hd * it.next + c;
        *reinterpret_cast<v4f_t*>(a.part + at * D + d) = acc;
        if (d == 0) a.ml[at] = make_float2(mm, l);
      }
    }
    if (prefix) return;
  }
}

// ---- four waves, QW query columns each, tiles of 8192 / D tokens through LDS -------------------------------------------------------
// For many columns over the same tokens (the prefix under a batch, 64 heads over one) the matrix unit is the time, and a token's K and V
// are read by four waves. A tile is staged through registers: e4m3 becomes bf16 there, and V is transposed there (four tokens by eight
// values a thread, a byte permutation a pair), so that both operands are 16-byte reads from LDS. Layouts (chunks of 16 bytes): K as rows of
// a token, V as rows of a d whose chunks hold the eight tokens that one lane's scores belong to, so that the scores are the second
// product's operand as they stand; the chunks of a row are XORed with its number, which spreads sixteen lanes' rows over all banks.
// Bound by the matrix unit and what is issued beside it: 128 columns of e4m3 keep it busy 60% of the time at the 1.7 GHz that the card then
// runs at; staging is a quarter of the rest, LDS reads are hidden four products ahead.
// QW 32 (D 64, 128): v_mfma_f32_32x32x16_bf16, 128 columns a workgroup; QW 16: v_mfma_f32_16x16x32_bf16, 64 columns.
typedef float v16f_t __attribute__((ext_vector_type(16)));

// a barrier for what passes through LDS alone: loads from memory stay on their way
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

template <int D, bool F8, int QW>
struct Wide {
  static constexpr int KV = 8192 / D;            // tokens a tile
  static constexpr int SR = QW / 16 * 4 * (QW / 16);  // accumulators of a tile a lane: 16 or 4
  static constexpr int LG = kWave / QW;          // lanes that share a column: 2 or 4
  static constexpr int KD = 8 * LG;              // k of one instruction: 16 or 32
  static constexpr int NS = D / KD, OT = D / QW;
  static constexpr int NSUB = KV / 32, TS = 32 / QW, NE = QW / 2, NP = NE / 8;  // thirty-twos of a tile; score tiles, scores a lane, products' steps of one
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
    // (D 256: the stores of a wave are of every eighth row, so the row's place among its four moves on with those: 8 rows of 64 heads over 50001
    // tokens 63.2 us instead of 67.9)
    const uint32_t row = RP == 4 ? (d & ~3u) | ((d + (d >> 3)) & 3) : d;
    return row * (CPR * 16) + ((c ^ (d / RP) ^ (RP == 4 ? d >> 5 : d >> 4)) & (CPR - 1)) * 16;
  }

  // The operands' reads as the lane's address XOR a constant, plus a constant: row QW u + col, chunk LG k + lg of a tile of K ..
  __device__ __forceinline__ static uint32_t k_read(uint32_t lane_at, int u, int k) { return (lane_at ^ (uint32_t)(LG * k * 16)) + (uint32_t)(QW * u * D * 2); }
  // .. and row QW i + col, chunk LG k + lg of one of V^T (the row's share of the XOR that i makes is i's alone: no carries)
  __device__ __forceinline__ static uint32_t v_read(uint32_t lane_at, int i, int k) {
    constexpr uint32_t CPR = KV / 8, RP = 16 / CPR;
    const uint32_t x = (uint32_t)(LG * k) ^ ((uint32_t)(QW * i / RP) & (CPR - 1)) ^ ((uint32_t)(QW * i / (RP == 4 ? 32 : 16)) & (CPR - 1));
    const uint32_t row = RP == 4 ? (uint32_t)(QW / 8 * i) & 3 : 0;  // (0 or 2: the sum is an XOR)
    return (lane_at ^ (x * 16) ^ (row * CPR * 16)) + (uint32_t)(QW * i) * (CPR * 16);
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
  __device__ __forceinline__ static void load(Stage& x, const uint8_t* kh, const uint8_t* vh, uint64_t offs, uint32_t ts, uint32_t tid, int wave) {
    // (a wave's rows of a load lie in one sixteen: its place is wave-uniform, but for V with D 64)
    auto off = [&](int sixteen) {
      const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)offs, sixteen), hi = __builtin_amdgcn_readlane((int)(offs >> 32), sixteen);
      return (uint64_t)hi << 32 | lo;
    };
#pragma unroll
    for (int i = 0; i < KN; ++i) {
      const uint32_t row = k_row(i, tid);
      x.k[i] = *(const DSGX_GLOBAL u32x4_t*)((const DSGX_GLOBAL uint8_t*)(uintptr_t)(kh + off((int)k_row(i, 64 * wave) / 16)) + ((row % 16) * ts + 16 * k_chunk(i, tid)));
    }
    const uint32_t grp = v_group(tid), dc = tid % (D / 8);
    const uint8_t* vb;
    if (D == 64) {
      const uint32_t o0 = __shfl((int)(uint32_t)offs, (int)(grp / 4)), o1 = __shfl((int)(offs >> 32), (int)(grp / 4));
      vb = vh + ((uint64_t)o1 << 32 | o0) + ((grp % 4) * 4 * ts + dc * VW * 4);
    } else {
      vb = vh + off((int)v_group(64 * wave) / 4) + ((grp % 4) * 4 * ts + dc * VW * 4);
    }
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
__device__ __forceinline__ void wide(const AttnArgs& a, int mode, const Role& role) {
  const bool prefix = role.prefix;
  using W = Wide<D, F8, QW>;
  using acc_t = typename W::acc_t;
  constexpr int KV = W::KV, COLS = 4 * QW;
  extern __shared__ __align__(16) uint8_t tiles[];  // two tiles of K and V each
  __shared__ int any_odd;
  const uint32_t tid = threadIdx.x, lane = tid & 63;
  const int wave = uni((int)tid >> 6), lg = lane / QW, col = lane % QW;
  constexpr int esz = F8 ? 1 : 2;
  const uint32_t ts = (uint32_t)(a.c.tok_stride * esz);
  Seq s0{};
  Cut cut{0, a.pre.heads};
  if (!begin_plan(a, mode, role, lane, wave, s0, cut)) return;
  for (int item = role.block;; item += role.blocks) {
    Item it;
    if (prefix) {
      bool any;
      it = prefix_item(a, role.block, any);
      if (!any) return;
    } else if (!own_item(a, s0, cut, item_of(cut, item), lane, it)) {
      return;
    }
    it = uniform(it);
    const int h = it.head, len = it.len, rows = it.rows, G = a.G, cols = rows * G, x0 = it.tile * COLS, lo = it.lo, first = it.first;
    const table_t tab = it.tab;
    const uint8_t *kh = static_cast<const uint8_t*>(a.c.k) + h * a.c.head_stride * esz, *vh = static_cast<const uint8_t*>(a.c.v) + h * a.c.head_stride * esz;
    const float s2 = F8 ? a.scale2 * a.c.ks[h] : a.scale2, vs = F8 ? a.c.vs[h] : 1.f;
    const int x = x0 + wave * QW + col, row = x / G, head = h * G + x % G;
    const bool live = x < cols;
    const int lim_hi = it.causal ? len - rows + min(x0 + COLS - 1, cols - 1) / G + 1 : len, stop = min(it.hi, lim_hi);
    const int lim_lo = min(it.hi, it.causal ? len - rows + x0 / G + 1 : len);
    const int lim = !live ? 0 : min(it.hi, it.causal ? len - rows + row + 1 : len);
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
    auto page_of = [&](int t0) { return tab[min(t0 + 16 * (int)lane, stop - 1) >> a.page_shift]; };  // (asked for with stop > 0 alone)
    auto place = [&](int t0, int page, uint32_t& there) {
      const int t = t0 + 16 * (int)lane;
      const bool ok = (int)lane < KV / 16 && t < stop && page >= 0 && page < a.c.npages;
      there = (uint32_t)__builtin_amdgcn_ballot_w64(ok);
      return ok ? (uint64_t)(((int64_t)page * a.c.page_stride + (int64_t)(t & (a.c.page - 1)) * a.c.tok_stride) * esz) : 0ull;
    };
    constexpr uint32_t kAll = (1u << (KV / 16)) - 1;
    bool odd = false;  // see clean_edge
    auto clean = [&](typename W::Stage& st, int t0, uint32_t there) {
      const uint32_t grp = W::v_group(tid);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int t = t0 + 4 * (int)grp + j;
        const bool out = !(there >> (grp / 4) & 1) || t >= stop;
#pragma unroll
        for (int w = 0; w < W::VW; ++w) st.v[j][w] = out ? 0u : st.v[j][w];
        if (lim_lo < stop) odd |= clean_edge<F8, W::VW>(st.v[j], t >= lim_lo);
      }
    };

    // Thirty-two tokens at a time: while the matrix unit makes the next ones' scores, the vector unit makes these ones' numerators. A tile's
    // successor is stored in its second half of LDS after everyone is done with the tile before (the turn's first barrier) and read
    // after the second; the successor's successor is on its way in registers.
    const uint32_t k_at = W::k_addr(col, lg), v_at = W::v_addr(col, lg);
    auto scores = [&](const uint8_t* kt, uint32_t ka, int j, float (&e)[W::NE]) {
      acc_t s[W::TS];
#pragma unroll
      for (int u = 0; u < W::TS; ++u)
#pragma unroll
        for (int i = 0; i < W::SR; ++i) s[u][i] = 0.f;
#pragma unroll
      for (int k = 0; k < W::NS; ++k)
#pragma unroll
        for (int u = 0; u < W::TS; ++u)
          s[u] = W::mfma(__builtin_bit_cast(v8bf_t, *reinterpret_cast<const u32x4_t*>(kt + W::k_read(ka, W::TS * j + u, k))), q[k], s[u]);
#pragma unroll
      for (int u = 0; u < W::TS; ++u)
#pragma unroll
        for (int i = 0; i < W::SR; ++i) e[u * W::SR + i] = s[u][i];
    };
    auto fetch = [&](typename W::Stage& st, int t0, int page, uint32_t& there) {
      const uint64_t at = place(t0, page, there);
      W::load(st, kh, vh, at, ts, tid, wave);
    };
    typename W::Stage st;
    uint32_t there = 0, there1 = 0, there2 = 0;  // of the tile, the next, the one after
    float e[W::NE];
    lds_barrier();  // (the tiles of an item before this one have been read)
    if (lo < stop) {
      int ahead = page_of(lo + KV);
      fetch(st, lo, page_of(lo), there);
      if (there != kAll || lo + KV > lim_lo) clean(st, lo, there);
      W::store(st, tiles, tiles + W::kTile, tid);
      fetch(st, lo + KV, ahead, there1);
      ahead = page_of(lo + 2 * KV);
      lds_barrier();
      scores(tiles, k_at, 0, e);
      int buf = 0;
      for (int t0 = lo; t0 < stop; t0 += KV, buf ^= 1) {
        const uint8_t *kt = tiles + buf * 2 * W::kTile, *vt = kt + W::kTile;
        uint8_t* nt = tiles + (buf ^ 1) * 2 * W::kTile;
        uint32_t ka = k_at, va = v_at;
        asm volatile("" : "+v"(ka), "+v"(va));  // (else every operand's address is kept in a register of its own)
        if (there1 != kAll || t0 + 2 * KV > lim_lo) clean(st, t0 + KV, there1);
        const bool all = there == kAll && t0 + KV <= lim_lo;
        lds_barrier();
#pragma unroll
        for (int j = 0; j < W::NSUB; ++j) {
          if (!all) {
#pragma unroll
            for (int i = 0; i < W::NE; ++i) {
              const int tk = 32 * j + W::token_of(i, lg);
              if (!(there >> (tk / 16) & 1) || t0 + tk >= lim) e[i] = -__builtin_inff();
            }
          }
          float mx = e[0];
#pragma unroll
          for (int i = 1; i < W::NE; ++i) mx = fmaxf(mx, e[i]);
          mx = __fmul_rn(column_max<QW>(mx), s2);
          if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {  // (-inf + slack: the first scores move it)
            const float to = fmaxf(m, mx), base = to == -__builtin_inff() ? 0.f : to, alpha = exp2_hw(m - base);
            l *= alpha, m = to;
#pragma unroll
            for (int i = 0; i < W::OT; ++i)
#pragma unroll
              for (int k = 0; k < W::SR; ++k) o[i][k] *= alpha;
          }
          const float base = m == -__builtin_inff() ? 0.f : m;
          if (j == 0) {
            W::store(st, nt, nt + W::kTile, tid);
            fetch(st, t0 + 2 * KV, ahead, there2);  // (past the end: a tile of page 0, which is not looked at)
            ahead = page_of(t0 + 3 * KV);
          }
          // The products of the next thirty-two's scores (M1), then of these numerators with V (M2), each with its share of the vector unit's
          // work beside it, the operands read from LDS four products ahead. (sched_barrier: left to itself the compiler reads an operand
          // right before its product, and every product waits for LDS.)
          constexpr int M1 = W::NS * W::TS, M2 = W::NP * W::OT, PAIRS = W::NE / 2;
          if (j == W::NSUB - 1) lds_barrier();
          const uint8_t* kn = j < W::NSUB - 1 ? kt : nt;
          auto operand = [&](int i) {
            return i < M1 ? *reinterpret_cast<const u32x4_t*>(kn + W::k_read(ka, (j < W::NSUB - 1 ? W::TS * (j + 1) : 0) + i % W::TS, i / W::TS))
                          : *reinterpret_cast<const u32x4_t*>(vt + W::v_read(va, (i - M1) % W::OT, W::NP * j + (i - M1) / W::OT));
          };
          u32x4_t ring[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) ring[i] = operand(i);
          acc_t s[W::TS];
#pragma unroll
          for (int u = 0; u < W::TS; ++u)
#pragma unroll
            for (int i = 0; i < W::SR; ++i) s[u][i] = 0.f;
          uint32_t pw[PAIRS];
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < M1 + M2; ++i) {
            if (i < M1) s[i % W::TS] = W::mfma(__builtin_bit_cast(v8bf_t, ring[i % 4]), q[i / W::TS], s[i % W::TS]);
            else {
              const int k = (i - M1) / W::OT, ot = (i - M1) % W::OT;
              o[ot] = W::mfma(__builtin_bit_cast(v8bf_t, ring[i % 4]), __builtin_bit_cast(v8bf_t, u32x4_t{pw[4 * k], pw[4 * k + 1], pw[4 * k + 2], pw[4 * k + 3]}), o[ot]);
            }
            if (i + 4 < M1 + M2) ring[i % 4] = operand(i + 4);
            if (i < M1) {
#pragma unroll
              for (int w = i * PAIRS / M1; w < (i + 1) * PAIRS / M1; ++w) {
                const float p0 = exp2_hw(fmaf(e[2 * w], s2, -base)), p1 = exp2_hw(fmaf(e[2 * w + 1], s2, -base));
                l += p0, l += p1;
                pw[w] = pack_bf16(p0, p1);
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
#pragma unroll
          for (int u = 0; u < W::TS; ++u)
#pragma unroll
            for (int i = 0; i < W::SR; ++i) e[u * W::SR + i] = s[u][i];
        }
        there = there1, there1 = there2;
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
    if (live && it.alone) {
      const float inv = l == 0.f ? 0.f : __fdiv_rn(vs, l);
      uint16_t* dst = a.out + (size_t)(first + row) * a.ldo + (size_t)head * D;
#pragma unroll
      for (int i = 0; i < W::OT; ++i)
#pragma unroll
        for (int j = 0; j < W::SR; j += 4)
          *reinterpret_cast<uint2*>(dst + QW * i + W::LG * j + 4 * lg) = make_uint2(pack_bf16(o[i][j] * inv, o[i][j + 1] * inv), pack_bf16(o[i][j + 2] * inv, o[i][j + 3] * inv));
      if (lg == 0 && a.lse) a.lse[(size_t)(first + row) * a.Hq + head] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
    } else if (live) {
      const int64_t at = it.place + wave * QW + col;
      float* dst = a.part + at * D;
#pragma unroll
      for (int i = 0; i < W::OT; ++i)
#pragma unroll
        for (int j = 0; j < W::SR; j += 4) *reinterpret_cast<v4f_t*>(dst + QW * i + W::LG * j + 4 * lg) = v4f_t{o[i][j], o[i][j + 1], o[i][j + 2], o[i][j + 3]};
      if (lg == 0) a.ml[at] = make_float2(m, l);
    }
    if (prefix) return;
  }
}

template <int D, bool F8, int NQ>
__global__ void __launch_bounds__(256, (kNarrowWaves<D, F8, NQ>)) k_attn_narrow(AttnArgs a, int mode) {
  narrow<D, F8, NQ>(a, mode, role_of(a, mode));
}
template <int D, bool F8, int QW>
__global__ void __launch_bounds__(256, 2) k_attn_wide(AttnArgs a, int mode) {
  wide<D, F8, QW>(a, mode, role_of(a, mode));
}
// The prefix with 128 columns a workgroup and the sequences' own tokens with 16 NQ, in one launch
template <int D, bool F8, int NQ>
__global__ void __launch_bounds__(256, 2) k_attn_both(AttnArgs a) {
  const Role role = role_of(a, kBoth);
  if (role.prefix) wide<D, F8, 32>(a, kBoth, role);
  else narrow<D, F8, NQ>(a, kBoth, role);
}

// The ranges' outputs of a row's head joined by their maxima: WPH waves a head, D / 4 lanes a range
template <int D, int WPH>
__global__ void __launch_bounds__(WPH > 4 ? 64 * WPH : 256) k_combine(AttnArgs a) {
  constexpr int LR = D / 4, RW = kWave / LR, STEP = RW * WPH;  // lanes a range, ranges a wave, ranges a turn
  constexpr int WAVES = WPH > 4 ? WPH : 4;
  __shared__ v4f_t racc[WAVES][LR];
  __shared__ float rl[WAVES], rm[WAVES];
  const int lane = threadIdx.x & 63, wave = uni((int)threadIdx.x >> 6), part = wave % WPH, r = blockIdx.x, head = (int)blockIdx.y * (WAVES / WPH) + wave / WPH;
  const int chunk = uni(a.plan[0]);
  // the row's sequence
  Seq s{0, 0, 0, 0};
  int before = 0;
  bool found = false;
  for (int j0 = 0; j0 < a.b.B && !found; j0 += kWave) {
    const Seq t = seq_of(a, j0 + lane);
    const int first = j0 + lane < a.b.B ? a.plan[4 + j0 + lane] : 0;
    const uint64_t hit = __builtin_amdgcn_ballot_w64(t.rows > 0 && t.first <= r && r < t.first + t.rows);
    if (hit) {
      const int l = __builtin_ctzll(hit);
      before = __builtin_amdgcn_readlane(first, l), found = true;
      s = Seq{__builtin_amdgcn_readlane(t.first, l), __builtin_amdgcn_readlane(t.rows, l), __builtin_amdgcn_readlane(t.len, l), __builtin_amdgcn_readlane(t.tiles, l)};
    }
  }
  const int own = ranges_of(s.len, chunk);
  if (!found || (a.pre.splits == 0 && own == 1)) return;  // (the same for the whole workgroup)
  const bool live = head < a.Hq;
  const int h = (live ? head : 0) / a.G, px = r * a.G + head % a.G, ox = (r - s.first) * a.G + head % a.G;
  const int n = live ? a.pre.splits + own : 0;
  auto place_of = [&](int i) -> int64_t {
    if (i < a.pre.splits) return (int64_t)((i * a.c.Hkv + h) * a.pre.tiles + px / a.pre.cols) * a.pre.cols + px % a.pre.cols;
    const int item = (before + (i - a.pre.splits) * s.tiles + ox / a.own.cols) * a.c.Hkv + h;
    return item < a.own.most ? own_places(a) + (int64_t)item * a.own.cols + ox % a.own.cols : -1;
  };
  const int sub = lane / LR, d = 4 * (lane % LR);
  v4f_t acc = {0.f, 0.f, 0.f, 0.f};
  float m = -__builtin_inff(), l = 0.f;
  constexpr int U = 4;  // ranges in flight a lane
  for (int i0 = part * RW + sub; i0 < n; i0 += U * STEP) {
    float2 ml[U];
    v4f_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * STEP;
      const int64_t at = i < n ? place_of(i) : -1;
      ml[u] = at >= 0 ? a.ml[at] : make_float2(-__builtin_inff(), 0.f);
      v[u] = at >= 0 ? *reinterpret_cast<const v4f_t*>(a.part + at * D + d) : v4f_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float to = fmaxf(m, ml[u].x), base = to == -__builtin_inff() ? 0.f : to, w0 = exp2_hw(m - base), w1 = exp2_hw(ml[u].x - base);
      m = to, l = fmaf(l, w0, ml[u].y * w1);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[j] = fmaf(acc[j], w0, v[u][j] * w1);
    }
  }
  auto join = [&](float om, float ol, v4f_t ov) {
    const float to = fmaxf(m, om), base = to == -__builtin_inff() ? 0.f : to, w0 = exp2_hw(m - base), w1 = exp2_hw(om - base);
    m = to, l = fmaf(l, w0, ol * w1);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = fmaf(acc[j], w0, ov[j] * w1);
  };
#pragma unroll
  for (int k = LR; k < kWave; k <<= 1) {
    v4f_t ov;
#pragma unroll
    for (int j = 0; j < 4; ++j) ov[j] = __shfl_xor(acc[j], k);
    join(__shfl_xor(m, k), __shfl_xor(l, k), ov);
  }
  if (WPH > 1) {
    if (sub == 0) racc[wave][lane] = acc;
    if (lane == 0) rm[wave] = m, rl[wave] = l;
    __syncthreads();
    if (part) return;
#pragma unroll
    for (int k = 1; k < WPH; ++k) join(rm[wave + k], rl[wave + k], racc[wave + k][lane % LR]);
  }
  if (!live || sub) return;
  const float vs = a.c.fmt == DSGX_KV_E4M3 ? a.c.vs[h] : 1.f, inv = l == 0.f ? 0.f : __fdiv_rn(vs, l);
  *reinterpret_cast<uint2*>(a.out + (size_t)r * a.ldo + (size_t)head * D + d) = make_uint2(pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv));
  if (lane == 0 && a.lse) a.lse[(size_t)r * a.Hq + head] = l == 0.f ? -__builtin_inff() : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

int round_up(int64_t v, int m) { return (int)((v + m - 1) / m * m); }

// How `cols` query columns over the same tokens are worked on: 16 or 32 a workgroup from registers, 64 or 128 over tiles in LDS.
// 128 against 64, D 128: 6 x 8 rows of 16 heads over each of 4, 5000 to 8000 tokens 33.5 us, 37.2; 8011 tokens before 48 rows of 64 heads over 8 28.8, 36.2.
// D 256 by 128 columns takes over half a SIMD's registers, and its one wave a SIMD waits for whatever it waits for: 5 rows of 64 heads over
// one, 50001 tokens 53.2 us (e4m3 51.9), by 64 columns 50.1 (43.0; both before tiles over the same tokens shared an XCD). By 16 from registers it
// is so too for BF16: 16 rows of 8 heads over each of 2, 300 to 8000 tokens 28.7 us, by 64 columns 23.5 (e4m3 18.0, 22.8); and behind a prefix
// one launch has both.
enum Kind { kNarrow16, kNarrow32, kWide64, kWide128 };
Kind kind_of(int64_t cols, int D, bool f8, bool prefix) {
  if (D == 256) return cols <= 16 && f8 && !prefix ? kNarrow16 : kWide64;
  return cols <= 16 ? kNarrow16 : cols <= 32 ? kNarrow32 : cols <= 64 ? kWide64 : kWide128;
}
int cols_of(Kind k) { return 16 << k; }
// workgroups a CU holds
int resident(Kind k, int D) {
  return k <= kNarrow32 && D == 64 ? 3 : 2;
}

// Heads side by side a workgroup of the register kernels: their tokens' rows are neighbours in the usual layout of a page
int heads_of(Kind k, const dsgx_kv_cache& c) {
  return k > kNarrow32 || c.head_stride > c.tok_stride ? 1 : c.Hkv % 4 == 0 ? 4 : c.Hkv % 2 == 0 ? 2 : 1;
}

struct Layout {
  Kind kp, ko;
  Part pre;
  Own own;
  int own_grid;
  bool both;  // prefix and own tokens in one launch
  size_t ml, part, plan;  // bytes
};
Layout make_layout(const dsgx_kv_cache& c, const dsgx_kv_batch& b, int Hq) {
  const int G = Hq / c.Hkv, cus = num_cus_cached();
  const bool f8 = c.fmt == DSGX_KV_E4M3;
  Layout y{};
  int64_t slots = 0;
  y.ko = kind_of((int64_t)b.max_rows * G, c.D, f8, b.prefix_len > 0);
  if (b.prefix_len) {
    y.kp = kind_of((int64_t)b.rows * G, c.D, f8, true);
    // A wider form than the columns ask for, so that one launch can have both. Own tokens of 12 x 2 rows by 32 columns behind 3000 tokens: 40.4 us in
    // two launches, 27.2 in one. The prefix by 128 columns for 56: 3000 tokens 25.0 us, 14.3; 25000 41.4, 33.0 (e4m3 34.6, 27.4); 60000 70.0, 68.9
    // (e4m3 52.2, 61.8).
    if (y.kp == kNarrow32 && b.max_len <= 32768) y.ko = kNarrow32;
    if (y.kp == kWide64 && y.ko <= kNarrow32 && b.prefix_len <= 32768) y.kp = kWide128;
  }
  y.own.cols = cols_of(y.ko), y.own.heads = heads_of(y.ko, c), y.own.tiles = (int)(((int64_t)b.max_rows * G + y.own.cols - 1) / y.own.cols);
  int room = cus * resident(y.ko, c.D);
  if (b.prefix_len) {
    const int64_t cols = (int64_t)b.rows * G;
    y.pre.cols = cols_of(y.kp), y.pre.tiles = (int)((cols + y.pre.cols - 1) / y.pre.cols);
    y.pre.heads = heads_of(y.kp, c);
    const int64_t each = (int64_t)(c.Hkv / y.pre.heads) * y.pre.tiles;
    y.both = y.kp == y.ko || (y.kp == kWide128 && y.ko <= kNarrow32);
    double pre_room = cus * resident(y.kp, c.D);
    // (8011 tokens before 48 rows: at least half of it for the prefix 36.1 us, two thirds 35.4, four fifths 39.5.)
    // In one launch the room is shared by the work (tokens times tiles; of max_len half, on average), two thirds at least for the prefix, whose
    // ranges are cut here; what is left of it is the own tokens', or all of it where they are most of the work and come second.
    const double mine = 0.5 * b.B * b.max_len * (((int64_t)b.max_rows * G + y.own.cols - 1) / y.own.cols), theirs = (double)b.prefix_len * y.pre.tiles;
    if (y.both) room = std::min(room, (int)pre_room), pre_room = room * std::max(2. / 3, theirs / (theirs + mine));
    const int64_t splits = std::max<int64_t>(1, (int64_t)(pre_room / each + (y.both ? 0.5 : 0)));
    y.pre.chunk = std::max(256, round_up((b.prefix_len + splits) / splits, 128));
    y.pre.splits = (b.prefix_len + y.pre.chunk - 1) / y.pre.chunk;
    slots = each * y.pre.heads * y.pre.splits * y.pre.cols;
    if (y.both && mine < 2 * theirs) room = (int)std::max((int64_t)room / 3, room - each * y.pre.splits);
  }
  // short contexts without a prefix: a range a sequence, which leaves nothing to join
  y.own.target = !b.prefix_len && b.max_len <= 512 ? 0 : room, y.own.least = 256;
  const int64_t most = 4 * (int64_t)y.own.target * y.own.heads + (int64_t)c.Hkv * (((int64_t)b.rows * G) / y.own.cols + b.B + 1);
  y.own.most = (int)std::min<int64_t>(most, 1 << 30);
  y.own_grid = (int)std::min<int64_t>(room, most);
  slots += (int64_t)y.own.most * y.own.cols;
  y.ml = align256((size_t)slots * sizeof(float2)), y.part = align256((size_t)slots * c.D * 4), y.plan = align256((size_t)(b.B + 4) * 4);
  return y;
}

template <int D, bool F8>
size_t lds_of(Kind k) {
  return k <= kNarrow32 ? (size_t)(4 * cols_of(k) * (D + 4) + 8 * cols_of(k)) * 4 : 4 * Wide<D, F8, 16>::kTile;
}
template <int D, bool F8>
int launch_part(const AttnArgs& a, Kind k, unsigned grid, Mode mode, hipStream_t st) {
  const size_t lds = lds_of<D, F8>(k);
  void (*kern)(AttnArgs, int);
  if constexpr (D == 256 && F8) kern = k == kNarrow16 ? k_attn_narrow<D, F8, 1> : k_attn_wide<D, F8, 16>;
  else if constexpr (D == 256) kern = k_attn_wide<D, F8, 16>;
  else kern = k == kNarrow16 ? k_attn_narrow<D, F8, 1> : k == kNarrow32 ? k_attn_narrow<D, F8, 2> : k == kWide64 ? k_attn_wide<D, F8, 16> : k_attn_wide<D, F8, 32>;
  if (int rc = allow_dynamic_lds((const void*)kern, lds)) return rc;
  hipLaunchKernelGGL(kern, dim3(grid), dim3(256), lds, st, a, (int)mode);
  DSGX_HIP(hipGetLastError());
  return DSGX_OK;
}
template <int D, bool F8>
int launch_both(const AttnArgs& a, Kind ko, unsigned grid, hipStream_t st) {
  if constexpr (D < 256) {
    const size_t lds = std::max(lds_of<D, F8>(kWide128), lds_of<D, F8>(ko));
    auto kern = ko == kNarrow16 ? k_attn_both<D, F8, 1> : k_attn_both<D, F8, 2>;
    if (int rc = allow_dynamic_lds((const void*)kern, lds)) return rc;
    hipLaunchKernelGGL(kern, dim3(grid), dim3(256), lds, st, a);
    DSGX_HIP(hipGetLastError());
  }
  return DSGX_OK;
}
// One launch for prefix and own tokens where one kernel has both their forms: a launch's ramp and its first chain of loads take about 10 us.
// 8011 tokens before 48 rows of 64 heads: 49.9 us in two launches, 35.7 in one; 32768 before 300 of 32 (e4m3): 262, 240; 5000 before 2 of 32: 31.4, 20.0;
// 9000 before 20 of 16 heads of 256 over one: 45.9, 19.3.
template <int D, bool F8>
int launch(AttnArgs& a, const Layout& y, hipStream_t st) {
  const unsigned own = ((unsigned)y.own_grid + 7) / 8 * 8;  // (more than there are items do nothing)
  if (a.pre.splits) {
    const int64_t pairs = (int64_t)a.pre.splits * (a.c.Hkv / a.pre.heads);
    const unsigned pre = (unsigned)((pairs * a.pre.tiles + 7) / 8 * 8);
    a.pre_blocks = (int)pre;
    if (y.kp == y.ko) {
      if (int rc = launch_part<D, F8>(a, y.kp, pre + own, kBoth, st)) return rc;
    } else if (y.both) {
      if (int rc = launch_both<D, F8>(a, y.ko, pre + own, st)) return rc;
    } else {
      if (int rc = launch_part<D, F8>(a, y.kp, pre + 1, kPrefixOnly, st)) return rc;
      if (int rc = launch_part<D, F8>(a, y.ko, own, kOwnOnly, st)) return rc;
    }
  } else {
    if (int rc = launch_part<D, F8>(a, y.ko, own, kOwnOnly, st)) return rc;
  }
  if (!a.pre.splits && !a.own.target) return DSGX_OK;
  // Waves a head, by how many heads there are and about how many ranges each has: 128 ranges of 32 heads of 256 values 14.5 us by four waves, 7.4
  // by eight, 7.6 by sixteen; 102 of 320 heads 9.8, 9.5, 13.9; 16 of 256 heads 4.8 by four, 5.9 by sixteen.
  const int64_t ranges = a.pre.splits + std::min<int64_t>(a.b.max_len / a.own.least, (int64_t)a.own.target * a.own.heads / ((int64_t)a.c.Hkv * a.b.B));
  if ((int64_t)a.b.rows * a.Hq <= 512 && ranges > 32) hipLaunchKernelGGL((k_combine<D, 8>), dim3(a.b.rows, a.Hq), dim3(512), 0, st, a);
  else if ((int64_t)a.b.rows * a.Hq <= 1024) hipLaunchKernelGGL((k_combine<D, 4>), dim3(a.b.rows, a.Hq), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((k_combine<D, 1>), dim3(a.b.rows, (a.Hq + 3) / 4), dim3(256), 0, st, a);
  DSGX_HIP(hipGetLastError());
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
  // At least every layout's, whatever lengths and prefix, and growing with sequences and rows: a program's largest batch sizes it. Columns of
  // places: own items are 4 target + one a tile and sequence (own_plan's chunk is the work's share of the room at least), the prefix's
  // workgroups the room + one a tile and head.
  const int64_t cols = (int64_t)batch->rows * (Hq / cache->Hkv);
  int64_t room = 0;
  for (int k = kNarrow16; k <= kWide128; ++k) room = std::max(room, (int64_t)num_cus_cached() * resident((Kind)k, cache->D) * heads_of((Kind)k, *cache) * cols_of((Kind)k));
  const size_t slots = (size_t)(5 * room + cache->Hkv * (2 * cols + ((int64_t)batch->B + 2) * cols_of(kWide128)));
  return align256(slots * sizeof(float2)) + align256(slots * cache->D * 4) + align256((size_t)(batch->B + 4) * 4);
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
  const Layout y = make_layout(*cache, *batch, Hq);
  a.c = *cache, a.b = *batch, a.pre = y.pre, a.own = y.own;
  a.q = q, a.out = out, a.lse = lse, a.ldq = ldq, a.ldo = ldo, a.Hq = Hq, a.G = Hq / cache->Hkv, a.page_shift = __builtin_ctz((unsigned)cache->page);
  a.scale2 = scale == 0.f ? 1.f : std::fabs(scale) * kLog2e, a.q_flip = scale < 0.f ? 0x80008000u : 0u, a.q_keep = scale == 0.f ? 0u : 0xFFFFFFFFu;
  a.ml = static_cast<float2*>(ws);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + y.ml);
  a.plan = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(ws) + y.ml + y.part);
  hipStream_t st = static_cast<hipStream_t>(stream);
  const bool f8 = cache->fmt == DSGX_KV_E4M3;
  switch (cache->D) {
    case 64: return f8 ? launch<64, true>(a, y, st) : launch<64, false>(a, y, st);
    case 128: return f8 ? launch<128, true>(a, y, st) : launch<128, false>(a, y, st);
    default: return f8 ? launch<256, true>(a, y, st) : launch<256, false>(a, y, st);
  }
}
