// Attention of new tokens over a KV cache in pages of 8-bit codes.
//
// Sequence b has len committed tokens and count new ones, whose keys and values are in the
// slots behind them. Slot x is row x % page of page tables[b, x / page]; its key is
// code * k_scale, its value code * v_scale, with one power-of-two scale for a head's page.
// New token t sees the slots in [max(0, len + t - window), len + t] that have a page:
//
//   s = scale q . k,  o = sum exp(s - m) v / l,  l = sum exp(s - m),  lse = m + log l
//
// in one pass over the pages, m and l running. Codes become bf16, exactly (four bits and a
// power of two), on their way into the matrix cores; what has more bits goes in as a sum of
// bf16 pieces: q and the probabilities of fp16 as two, of fp32 as three, so the only
// roundings are those of the probabilities to the sum of their pieces and of fp32 sums.
#include <algorithm>
#include <type_traits>

#include "attn_mfma.hpp"
#include "paged.hpp"

namespace sfl {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPagedWaves = 4;
constexpr int kPagedTile = 64;  // keys of a wave's tile
constexpr int kMaxTokens = 128;
constexpr float kLn2 = 0.6931471805599453f;

struct PagedArgs {
  const void* q;
  const uint8_t *k, *v;
  const float *k_scale, *v_scale;
  const int32_t *tables, *lengths, *counts;
  float *pmax, *psum, *pout;
  void* out;
  float* lse;
  long qs[3], os[3];  // strides in elements: batch, head, token
  int kv_heads, places, pages, page_log2, tokens, group_log2, row_blocks, splits, groups;
  int window;  // slots before its own that a token sees; < 0: all
  float cs;    // scale * log2(e): scores are kept in base 2
};

template <typename T> constexpr int pieces_of() { return std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, f16_t>::value ? 2 : 3; }

// What a sequence has: committed tokens, new ones in use, slots.
struct PagedRow {
  int len, count, cap;
};
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& a, int b) {
  typedef const __attribute__((address_space(4))) int32_t* Constant;  // read by scalar loads
  b = __builtin_amdgcn_readfirstlane(b);
  PagedRow r;
  r.cap = a.places << a.page_log2;
  r.len = min(max(Constant(a.lengths)[b], 0), r.cap);
  r.count = a.counts ? min(max(Constant(a.counts)[b], 0), a.tokens) : a.tokens;
  r.count = min(r.count, r.cap - r.len);  // tokens that have a slot
  return r;
}

__device__ __forceinline__ f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Eight codes as bf16 values under a scale.
__device__ __forceinline__ u32x4 from_codes(uint32_t lo, uint32_t hi, float scale) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true))};
}

// 0xff in each byte of w that is the code of NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
  const uint32_t t = (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7;
  return (t << 8) - t;
}
// The first n bytes of a word.
__device__ __forceinline__ uint32_t first_bytes(int n) { return n <= 0 ? 0u : n >= 4 ? ~0u : (1u << (8 * n)) - 1; }

// A wave's tile of 64 keys, lane = 16 g + n. MFMA t (0..3) of S^T = K Q^T takes as its row
// 4 g' + i the key 16 g' + 4 t + i, so that lane (g, n) comes to hold the scores of the keys
// 16 g .. 16 g + 15 of query row n, which is what O^T += V^T P^T takes as the k-slots of
// lane group g: probabilities never leave their lane, and the lane's codes of V^T, 16 keys
// of a dim, are 16 bytes of the page's [D, page]. A lane's keys lie in one page (pages hold
// a multiple of 16), for K that of key 16 (n / 4), for V and the scores that of key 16 g.
template <int D>
struct Tile {
  static constexpr int kSteps = (D + 31) / 32;  // of 32 dims in the products with K
  static constexpr int kDims = D / 16;          // tiles of 16 dims of V
  static constexpr int kWords = D >= 64 ? D / 16 : 2;  // of a lane's part of a row of K

  // Dims of step s in lane group g: heads of 64 and 128 take 16 bytes in a row for two steps.
  static __device__ __forceinline__ int dim(int s, int g) { return D >= 64 ? s / 2 * 64 + g * 16 + s % 2 * 8 : 8 * g; }

  static __device__ __forceinline__ void load_k(const uint8_t* row, int g, uint32_t (&w)[kWords]) {
    if constexpr (D >= 64) {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        const u32x4 r = *reinterpret_cast<const u32x4*>(row + 64 * e + 16 * g);
#pragma unroll
        for (int x = 0; x < 4; ++x) w[4 * e + x] = r[x];
      }
    } else {
      const u32x2 r = *reinterpret_cast<const u32x2*>(row + (D == 32 ? 8 * g : 8 * (g & 1)));
      w[0] = D == 16 && g > 1 ? 0u : r[0], w[1] = D == 16 && g > 1 ? 0u : r[1];
    }
  }
};

// One query row's operand of step s, as pieces.
template <typename T, int D>
__device__ __forceinline__ void load_q(const T* row, int s, int g, u32x4 (&q)[pieces_of<T>()]) {
  constexpr int P = pieces_of<T>(), E = vec_elems<T>();
  const bool on = D > 16 || g < 2;
  const T* at = row + Tile<D>::dim(s, D > 16 ? g : g & 1);
  if constexpr (P == 1) {
    const uint4 r = load16(at);
    q[0] = on ? u32x4{r.x, r.y, r.z, r.w} : u32x4{0u, 0u, 0u, 0u};
  } else {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8 / E; ++e) unpack16<T>(load16(at + e * E), &x[e * E]);
#pragma unroll
    for (int p = 0; p < P; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t lo = __float_as_uint(x[2 * e]), hi = __float_as_uint(x[2 * e + 1]);
        q[p][e] = on ? (lo >> 16) | (hi & 0xffff0000u) : 0u;  // cut, so that the pieces' sum is x
        x[2 * e] -= __uint_as_float(lo & 0xffff0000u);
        x[2 * e + 1] -= __uint_as_float(hi & 0xffff0000u);
      }
  }
}

// Where a lane's keys lie.
struct Spot {
  int page;  // 0 where there is none
  bool on;
};
__device__ __forceinline__ Spot spot_of(const PagedArgs& a, int entry, int slot, int cap) {
  const bool on = slot < cap && entry >= 0 && entry < a.pages;
  return Spot{on ? entry : 0, on};
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  }
}

// A workgroup has up to 16 NC query rows (the G heads of a KV head times the tokens, row
// r = t G + g) and a split of the keys; its waves take the split's tiles in turn and are
// joined through LDS at the end.
template <typename T, int D, int NC>
__global__ __launch_bounds__(kPagedWaves * kWave) void paged_attention_kernel(const PagedArgs a) {
  using L = Tile<D>;
  constexpr int P = pieces_of<T>(), W = kPagedWaves, BT = kPagedTile, kRows = 16 * NC, kLine = D + 4;
  __shared__ float merged[W][kRows][kLine];
  __shared__ float tops[W][kRows], sums[W][kRows];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave, g = lane / 16, n = lane % 16;
  // Row blocks of one unit run on one XCD, whose L2 then holds its pages.
  const int slice = int(blockIdx.x) / kXcds;
  const int unit = slice / a.row_blocks * kXcds + int(blockIdx.x) % kXcds;
  if (unit >= a.groups * a.splits) return;
  const int r0 = slice % a.row_blocks * kRows;
  const int group = __builtin_amdgcn_readfirstlane(unit / a.splits), part = unit - group * a.splits;
  const int b = __builtin_amdgcn_readfirstlane(group / a.kv_heads), hk = group - b * a.kv_heads;
  const PagedRow row = paged_row(a, b);
  const int rows = a.tokens << a.group_log2, G = 1 << a.group_log2;
  const int t0 = r0 >> a.group_log2, t1 = min((min(r0 + kRows, rows) - 1) >> a.group_log2, row.count - 1);  // tokens

  // Slots that some row of the block sees, in whole tiles of which this split has some.
  const int end = t1 >= t0 ? row.len + t1 + 1 : 0;
  const int start = a.window >= 0 ? max(row.len + t0 - a.window, 0) : 0;
  const int tile0 = start / BT, tiles = max((end + BT - 1) / BT - tile0, 0);
  const int begin = tile0 + int(long(tiles) * part / a.splits), stop = tile0 + int(long(tiles) * (part + 1) / a.splits);

  u32x4 q[NC][L::kSteps][P];
  int seen_from[NC], seen_to[NC];  // first and last slot of the lane's query row
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = min(r0 + 16 * c + n, rows - 1), t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
    const T* at = static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[1] + t * a.qs[2];
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) load_q<T, D>(at, s, g, q[c][s]);
    seen_to[c] = t < row.count ? row.len + t : -1;
    seen_from[c] = a.window >= 0 ? row.len + t - a.window : 0;
  }
  f32x4 o[NC][L::kDims];
  float top[NC], sum[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    top[c] = -INFINITY, sum[c] = 0.f;
#pragma unroll
    for (int d = 0; d < L::kDims; ++d) o[c][d] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  const int32_t* table = a.tables + long(b) * a.places;
  const int page_mask = (1 << a.page_log2) - 1;
  const int off_k = n / 4 * 16, off_v = g * 16;  // of the lane's keys in a tile
  const auto entry = [&](int slot) { return table[min(slot >> a.page_log2, a.places - 1)]; };
  uint32_t kw[4][L::kWords];
  float ks = 0.f;
  const auto fetch_k = [&](int tile, int e) {
    const int slot = tile * BT + off_k;
    const long block = long(spot_of(a, e, slot, row.cap).page) * a.kv_heads + hk;
    ks = a.k_scale[block];
    const uint8_t* at = a.k + ((block << a.page_log2) + (slot & page_mask) + n % 4) * D;
#pragma unroll
    for (int t = 0; t < 4; ++t) L::load_k(at + 4 * t * D, g, kw[t]);
  };

  int tile = begin + wave, ek = 0, ev = 0;
  if (tile < stop) {
    ek = entry(tile * BT + off_k), ev = entry(tile * BT + off_v);
    fetch_k(tile, ek);
  }
  for (; tile < stop; tile += W) {
    const int slot0 = tile * BT;
    const Spot spot = spot_of(a, ev, slot0 + off_v, row.cap);
    u32x4 vw[L::kDims];
    const long block = long(spot.page) * a.kv_heads + hk;
    const float vs = a.v_scale[block];
    const uint8_t* at = a.v + (((block * D) + n) << a.page_log2) + ((slot0 + off_v) & page_mask);
#pragma unroll
    for (int d = 0; d < L::kDims; ++d) vw[d] = *reinterpret_cast<const u32x4*>(at + (d * 16 << a.page_log2));
    const int next = min(tile + W, stop - 1);
    ek = entry(next * BT + off_k), ev = entry(next * BT + off_v);

    f32x4 s[NC][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int c = 0; c < NC; ++c) s[c][t] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int st = 0; st < L::kSteps; ++st) {
        const u32x4 key = from_codes(kw[t][2 * st], kw[t][2 * st + 1], ks);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int p = P - 1; p >= 0; --p) s[c][t] = mfma16(key, q[c][st][p], s[c][t]);
      }
    }
    fetch_k(next, ek);

    // Tiles that some row does not see whole.
    uint32_t seen[NC];
    const bool masked = slot0 + BT - 1 > row.len + t0 || (a.window >= 0 && slot0 < row.len + t1 - a.window) || __any(!spot.on);
    if (masked) {
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        seen[c] = 0;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int slot = slot0 + off_v + e;
          const bool on = spot.on && slot <= seen_to[c] && slot >= seen_from[c];
          seen[c] |= uint32_t(on) << e;
          s[c][e / 4][e % 4] = on ? s[c][e / 4][e % 4] : -INFINITY;
        }
      }
    }
    u32x4 prob[NC][2][P];
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      float high = s[c][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) high = fmaxf(high, s[c][e / 4][e % 4]);
      high = fmaxf(high, lane_xor(high, 16));
      high = fmaxf(high, lane_xor(high, 32)) * a.cs;
      // The reference moves when it has come to lie far below the maximum.
      const bool raise = high > top[c] + kLazyMax;
      if (__any(raise)) {
        const float now = raise ? high : top[c];
        const float keep = raise ? __builtin_amdgcn_exp2f(top[c] - now) : 1.f;
        top[c] = now;
        sum[c] *= keep;
#pragma unroll
        for (int d = 0; d < L::kDims; ++d) o[c][d] *= keep;
      }
      const float base = top[c] == -INFINITY ? 0.f : top[c];
      float x[16];
#pragma unroll
      for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(s[c][e / 4][e % 4], a.cs, -base));
#pragma unroll
      for (int e = 0; e < 16; ++e) sum[c] += x[e];
#pragma unroll
      for (int p = 0; p < P; ++p)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const uint32_t w = pack2<bf16_t>(x[2 * e], x[2 * e + 1]);
          prob[c][e / 4][p][e % 4] = w;
          x[2 * e] -= bf16_lo(w), x[2 * e + 1] -= bf16_hi(w);
        }
    }
    if (masked) {
      // Values of slots that nobody sees become zeros: old codes there may be NaN. NaN in slots
      // that some rows see makes the sums of those rows NaN, and only those.
      const int from = start - (slot0 + off_v), to = spot.on ? end - (slot0 + off_v) : 0;
      uint32_t bad = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t keep = first_bytes(to - 4 * x) & ~first_bytes(from - 4 * x);
#pragma unroll
        for (int d = 0; d < L::kDims; ++d) {
          vw[d][x] &= keep;
          bad |= nan_bytes(vw[d][x]);
        }
      }
      if (__any(bad != 0)) {
        u32x4 sees[NC][2];
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            sees[c][e / 4][e % 4] = (seen[c] >> (2 * e) & 1 ? 0x3f80u : 0u) | (seen[c] >> (2 * e + 1) & 1 ? 0x3f800000u : 0u);
#pragma unroll
        for (int d = 0; d < L::kDims; ++d) {
          u32x4 is_nan[2];
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const uint32_t m = nan_bytes(vw[d][x]);
            vw[d][x] &= ~m;
            is_nan[x / 2][x % 2 * 2] = (m & 0xff ? 0x3f80u : 0u) | (m & 0xff00 ? 0x3f800000u : 0u);
            is_nan[x / 2][x % 2 * 2 + 1] = (m & 0xff0000 ? 0x3f80u : 0u) | (m & 0xff000000u ? 0x3f800000u : 0u);
          }
#pragma unroll
          for (int c = 0; c < NC; ++c) {
            f32x4 hit = mfma16(is_nan[0], sees[c][0], f32x4{0.f, 0.f, 0.f, 0.f});
            hit = mfma16(is_nan[1], sees[c][1], hit);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[c][d][e] = hit[e] > 0.f ? NAN : o[c][d][e];
          }
        }
      }
    }
#pragma unroll
    for (int d = 0; d < L::kDims; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 value = from_codes(vw[d][2 * h], vw[d][2 * h + 1], vs);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int p = P - 1; p >= 0; --p) o[c][d] = mfma16(value, prob[c][h][p], o[c][d]);
      }
  }

#pragma unroll
  for (int c = 0; c < NC; ++c) {
    sum[c] += lane_xor(sum[c], 16);
    sum[c] += lane_xor(sum[c], 32);
    if (top[c] == -INFINITY && sum[c] != sum[c]) top[c] = 0.f;  // every score in sight is NaN: so is the row, which is not empty
    if (g == 0) tops[wave][16 * c + n] = top[c], sums[wave][16 * c + n] = sum[c];
#pragma unroll
    for (int d = 0; d < L::kDims; ++d)
      *reinterpret_cast<f32x4*>(&merged[wave][16 * c + n][16 * d + 4 * g]) = o[c][d];
  }
  __syncthreads();
  for (int y = threadIdx.x; y < kRows * D / 4; y += W * kWave) {
    const int i = y / (D / 4), d = y % (D / 4) * 4, r = r0 + i;
    if (r >= rows) break;
    float base = -INFINITY, den = 0.f, num[4] = {};
#pragma unroll
    for (int w = 0; w < W; ++w) base = fmaxf(base, tops[w][i]);
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float weight = tops[w][i] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(tops[w][i] - base);
      den = fmaf(weight, sums[w][i], den);
      const f32x4 part_o = *reinterpret_cast<const f32x4*>(&merged[w][i][d]);
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = tops[w][i] == -INFINITY ? num[e] : fmaf(weight, part_o[e], num[e]);
    }
    const int t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
    if (a.splits > 1) {
      const long to = (long(group) * a.splits + part) * rows + r;
      if (d == 0) a.pmax[to] = base, a.psum[to] = den;
      store4<float>(a.pout + to * D + d, num);
    } else {
      const bool empty = base == -INFINITY || t >= row.count;
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = empty ? 0.f : num[e] / den;
      store4<T>(static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2] + d, num);
      if (d == 0) a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (base + __builtin_log2f(den)) * kLn2;
    }
  }
}

// The splits of a row joined: a wave to a row, kRound splits' loads at a time.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedArgs a) {
  constexpr int DPL = (D + kWave - 1) / kWave, kRound = 8;
  const int lane = threadIdx.x % kWave;
  const int rows = a.tokens << a.group_log2, G = 1 << a.group_log2;
  const long at = long(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (at >= long(a.groups) * rows) return;
  const int group = int(at / rows), r = int(at - long(group) * rows);
  const int b = group / a.kv_heads, hk = group - b * a.kv_heads;
  const PagedRow row = paged_row(a, b);
  const int t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
  float top = -INFINITY, den = 0.f, num[DPL] = {};
  for (int s0 = 0; s0 < a.splits; s0 += kRound) {
    const auto part = [&](int s) { return (long(group) * a.splits + min(s0 + s, a.splits - 1)) * rows + r; };
    const bool on = lane < kRound && s0 + lane < a.splits;
    const float mine = on ? a.pmax[part(lane % kRound)] : -INFINITY, sum = a.psum[part(lane % kRound)];
    float x[kRound][DPL];
#pragma unroll
    for (int s = 0; s < kRound; ++s)
#pragma unroll
      for (int i = 0; i < DPL; ++i) x[s][i] = a.pout[part(s) * D + min(lane + i * kWave, D - 1)];
    const float now = fmaxf(top, wave_max(mine));
    const float base = now == -INFINITY ? 0.f : now;
    const float keep = __builtin_amdgcn_exp2f(top - base);
    const float w = mine == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mine - base);
    den = den * keep + wave_sum(mine == -INFINITY ? 0.f : w * sum);
#pragma unroll
    for (int i = 0; i < DPL; ++i) num[i] *= keep;
#pragma unroll
    for (int s = 0; s < kRound; ++s) {
      const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
      const float ms = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(mine), s));
#pragma unroll
      for (int i = 0; i < DPL; ++i) num[i] = ms == -INFINITY ? num[i] : fmaf(ws, x[s][i], num[i]);
    }
    top = now;
  }
  const bool empty = top == -INFINITY || t >= row.count;
  T* o = static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
#pragma unroll
  for (int i = 0; i < DPL; ++i)
    if (lane + i * kWave < D) store_scalar<T>(o + lane + i * kWave, empty ? 0.f : num[i] / den);
  if (lane == 0)
    a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (top + __builtin_log2f(den)) * kLn2;
}

constexpr long kMostGroups = 1L << 24;  // a launch holds fewer than 2^32 threads

template <typename T, int D>
int launch_paged(PagedArgs& a, hipStream_t stream) {
  const char* what = "page_attention";
  const int rows = a.tokens << a.group_log2;
  const int block = rows <= 16 ? 16 : 32;
  a.row_blocks = (rows + block - 1) / block;
  const long units = (long(a.groups) * a.splits + kXcds - 1) / kXcds * kXcds;
  const long merged = long(a.groups) * rows;
  if (units * a.row_blocks >= kMostGroups || merged / 4 >= kMostGroups - 1)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: too many workgroups", what);
  const auto kernel = rows <= 16 ? paged_attention_kernel<T, D, 1> : paged_attention_kernel<T, D, 2>;
  hipLaunchKernelGGL(kernel, dim3(unsigned(units * a.row_blocks)), dim3(kPagedWaves * kWave), 0, stream, a);
  if (int rc = check_launch(what)) return rc;
  if (a.splits == 1) return SFL_OK;
  hipLaunchKernelGGL((paged_merge_kernel<T, D>), dim3(unsigned((merged + 3) / 4)), dim3(256), 0, stream, a);
  return check_launch(what);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace sfl

extern "C" int sfl_page_attention(const void* q, const void* k_codes, const void* v_codes, const float* k_scale,
                                  const float* v_scale, const int32_t* tables, const int32_t* lengths,
                                  const int32_t* counts, float* partial_max, float* partial_sum, float* partial_out,
                                  void* out, float* lse, const long* strides, int batch, int q_heads, int kv_heads,
                                  int tokens, int places, int pages, int page_size, int head_dim, int window_left,
                                  int splits, float scale, int dtype, void* stream) {
  using namespace sfl;
  const char* what = "page_attention";
  if (!q || !k_codes || !v_codes || !k_scale || !v_scale || !tables || !lengths || !out || !lse || !strides)
    return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (int rc = check_paged(what, batch, places, pages, page_size)) return rc;
  if (int rc = check_head_dim(what, head_dim)) return rc;
  if (q_heads <= 0 || kv_heads <= 0 || tokens <= 0)
    return set_error(SFL_ERR_INVALID, "%s: heads and tokens must be positive", what);
  if (tokens > kMaxTokens) return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d new tokens", what, kMaxTokens);
  if (q_heads % kv_heads) return set_error(SFL_ERR_INVALID, "%s: query heads must be divisible by KV heads", what);
  const int ratio = q_heads / kv_heads;
  if (ratio != 1 && ratio != 2 && ratio != 4 && ratio != 8)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported GQA ratio %d", what, ratio);
  if (dtype != SFL_DTYPE_F32 && dtype != SFL_DTYPE_BF16 && dtype != SFL_DTYPE_F16)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: dtype must be F32, BF16 or F16", what);
  if (!(scale > 0.f) || !__builtin_isfinite(scale)) return set_error(SFL_ERR_INVALID, "%s: scale must be finite and positive", what);
  if (splits < 1 || splits > 1024) return set_error(SFL_ERR_INVALID, "%s: splits must be in [1, 1024]", what);
  if (splits > 1 && (!partial_max || !partial_sum || !partial_out))
    return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (long(batch) * kv_heads > (1L << 24)) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many KV heads", what);
  if (!aligned16(q) || !aligned16(out) || !aligned16(k_codes) || !aligned16(v_codes))
    return set_error(SFL_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  const int piece = dtype == SFL_DTYPE_F32 ? 4 : 8;
  for (int i = 0; i < 6; ++i)
    if (strides[i] % piece) return set_error(SFL_ERR_INVALID, "%s: strides must be multiples of 16 bytes", what);
  PagedArgs a{q, static_cast<const uint8_t*>(k_codes), static_cast<const uint8_t*>(v_codes), k_scale, v_scale, tables, lengths,
              counts, partial_max, partial_sum, partial_out, out, lse};
  for (int i = 0; i < 3; ++i) a.qs[i] = strides[i], a.os[i] = strides[3 + i];
  a.kv_heads = kv_heads, a.places = places, a.pages = pages, a.page_log2 = log2_of(page_size), a.tokens = tokens;
  a.group_log2 = ratio == 8 ? 3 : ratio / 2, a.splits = splits, a.groups = batch * kv_heads;
  a.window = std::max(window_left, -1);
  a.cs = scale * kLog2e;
  return paged_types(dtype, head_dim, [&](auto t, auto d) {
    return launch_paged<decltype(t), decltype(d)::value>(a, static_cast<hipStream_t>(stream));
  });
}
