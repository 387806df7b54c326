// Attention of drafted tokens over a KV cache, and the attention weights by slot.
//
// A sequence has len committed keys in slots [0, len) of its cache and its count
// drafted tokens' keys in slots [len, len + count). Draft t sees every committed
// key and the drafts j with mask[t, j]:
//
//   s = scale q . k over the keys in sight,  o = sum exp(s - m) v / l,
//   m near max s,  l = sum exp(s - m),  lse = m + log l     (one pass, m and l running)
//   weights[slot] += sum over counted drafts and the group's heads of exp(s - lse)
//
// The G query heads that share a KV head, times the T drafts, are one block of
// R = T G query rows (row r = t G + g) over the same keys, so a key is read once
// for all of them and the products are matrix products: 16 rows to a tile.
#include <algorithm>
#include <type_traits>

#include "attn_mfma.hpp"
#include "lds_dma.hpp"

namespace sfl {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr int kTreeWaves = 4;
constexpr int kTreeTile = 32;  // keys of a wave's tile: two MFMA tiles of 16
constexpr int kMaxDrafts = 128;
constexpr float kLn2 = 0.6931471805599453f;

// Probabilities are exp2(score - m) with a reference m that moves seldom: to kProbBase below
// the running maximum when that has come to lie more than kProbTop above m. They are rounded
// to the type of V for the products. bf16 has the exponents of fp32 (m is a maximum itself);
// fp16 ends at 2^16 and has its full 11 bits down to 2^-14, so probabilities take the top of
// its range: one of w (relative to the row's largest) is off by at most half a step, 2^-11 of
// it, where w >= 2^-25, and by 2^-36 below. (With m at the maximum the tail behind one heavy
// key was lost from 2^-14 on, while the sum kept it. Rescaled more often, 512 rows over
// 65536 fp16 keys take 97.6 us instead of 95.4.)
template <typename T>
constexpr float kProbTop = std::is_same<T, f16_t>::value ? 15.f : kLazyMax;
template <typename T>
constexpr float kProbBase = std::is_same<T, f16_t>::value ? 11.f : 0.f;

struct TreeArgs {
  const void *q, *k, *v;
  const int32_t *lengths, *counts;
  const uint8_t* mask;
  float *pmax, *psum, *pout;
  void* out;
  float* lse;
  long qs[3], ks[3], vs[3], os[3];  // strides in elements: batch, head, row
  long ms[3];                       // mask: batch, draft, key draft
  int kv_heads, cap, tokens, group_log2, splits, row_blocks, groups;
  float cs;  // scale * log2(e): scores are kept in base 2
};

// What a sequence (the same for a whole wave) has: committed keys, drafts in use, keys in all inside the cache.
struct TreeRow {
  int len, count, total;
};
__device__ __forceinline__ TreeRow tree_row(const int32_t* lengths, const int32_t* counts, int b, int cap, int tokens) {
  TreeRow r;
  typedef const __attribute__((address_space(4))) int32_t* Constant;  // read by scalar loads
  b = __builtin_amdgcn_readfirstlane(b);
  r.len = min(max(Constant(lengths)[b], 0), cap);
  r.count = counts ? min(max(Constant(counts)[b], 0), tokens) : tokens;
  r.total = min(r.len + r.count, cap);
  return r;
}

// Keys of one split: whole rounds of the workgroup's waves, so that a row's keys are
// shared evenly among the splits whatever its length.
__device__ __forceinline__ int split_chunk(int total, int splits) {
  constexpr int kRound = kTreeTile * kTreeWaves;
  return (__builtin_amdgcn_readfirstlane((total + splits - 1) / splits) + kRound - 1) / kRound * kRound;
}

// Without branches (the mask is read for every key, from a clamped place): the loads
// of a tile's keys go out together.
__device__ __forceinline__ bool draft_sees(const TreeArgs& a, int b, const TreeRow& row, int t, int key) {
  const int j = min(max(key - row.len, 0), a.tokens - 1);
  const bool on = a.mask[b * a.ms[0] + t * a.ms[1] + j * a.ms[2]] != 0;
  return (key < row.len) | (on & (key < row.total));
}

// Operand registers of a wave's tile of 32 keys. MFMA tile h (0, 1) holds keys
// 16 h .. 16 h + 15; lane = 16 g + n. Scores S^T = K Q^T come out with lane
// (g, n) holding keys 16 h + 4 g + i (i < 4) of query row n, which is also how
// O^T += V^T P^T takes P (k-slot (g, 4 h + i) of a 16-bit MFMA, k-slot g of the
// fp32 MFMA (h, i)), so probabilities never leave their lane. For V^T, lane
// (g, n) loads dims kVec n .. kVec n + kVec - 1 of its 8 keys: accumulator f
// holds dims kVec m + f for m = 0..15, and the 16-bit pairs are put together
// from two keys' words in registers.
template <typename T, int D>
struct TreeOps {
  static constexpr bool kF32 = std::is_same<T, float>::value;
  static constexpr int kVec = D / 16;                            // dims of V per lane and key
  static constexpr int kSteps = kF32 ? D / 16 : (D + 31) / 32;   // 16-byte pieces of a K or Q row per lane
  static constexpr int kWords = kF32 ? kVec : (kVec + 1) / 2;    // 32-bit words of V per lane and key

  // One row's operand: step s, lane group g takes dims (fp32) 16 s + 4 g .. + 3 or
  // (16-bit) 32 s + 8 g .. + 7; head dim 16 fills half of a 16-bit step.
  static __device__ __forceinline__ void load_row(const T* row, int g, u32x4 (&r)[kSteps]) {
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      if constexpr (kF32) {
        r[s] = *reinterpret_cast<const u32x4*>(row + 16 * s + 4 * g);
      } else if constexpr (D == 16) {
        r[s] = *reinterpret_cast<const u32x4*>(row + 8 * (g & 1));
        if (g > 1) r[s] = u32x4{0u, 0u, 0u, 0u};
      } else {
        r[s] = *reinterpret_cast<const u32x4*>(row + 32 * s + 8 * g);
      }
    }
  }

  static __device__ __forceinline__ f32x4 dot(const u32x4& k, const u32x4& q, f32x4 c) {
    if constexpr (kF32) {
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(k[e]), __uint_as_float(q[e]), c, 0, 0, 0);
      return c;
    } else if constexpr (std::is_same<T, bf16_t>::value) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k), __builtin_bit_cast(bf16x8, q), c, 0, 0, 0);
    } else {
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q), c, 0, 0, 0);
    }
  }

  static __device__ __forceinline__ void load_v(const T* row, int n, uint32_t (&w)[kWords]) {
    const T* p = row + kVec * n;
    if constexpr (!kF32 && kVec == 1) {
      w[0] = p->bits;
    } else if constexpr (kWords == 1) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (kWords == 2) {
      const uint2 r = *reinterpret_cast<const uint2*>(p);
      w[0] = r.x, w[1] = r.y;
    } else {
#pragma unroll
      for (int j = 0; j < kWords / 4; ++j) {
        const u32x4 r = reinterpret_cast<const u32x4*>(p)[j];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[4 * j + e] = r[e];
      }
    }
  }

  static __device__ __forceinline__ float v_value(const uint32_t (&w)[kWords], int f) {
    if constexpr (kF32) return __uint_as_float(w[f]);
    const uint32_t bits = (f & 1) ? w[f / 2] >> 16 : w[f / 2] & 0xffffu;
    if constexpr (std::is_same<T, bf16_t>::value) return __uint_as_float(bits << 16);
    return f16_bits_to_f32(uint16_t(bits));
  }
  static __device__ __forceinline__ void zero_value(uint32_t (&w)[kWords], int f) {
    if constexpr (kF32) w[f] = 0u;
    else w[f / 2] &= (f & 1) ? 0x0000ffffu : 0xffff0000u;
  }

  // acc[f] += V^T P^T for the tile; p[h][i] the lane's probabilities. 16-bit types round
  // them to the type of V, as the products of the matrix cores ask: each is off by at
  // most half a step (bf16 2^-8, fp16 2^-11 of its value; kProbBase), of either sign, which
  // over many keys stays near the rounding of the output itself; l sums them unrounded.
  static __device__ __forceinline__ void add_pv(const uint32_t (&v)[8][kWords], const float (&p)[2][4], f32x4 (&acc)[kVec]) {
    if constexpr (kF32) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int f = 0; f < kVec; ++f)
          acc[f] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v[j][f]), p[j / 4][j % 4], acc[f], 0, 0, 0);
    } else {
      u32x4 pk;
#pragma unroll
      for (int a = 0; a < 4; ++a) pk[a] = pack2<T>(p[a / 2][2 * (a % 2)], p[a / 2][2 * (a % 2) + 1]);
#pragma unroll
      for (int f = 0; f < kVec; ++f) acc[f] = dot(v_operand(v, f), pk, acc[f]);
    }
  }
  static __device__ __forceinline__ u32x4 v_operand(const uint32_t (&v)[8][kWords], int f) {
    u32x4 r;
#pragma unroll
    for (int a = 0; a < 4; ++a)
      r[a] = __builtin_amdgcn_perm(v[2 * a + 1][f / 2], v[2 * a][f / 2], (f & 1) ? 0x07060302u : 0x05040100u);
    return r;
  }
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < INFINITY; }

// A draft that does not see a key takes nothing from it, also where the key's value
// is infinite or NaN, which a product with a probability of 0 would spread over
// every row of an MFMA tile. Tiles with drafts in them therefore lose such values
// before the products, and where there were any, the wave adds them here, key by key
// and row by row, to those that see them: add(p, value row) with p = exp2(s - m), of
// which only the sign matters there. (Apart from the tiles' loop, whose registers
// decide how many waves a SIMD holds.)
template <typename T, int D, typename Add>
__device__ __forceinline__ void add_nonfinite(const T* q, const T* k, const T* v, float m, float cs, bool sees, Add&& add) {
  bool bad = false;
  for (int d = int(threadIdx.x) % kWave; d < D; d += kWave) bad |= !finite(load_scalar<T>(v + d));
  if (!__ballot(bad)) return;
  float s = 0.f;
#pragma unroll 1
  for (int d = 0; d < D; ++d) s = fmaf(load_scalar<T>(q + d), load_scalar<T>(k + d), s);
  if (sees) add(__builtin_amdgcn_exp2f(fmaf(s, cs, -m)), v);
}

// Workgroup -> (KV head of a sequence, split, row block). Workgroups go to the 8
// XCDs in turn; the row blocks that read the same keys take consecutive places
// of one XCD, so that all but the first find them in its L2.
struct TreeBlock {
  int group, split, rb;
};
__device__ __forceinline__ TreeBlock tree_block(const TreeArgs& a) {
  const int work = a.groups * a.splits;
  const int x = int(blockIdx.x) % kXcds, y = int(blockIdx.x) / kXcds;
  // (Quotients of scalars are formed on the vector unit; readfirstlane takes them back.)
  const int q = __builtin_amdgcn_readfirstlane(y / a.row_blocks), unit = q * kXcds + x;
  TreeBlock t;
  t.rb = y - q * a.row_blocks;
  t.group = unit < work ? __builtin_amdgcn_readfirstlane(unit / a.splits) : -1;
  t.split = unit - t.group * a.splits;
  return t;
}

// The 32-row form for 16-bit types and head dims 64 and 128: 32x32x16 MFMAs on
// 32 keys x 32 query rows, S^T = K Q^T and O^T += V^T P^T as in the masked prefill
// attention, keys and values staged in LDS by DMA (K rows swizzled for the operand
// reads, V rows laid out for the transpose reads). WR of the 4 waves share a tile of
// 32 keys, each with 32 query rows of its own, and the 4 / WR groups of waves take
// tiles in turn. A key costs 4 D operations a row: with few rows the launch streams
// the cache (WR = 1: the waves' tiles are their own, no barrier), with 128 rows to a
// workgroup a tile is read from memory once for all of them and the waves bound it:
// for each tile 16 MFMAs (0.25 us), 102 VALU instructions, 16 of them exp (0.28), and
// 24 LDS reads (0.23), of which two waves to a SIMD overlap little. Measured: 512 rows
// over 65536 fp16 keys of 4 heads 90 us (765 TFLOP/s; the 16-row kernel 170), 8 sequences of
// 108 rows over 1K to 8K keys of 8 heads 44 us (3.8 TB/s), 8 rows over 1024 keys 8 us.
template <int D, int WR>
struct TileShape {
  static constexpr int WK = kTreeWaves / WR;      // tiles taken side by side
  static constexpr int TP = WR == 4 ? 2 : 1;      // tiles a wave takes in a round (a barrier's worth)
  static constexpr int NB = 2;                    // rounds of tiles in LDS
  static constexpr int SL = D / 8;                // 16-byte slots of a row
  static constexpr int RPL = kWave / SL;          // rows one DMA load moves
  static constexpr int NLD = kTreeTile / RPL;     // loads of a tile and operand
  static constexpr int L = 2 * NLD / WR;          // a wave's loads of a tile
  static constexpr int kTiles = NB * WK * TP * 2 * kTreeTile * SL * 16, kMerge = WK > 1 ? WK * 32 * WR * (D + 2) * 4 : 0;
  static constexpr int kBytes = kTiles > kMerge ? kTiles : kMerge;
  static constexpr int kGroups = kBytes > 80 * 1024 ? 1 : 2;  // workgroups a CU holds, at least
};

// One tile: scores, running maximum and sum, products with V. kMask: the tile holds
// keys past the committed ones; sees: which of the lane's keys its row sees.
template <typename T, int D, bool kMask>
__device__ __forceinline__ void tile_step(const uint4 (*kt)[D / 8], const uint4 (*vt)[D / 8], const u32x4 (&q)[D / 16],
                                          f32x16 (&acc)[D / 32], float& m, float& l, int c, int h, uint32_t sees,
                                          bool bad, float cs, const unsigned (&vlane)[D / 32]) {
  f32x16 s;
#pragma unroll
  for (int j = 0; j < 16; ++j) s[j] = 0.f;
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) {
    const uint4 r = kt[c][(D / 16 * h + ks) ^ k_swizzle<D>(c)];
    s = mfma32<T>(u32x4{r.x, r.y, r.z, r.w}, q[ks], s);
  }
  if constexpr (kMask) {
#pragma unroll
    for (int j = 0; j < 16; ++j) s[j] = sees >> j & 1u ? s[j] : -INFINITY;
  }
  float mx = fmaxf(s[0], s[1]);
#pragma unroll
  for (int j = 2; j < 16; j += 2) mx = fmaxf(fmaxf(mx, s[j]), s[j + 1]);
  mx = fmaxf(mx, lane_xor(mx, 32));
  const bool grow = mx * cs > m + kProbTop<T>;  // seldom, as below
  if (__ballot(grow)) {
    const float mn = grow ? mx * cs - kProbBase<T> : m;
    const float alpha = grow ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
    m = mn;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < D / 32; ++t) acc[t] *= alpha;
  }
  const unsigned vbase = lds_offset(&vt[0][0]);
  const auto v_operand = [&](int s2, int t) {
    const unsigned off = vbase + vlane[t] + 32u * D * unsigned(s2);
    const i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(size_t)(off));
    const i16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4_t*)(size_t)(off + 16u * D));
    const uint2 a = __builtin_bit_cast(uint2, lo), b = __builtin_bit_cast(uint2, hi);
    return u32x4{a.x, a.y, b.x, b.y};
  };
  const float ms = m == -INFINITY ? 0.f : m;
  float p[16], sum[2] = {0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    p[j] = __builtin_amdgcn_exp2f(fmaf(s[j], cs, -ms));
    sum[j & 1] += p[j];
  }
  l += sum[0] + sum[1];
  // Probabilities in the type of V for the products, half a step each (kProbBase) and of
  // either sign; l sums them unrounded.
  const auto pack8 = [](const float* x) {
    return u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
  };
  u32x4 pk[2] = {pack8(p), pack8(p + 8)};
  // Each 16-bit value of an operand through f(bits) -> bits.
  const auto each = [](u32x4 w, auto&& f) {
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = f(w[e] & 0xffffu) | f(w[e] >> 16) << 16;
    return w;
  };
  constexpr uint32_t kExp = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
  for (int s2 = 0; s2 < 2; ++s2) {
#pragma unroll
    for (int t = 0; t < D / 32; ++t) {
      u32x4 v = v_operand(s2, t);
      if constexpr (kMask) {
        if (bad) v = each(v, [](uint32_t x) { return (x & kExp) == kExp ? 0u : x; });
      }
      acc[t] = mfma32<T>(v, pk[s2], acc[t]);
    }
  }
}

template <typename T, int D, int WR>
__global__ __launch_bounds__(kTreeWaves * kWave, (TileShape<D, WR>::kGroups)) void tree_tile_kernel(const TreeArgs a) {
  using S = TileShape<D, WR>;
  constexpr int WK = S::WK, TP = S::TP, NB = S::NB, SL = S::SL, RPL = S::RPL, BT = kTreeTile, BK = BT * WK * TP;
  __shared__ __align__(16) unsigned char lds[S::kBytes];
  typedef uint4 Tile[BT][SL];
  Tile* tiles = reinterpret_cast<Tile*>(lds);  // [buffer][tile of the round, TP of each wave][K, V]
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave, c = lane % 32, h = lane / 32;
  const int wk = wave / WR, wr = wave % WR;
  const TreeBlock blk = tree_block(a);
  if (blk.group < 0) return;
  const int b = __builtin_amdgcn_readfirstlane(blk.group / a.kv_heads), hk = blk.group - b * a.kv_heads;
  const TreeRow row = tree_row(a.lengths, a.counts, b, a.cap, a.tokens);
  const int G = 1 << a.group_log2, rows = a.tokens << a.group_log2, used = row.count << a.group_log2;
  const int block0 = blk.rb * 32 * WR, row0 = block0 + 32 * wr;
  const int chunk = split_chunk(row.total, a.splits);
  const int begin = blk.split * chunk, end = min(row.total, begin + chunk);
  if (a.splits > 1 && (begin >= end || block0 >= used)) return;  // the merge does not read these

  // The split's keys as buffers whose range ends with its last key: rows past it read as zeros.
  const unsigned krow = unsigned(a.ks[2]) * 2u, vrow = unsigned(a.vs[2]) * 2u;
  const int keys = __builtin_amdgcn_readfirstlane(block0 < used ? max(end - begin, 0) : 0);
  const auto scalar = [](i32x4_t r) {  // 64-bit products are formed on the vector unit, too
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __builtin_amdgcn_readfirstlane(r[e]);
    return r;
  };
  const i32x4_t krsrc = scalar(buffer_rsrc(static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1] + long(begin) * a.ks[2],
                                           keys ? unsigned(keys - 1) * krow + 2u * D : 0u));
  const i32x4_t vrsrc = scalar(buffer_rsrc(static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1] + long(begin) * a.vs[2],
                                           keys ? unsigned(keys - 1) * vrow + 2u * D : 0u));
  // A wave's share of its tile's loads (load j moves rows RPL j .. RPL j + RPL - 1):
  // all of K and V where the tile is its own, else a part of K or a part of V.
  const int lrr = lane / SL, lpp = lane % SL;
  const auto slot = [&](bool values, int j) {  // 16-byte slot that lands in physical slot lpp of row RPL j + lrr
    return values ? 2u * ((unsigned(lpp) >> 1) ^ (unsigned(lrr) & 3u)) + (unsigned(lpp) & 1u)
                  : unsigned(lpp ^ k_swizzle<D>(RPL * j + lrr));
  };
  const auto offset = [&](bool values, unsigned stride, int j) {
    return unsigned(RPL * j + lrr) * stride + 16u * slot(values, j);
  };
  constexpr int kLoads = WR == 1 ? S::NLD : S::L;
  unsigned koff[WR == 1 ? S::NLD : 1], off[kLoads];  // K's where the tile is the wave's own; V's, or those of its part
  const bool values = WR == 1 || wr >= WR / 2;
  const i32x4_t mine = scalar(values ? vrsrc : krsrc);
  const unsigned mrow = values ? vrow : krow;
  const int j0 = WR == 1 ? 0 : (wr % std::max(WR / 2, 1)) * S::L;
#pragma unroll
  for (int i = 0; i < kLoads; ++i) off[i] = offset(values, mrow, j0 + i);
  if constexpr (WR == 1) {
#pragma unroll
    for (int i = 0; i < S::NLD; ++i) koff[i] = offset(false, krow, i);
  }
  const auto issue = [&](int round) {
#pragma unroll
    for (int tp = 0; tp < TP; ++tp) {
      Tile* to = tiles + (((round % NB) * WK + wk) * TP + tp) * 2;
      // A tile past the keys (the round's last ones) starts at the last key: the range check
      // of a load counts from its scalar offset, which has to lie inside.
      const unsigned first = unsigned(min(round * BK + (wk * TP + tp) * BT, keys - 1));
      const unsigned kfirst = first * krow, mfirst = first * mrow;
      const unsigned at = lds_offset(&to[values][RPL * j0][0]);
      if constexpr (WR == 1) {
        const unsigned kat = lds_offset(&to[0][0][0]);
#pragma unroll
        for (int i = 0; i < S::NLD; ++i) lds_load16(krsrc, kat + 1024u * unsigned(i), koff[i], kfirst);
      }
#pragma unroll
      for (int i = 0; i < kLoads; ++i) lds_load16(mine, at + 1024u * unsigned(i), off[i], mfirst);
    }
  };
  unsigned vlane[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t) vlane[t] = vt_lane_offset<D>(lane, t);

  float m = -INFINITY, l = 0.f;
  f32x16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t)
#pragma unroll
    for (int j = 0; j < 16; ++j) acc[t][j] = 0.f;

  const int rounds = (keys + BK - 1) / BK;
  if (rounds > 0) issue(0);

  const int r = min(row0 + c, rows - 1);  // rows past the last repeat it and are not stored
  const int draft = r >> a.group_log2;
  const T* q_row = static_cast<const T*>(a.q) + b * a.qs[0] + long((hk << a.group_log2) + (r & (G - 1))) * a.qs[1] + draft * a.qs[2];
  u32x4 q[D / 16];
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) q[ks] = *reinterpret_cast<const u32x4*>(q_row + D / 2 * h + 8 * ks);
  // Waited for here, with the first tiles: the compiler would wait for them where they
  // are used first, in the loop, and there for every tile in flight.
#pragma unroll
  for (int ks = 0; ks < D / 16; ++ks) asm volatile("" : "+v"(q[ks]));

  const auto arrive = [&](int i) {
    if constexpr (WR == 1) {
      // The tiles are the wave's own: it refills the one it has read and waits for this one.
      wait_lds_reads();
      if (i + 1 < rounds) issue(i + 1);
      wait_younger<1, S::L * TP>(min(1, rounds - 1 - i));
    } else {
      // Every wave's part of this round has landed, and everyone has read the round
      // before, whose place the load after the barrier takes.
      __builtin_amdgcn_s_waitcnt(sfl_vmcnt(0));
      wait_lds_reads();
      __syncthreads();
      if (i + 1 < rounds) issue(i + 1);
    }
    return tiles + ((i % NB) * WK + wk) * TP * 2;
  };
  const bool busy = row0 < used;  // uniform over the wave
  // Rounds of committed keys alone, then those with drafts or the end in them (two
  // loops: with a choice inside one, the accumulators are copied in every round).
  const int full = min(rounds, max(0, min(row.len, end) - begin) / BK);
  for (int i = 0; i < full; ++i) {
    const Tile* tile = arrive(i);
    if (!busy) continue;
#pragma unroll
    for (int tp = 0; tp < TP; ++tp)
      tile_step<T, D, false>(tile[2 * tp], tile[2 * tp + 1], q, acc, m, l, c, h, 0u, false, a.cs, vlane);
  }
  bool lost = false;  // values left out of the products
  for (int i = full; i < rounds; ++i) {
    const Tile* tile = arrive(i);
#pragma unroll 1
    for (int tp = 0; tp < TP; ++tp, tile += 2) {
      const int t0 = begin + i * BK + (wk * TP + tp) * BT;
      if (!busy || t0 >= end) break;
      uint32_t sees = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int key = t0 + 8 * (j / 4) + 4 * h + j % 4;
        sees |= uint32_t((key < end) & draft_sees(a, b, row, draft, key)) << j;
      }
      bool bad = false;
      constexpr uint32_t kExp = std::is_same<T, bf16_t>::value ? 0x7f80u : 0x7c00u;
#pragma unroll
      for (int x = 0; x < BT * SL / kWave; ++x) {
        const uint4 w = (&tile[1][0][0])[x * kWave + lane];
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= (u[e] & kExp) == kExp || (u[e] >> 16 & kExp) == kExp;
      }
      bad = __ballot(bad) != 0;
      lost |= bad;
      tile_step<T, D, true>(tile[0], tile[1], q, acc, m, l, c, h, sees, bad, a.cs, vlane);
    }
  }
  if (lost) {
    const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1];
    const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1];
    for (int t0 = begin + full * BK + wk * BT * TP; t0 < end; t0 += BK)
      for (int key = t0; key < min(t0 + BT * TP, end); ++key)
        add_nonfinite<T, D>(q_row, kp + key * a.ks[2], vp + key * a.vs[2], m, a.cs, draft_sees(a, b, row, draft, key),
                            [&](float p, const T* value) {
#pragma unroll
                              for (int t = 0; t < D / 32; ++t)
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                  const float x = load_scalar<T>(value + 32 * t + 8 * (j / 4) + 4 * h + j % 4);
                                  if (!finite(x)) acc[t][j] += p * x;
                                }
                            });
  }
  l += lane_xor(l, 32);

  const auto store = [&](int at, int d0, const float(&num)[4], float top, float den) {  // four dims of query row at
    if (a.splits > 1) {
      const long part = (long(blk.group) * a.splits + blk.split) * rows + at;
      *reinterpret_cast<float4*>(a.pout + part * D + d0) = make_float4(num[0], num[1], num[2], num[3]);
      if (d0 == 0) {
        a.pmax[part] = top;
        a.psum[part] = den;
      }
      return;
    }
    const int t = at >> a.group_log2, head = (hk << a.group_log2) + (at & (G - 1));
    const bool empty = t >= row.count || den == 0.f;
    const float inv = empty ? 0.f : 1.f / den;
    uint2 w = make_uint2(pack2<T>(num[0] * inv, num[1] * inv), pack2<T>(num[2] * inv, num[3] * inv));
    if (empty) w = make_uint2(0u, 0u);
    *reinterpret_cast<uint2*>(static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2] + d0) = w;
    if (d0 == 0)
      a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (top + __builtin_log2f(den)) * kLn2;
  };
  if constexpr (WK == 1) {
    if (row0 + c < rows) {
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float num[4] = {acc[t][j], acc[t][j + 1], acc[t][j + 2], acc[t][j + 3]};
          store(row0 + c, 32 * t + 2 * j + 4 * h, num, m, l);
        }
    }
  } else {
    // The groups' states through LDS, then four dims of a row by each thread.
    typedef float MergeRow[32 * WR][D + 2];
    MergeRow* sm = reinterpret_cast<MergeRow*>(lds);
    __syncthreads();  // everyone is done with the tiles
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
      for (int j = 0; j < 16; ++j) sm[wk][32 * wr + c][32 * t + 8 * (j / 4) + 4 * h + j % 4] = acc[t][j];
    if (h == 0) {
      sm[wk][32 * wr + c][D] = m;
      sm[wk][32 * wr + c][D + 1] = l;
    }
    __syncthreads();
    for (int x = threadIdx.x; x < 32 * WR * D / 4; x += kTreeWaves * kWave) {
      const int at = x / (D / 4), d0 = 4 * (x % (D / 4));
      if (block0 + at >= rows) break;
      float top = sm[0][at][D];
#pragma unroll
      for (int w = 1; w < WK; ++w) top = fmaxf(top, sm[w][at][D]);
      float den = 0.f, num[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float mw = sm[w][at][D];
        const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - top);
        den = fmaf(f, sm[w][at][D + 1], den);
#pragma unroll
        for (int e = 0; e < 4; ++e) num[e] = fmaf(f, sm[w][at][d0 + e], num[e]);
      }
      store(block0 + at, d0, num, top, den);
    }
  }
}

// The 16-row form, for fp32, short heads and caches past 32-bit offsets: each wave has
// tiles of 32 keys of its own, operands straight from memory (a lane's pieces of a row
// are 16 bytes, so nothing goes through LDS), and RT tiles of 16 rows to use them for.
// Bound by the fp32 MFMAs where there are many rows, else by the way from memory, as
// the next tile's loads wait for this one's products. Measured with the merge: 20 rows
// over 20000 16-bit keys of 32 heads of 32 20 us (4.0 TB/s), 64 fp32 rows over 8192 keys
// of 8 heads of 128 37 us (57 TFLOP/s).
template <typename T, int D, int RT>
__global__ __launch_bounds__(kTreeWaves * kWave) void tree_attention_kernel(const TreeArgs a) {
  using O = TreeOps<T, D>;
  constexpr int W = kTreeWaves, BT = kTreeTile, VEC = O::kVec;
  constexpr int kState = RT * (4 * VEC + 2);  // a lane's registers of a wave's state
  __shared__ float sm[2][kState][kWave];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave, g = lane / 16, n = lane % 16;
  const TreeBlock blk = tree_block(a);
  if (blk.group < 0) return;
  const int b = __builtin_amdgcn_readfirstlane(blk.group / a.kv_heads), hk = blk.group - b * a.kv_heads;
  const TreeRow row = tree_row(a.lengths, a.counts, b, a.cap, a.tokens);
  const int G = 1 << a.group_log2, rows = a.tokens << a.group_log2;
  const int row0 = blk.rb * 16 * RT;
  const int chunk = split_chunk(row.total, a.splits);
  const int begin = blk.split * chunk, end = min(row.total, begin + chunk);
  const bool idle = row0 >= row.count << a.group_log2;  // drafts not in use, whose rows are zeros
  if (a.splits > 1 && (begin >= end || idle)) return;   // the merge does not read these

  const auto q_row = [&](int rt) {  // rows past the last repeat it and are not stored
    const int r = min(row0 + 16 * rt + n, rows - 1);
    return static_cast<const T*>(a.q) + b * a.qs[0] + long((hk << a.group_log2) + (r & (G - 1))) * a.qs[1] +
           (r >> a.group_log2) * a.qs[2];
  };
  u32x4 q[RT][O::kSteps];
  int draft[RT];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    draft[rt] = min(row0 + 16 * rt + n, rows - 1) >> a.group_log2;
    O::load_row(q_row(rt), g, q[rt]);
  }
  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1];
  const T* vp = static_cast<const T*>(a.v) + b * a.vs[0] + hk * a.vs[1];

  float m[RT], l[RT];
  f32x4 acc[RT][VEC];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m[rt] = -INFINITY;
    l[rt] = 0.f;
#pragma unroll
    for (int f = 0; f < VEC; ++f) acc[rt][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  bool lost = false;  // values left out of the products
  if (!idle) {
    for (int t0 = begin + BT * wave; t0 < end; t0 += BT * W) {
      // Keys past the last one of the row are its last one again: nothing outside is read.
      u32x4 k[2][O::kSteps];
      uint32_t v[8][O::kWords];
#pragma unroll
      for (int h = 0; h < 2; ++h) O::load_row(kp + long(min(t0 + 16 * h + n, end - 1)) * a.ks[2], g, k[h]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        O::load_v(vp + long(min(t0 + 16 * (j / 4) + 4 * g + j % 4, end - 1)) * a.vs[2], n, v[j]);
      const bool masked = t0 + BT > min(row.len, end);

      float p[RT][2][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        f32x4 s[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          s[h] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < O::kSteps; ++st) s[h] = O::dot(k[h][st], q[rt][st], s[h]);
        }
        if (masked) {
          uint32_t sees = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int key = t0 + 16 * (j / 4) + 4 * g + j % 4;
            sees |= uint32_t((key < end) & draft_sees(a, b, row, draft[rt], key)) << j;
          }
#pragma unroll
          for (int j = 0; j < 8; ++j) s[j / 4][j % 4] = sees >> j & 1u ? s[j / 4][j % 4] : -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                         fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = fmaxf(mx, lane_xor(mx, 16));
        mx = fmaxf(mx, lane_xor(mx, 32));
        // m moves only when the tile's maximum is more than kProbTop above it, so that
        // probabilities stay below 2^kProbTop and the sums are rescaled seldom.
        const bool grow = mx * a.cs > m[rt] + kProbTop<T>;
        if (__ballot(grow)) {
          const float mn = grow ? mx * a.cs - kProbBase<T> : m[rt];
          const float alpha = grow ? __builtin_amdgcn_exp2f(m[rt] - mn) : 1.f;
          m[rt] = mn;
          l[rt] *= alpha;
#pragma unroll
          for (int f = 0; f < VEC; ++f) acc[rt][f] *= alpha;
        }
        const float ms = m[rt] == -INFINITY ? 0.f : m[rt];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[rt][h][i] = __builtin_amdgcn_exp2f(fmaf(s[h][i], a.cs, -ms));
            l[rt] += p[rt][h][i];
          }
      }
      if (masked) {
        bool bad = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int f = 0; f < VEC; ++f) bad |= !finite(O::v_value(v[j], f));
        if (__ballot(bad)) {
          lost = true;
#pragma unroll
          for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int f = 0; f < VEC; ++f)
              if (!finite(O::v_value(v[j], f))) O::zero_value(v[j], f);
        }
      }
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) O::add_pv(v, p[rt], acc[rt]);
    }
  }
  if (lost) {
    for (int t0 = begin + BT * wave; t0 < end; t0 += BT * W) {
      if (t0 + BT <= min(row.len, end)) continue;
      for (int key = t0; key < min(t0 + BT, end); ++key) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
          add_nonfinite<T, D>(q_row(rt), kp + key * a.ks[2], vp + key * a.vs[2], m[rt], a.cs, draft_sees(a, b, row, draft[rt], key),
                              [&](float p, const T* value) {
#pragma unroll
                                for (int f = 0; f < VEC; ++f)
#pragma unroll
                                  for (int i = 0; i < 4; ++i) {
                                    const float x = load_scalar<T>(value + VEC * (4 * g + i) + f);
                                    if (!finite(x)) acc[rt][f][i] += p * x;
                                  }
                              });
      }
    }
  }
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    l[rt] += lane_xor(l[rt], 16);
    l[rt] += lane_xor(l[rt], 32);
  }

  // Merge the waves' states in two rounds: the upper half of the waves hand theirs over.
#pragma unroll
  for (int half = W / 2; half >= 1; half /= 2) {
    if (wave >= half && wave < 2 * half) {
      float(*to)[kWave] = sm[wave - half];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        to[rt][lane] = m[rt];
        to[RT + rt][lane] = l[rt];
#pragma unroll
        for (int f = 0; f < VEC; ++f)
#pragma unroll
          for (int i = 0; i < 4; ++i) to[2 * RT + (rt * VEC + f) * 4 + i][lane] = acc[rt][f][i];
      }
    }
    __syncthreads();
    if (wave < half) {
      float(*from)[kWave] = sm[wave];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float mo = from[rt][lane], top = fmaxf(m[rt], mo);
        const float ca = m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[rt] - top);
        const float cb = mo == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mo - top);
        m[rt] = top;
        l[rt] = ca * l[rt] + cb * from[RT + rt][lane];
#pragma unroll
        for (int f = 0; f < VEC; ++f)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[rt][f][i] = ca * acc[rt][f][i] + cb * from[2 * RT + (rt * VEC + f) * 4 + i][lane];
      }
    }
    __syncthreads();
  }
  if (wave) return;

#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = row0 + 16 * rt + n;
    if (r >= rows) continue;
    if (a.splits > 1) {
      const long part = (long(blk.group) * a.splits + blk.split) * rows + r;
      if (g == 0) {
        a.pmax[part] = m[rt];
        a.psum[part] = l[rt];
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int f = 0; f < VEC; ++f) a.pout[part * D + VEC * (4 * g + i) + f] = acc[rt][f][i];
      continue;
    }
    const int t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
    const bool empty = t >= row.count || l[rt] == 0.f;
    const float inv = empty ? 0.f : 1.f / l[rt];
    T* o = static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int f = 0; f < VEC; ++f) store_scalar<T>(o + VEC * (4 * g + i) + f, empty ? 0.f : acc[rt][f][i] * inv);
    if (g == 0)
      a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (m[rt] + __builtin_log2f(l[rt])) * kLn2;
  }
}

// One wave per query row: the splits' states in one, then the output and lse. Bound by
// reading the partials (2048 rows of 32 splits, 34 MB, 8.6 us), below that by latency.
template <typename T, int D, int kRound>
__global__ __launch_bounds__(256) void tree_merge_kernel(const TreeArgs a) {
  constexpr int DPL = (D + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave;
  const int rows = a.tokens << a.group_log2, G = 1 << a.group_log2;
  const long at = long(blockIdx.x) * 4 + threadIdx.x / kWave;
  if (at >= long(a.groups) * rows) return;
  const int group = int(at / rows), r = int(at - long(group) * rows);
  const int b = group / a.kv_heads, hk = group - b * a.kv_heads;
  const TreeRow row = tree_row(a.lengths, a.counts, b, a.cap, a.tokens);
  const int t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
  float top = -INFINITY, den = 0.f, num[DPL] = {};
  if (t < row.count && row.total > 0) {
    const int chunk = split_chunk(row.total, a.splits);
    const int n = (row.total + chunk - 1) / chunk;
    // kRound splits at a time, all their loads before the first use (one after another
    // they took 7 us for 16 splits of 32 rows, together 3). Lane s holds the maximum and
    // the sum of split s.
    for (int s0 = 0; s0 < n; s0 += kRound) {
      const auto part = [&](int s) { return (long(group) * a.splits + min(s0 + s, n - 1)) * rows + r; };
      const float mine = a.pmax[part(lane % kRound)], sum = a.psum[part(lane % kRound)];
      float x[kRound][DPL];
#pragma unroll
      for (int s = 0; s < kRound; ++s)
#pragma unroll
        for (int i = 0; i < DPL; ++i) x[s][i] = a.pout[part(s) * D + min(lane + i * kWave, D - 1)];
      const bool on = lane < kRound && s0 + lane < n;
      const float mn = fmaxf(top, wave_max(on ? mine : -INFINITY));
      const float base = mn == -INFINITY ? 0.f : mn;
      const float keep = __builtin_amdgcn_exp2f(top - base);
      const float w = on ? __builtin_amdgcn_exp2f(mine - base) : 0.f;
      den = den * keep + wave_sum(on ? w * sum : 0.f);
#pragma unroll
      for (int i = 0; i < DPL; ++i) num[i] *= keep;
#pragma unroll
      for (int s = 0; s < kRound; ++s) {
        const float ws = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(w), s));
#pragma unroll
        for (int i = 0; i < DPL; ++i) num[i] = fmaf(ws, s0 + s < n ? x[s][i] : 0.f, num[i]);
      }
      top = mn;
    }
  }
  const bool empty = den == 0.f;
  T* o = static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
#pragma unroll
  for (int i = 0; i < DPL; ++i)
    if (lane + i * kWave < D) store_scalar<T>(o + lane + i * kWave, empty ? 0.f : num[i] / den);
  if (lane == 0)
    a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (top + __builtin_log2f(den)) * kLn2;
}

// weights[b, hk, slot] += sum over the counted drafts and the group's heads of
// exp(s - lse), scores as in the kernels above. A workgroup has a share of a head's
// keys, its waves tiles of 32 in turn; up to NT tiles of 16 counted rows stay in
// registers while K streams by, the next tile's keys and weights loaded ahead (more
// rows: another pass over the share, whose keys then come from L2). Bound by reading
// K: 16 rows of up to 8K keys of 16 heads of 64, 169 MB, 40 us (4.2 TB/s; without the
// loads ahead and with a workgroup for every 128 keys 60); one row of 4 short sequences
// (kernel 6.9 us for 2.3 of bytes) by the chain of length, rows, scores and store; many
// rows by the passes: 512 rows over 32768 keys of 4 heads of 128 122 us in bf16 (141
// TFLOP/s), 393 in fp32 (44). Every slot has one writer, and its terms one order.
template <typename T, int D, int NT>
__global__ __launch_bounds__(kTreeWaves * kWave) void tree_weights_kernel(const TreeArgs a, const uint8_t* __restrict__ counted,
                                                                          float* __restrict__ weights) {
  using O = TreeOps<T, D>;
  constexpr int BT = kTreeTile, W = kTreeWaves;
  __shared__ short list[kMaxDrafts];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave, g = lane / 16, n = lane % 16;
  const int group = __builtin_amdgcn_readfirstlane(int(blockIdx.x) / a.splits), part = int(blockIdx.x) - group * a.splits;
  const int b = __builtin_amdgcn_readfirstlane(group / a.kv_heads), hk = group - b * a.kv_heads;
  const TreeRow row = tree_row(a.lengths, a.counts, b, a.cap, a.tokens);
  const int G = 1 << a.group_log2;
  const int chunk = split_chunk(row.total, a.splits), begin = part * chunk, end = min(row.total, begin + chunk);
  if (begin >= end) return;

  const T* kp = static_cast<const T*>(a.k) + b * a.ks[0] + hk * a.ks[1];
  float* to = weights + (long(b) * a.kv_heads + hk) * a.cap;
  // The lane whose sum a slot's terms end up in: of the 16 rows' lanes, n = 2 j for key j of the 8.
  const int mine = 16 * (n >> 3) + 4 * g + (n >> 1 & 3);
  u32x4 k[2][O::kSteps];
  float old = 0.f;
  const auto fetch = [&](int t0) {
#pragma unroll
    for (int h = 0; h < 2; ++h) O::load_row(kp + long(min(t0 + 16 * h + n, end - 1)) * a.ks[2], g, k[h]);
    old = to[min(t0 + mine, end - 1)];
  };
  const int first = begin + BT * wave;
  if (first < end) fetch(first);

  // The counted drafts, in order.
  int drafts = 0;
#pragma unroll
  for (int w = 0; w < kMaxDrafts / kWave; ++w) {
    const int t = kWave * w + lane;
    const bool on = t < row.count && (!counted || counted[long(b) * a.tokens + t]);
    const uint64_t bits = __ballot(on);
    if (on && wave == 0) list[drafts + __builtin_popcountll(bits & ((1ull << lane) - 1))] = short(t);
    drafts += __builtin_popcountll(bits);
  }
  __syncthreads();
  const int rows = drafts << a.group_log2;

  for (int r0 = 0; r0 < rows; r0 += 16 * NT) {
    u32x4 q[NT][O::kSteps];
    float base[NT];
    int draft[NT];
#pragma unroll
    for (int rt = 0; rt < NT; ++rt) {
      const int at = r0 + 16 * rt + n, r = min(at, rows - 1);
      draft[rt] = list[r >> a.group_log2];
      const int head = (hk << a.group_log2) + (r & (G - 1));
      O::load_row(static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[1] + draft[rt] * a.qs[2], g, q[rt]);
      const float lse = a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + draft[rt]];
      // Rows past the last and rows that see nothing add exp2(-inf) = 0.
      base[rt] = at < rows && lse != -INFINITY ? lse * kLog2e : INFINITY;
    }
    if (r0 > 0 && first < end) fetch(first);
    for (int t0 = first; t0 < end; t0 += BT * W) {
      u32x4 now[2][O::kSteps];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int st = 0; st < O::kSteps; ++st) now[h][st] = k[h][st];
      const float held = old;
      if (t0 + BT * W < end) fetch(t0 + BT * W);
      const bool masked = t0 + BT > row.len;
      float sum[8] = {};
#pragma unroll
      for (int rt = 0; rt < NT; ++rt) {
        if (r0 + 16 * rt >= rows) break;
        uint32_t sees = ~0u;
        if (masked) {
          sees = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            sees |= uint32_t(draft_sees(a, b, row, draft[rt], t0 + 16 * (j / 4) + 4 * g + j % 4)) << j;
        }
        sees = base[rt] == INFINITY ? 0u : sees;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int st = 0; st < O::kSteps; ++st) s = O::dot(now[h][st], q[rt][st], s);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(fmaf(s[i], a.cs, -base[rt]));
            sum[4 * h + i] += sees >> (4 * h + i) & 1u ? p : 0.f;
          }
        }
      }
      // Over the 16 rows' lanes, each step handing half of the keys to the lane's partner.
#pragma unroll
      for (int m = 8, left = 4; m >= 2; m >>= 1, left >>= 1)
#pragma unroll
        for (int j = 0; j < left; ++j) {
          const float give = n & m ? sum[j] : sum[j + left], keep = n & m ? sum[j + left] : sum[j];
          sum[j] = keep + lane_xor(give, m);
        }
      const float total = sum[0] + lane_xor(sum[0], 1);
      if (!(n & 1) && t0 + mine < end) to[t0 + mine] = held + total;
    }
  }
}

constexpr long kMostGroups = 1L << 24;  // a launch holds fewer than 2^32 threads

// The launch of `kernel` on row blocks of `block` rows, and the merge of its splits.
template <typename T, int D>
int launch_blocks(void (*kernel)(TreeArgs), int block, TreeArgs& a, hipStream_t stream) {
  const int rows = a.tokens << a.group_log2;
  a.row_blocks = (rows + block - 1) / block;
  const long units = (long(a.groups) * a.splits + kXcds - 1) / kXcds * kXcds;
  const long merged = long(a.groups) * rows;
  if (units * a.row_blocks >= kMostGroups || merged / 4 >= kMostGroups - 1)
    return set_error(SFL_ERR_UNSUPPORTED, "tree_attention: too many workgroups");
  hipLaunchKernelGGL(kernel, dim3(unsigned(units * a.row_blocks)), dim3(kTreeWaves * kWave), 0, stream, a);
  if (int rc = check_launch("tree_attention")) return rc;
  if (a.splits == 1) return SFL_OK;
  const auto merge = a.splits <= 4 ? tree_merge_kernel<T, D, 4> : a.splits <= 8 ? tree_merge_kernel<T, D, 8> : tree_merge_kernel<T, D, 16>;
  hipLaunchKernelGGL(merge, dim3(unsigned((merged + 3) / 4)), dim3(256), 0, stream, a);
  return check_launch("tree_attention");
}

template <typename T, int D>
int launch_tree(TreeArgs& a, hipStream_t stream) {
  const int rows = a.tokens << a.group_log2;
  constexpr bool kF32 = std::is_same<T, float>::value;
  if constexpr (!kF32 && D >= 64) {
    // Buffer offsets are 32 bits; caches of 2 GiB a head and more take the kernel below (a call
    // over 8192 keys of one such head: 8 rows 13.5 us, 128 rows 14.8).
    // By rows, us with 1 / 2 / 4 waves to a tile, 64 heads of 4096 bf16 keys: D 128 32 rows
    // 31.5 / 28.9 / 31.8, 64 rows 38.7 / 31.6 / 34.5, 128 rows 96 / 48 / 44; D 64 8 rows
    // 18.2 / 18.1 / 22.7, 64 rows 21.1 / 20.2 / 25.8, 128 rows 43.2 / 29.3 / 29.4.
    if (long(a.cap) * std::max(a.ks[2], a.vs[2]) * 2 < (1L << 31)) {
      if (rows <= 32) return launch_blocks<T, D>(tree_tile_kernel<T, D, 1>, 32, a, stream);
      if (rows <= 64) return launch_blocks<T, D>(tree_tile_kernel<T, D, 2>, 64, a, stream);
      return launch_blocks<T, D>(tree_tile_kernel<T, D, 4>, 128, a, stream);
    }
    return launch_blocks<T, D>(tree_attention_kernel<T, D, 1>, 16, a, stream);
  } else {
    // us with blocks of 16 / 32 / 64 rows, 64 heads of 4096 keys: bf16 D 32 16 rows 12.6 / 13.2 /
    // 17.7, 32 rows 13.7 / 13.7 / 18.2, 64 rows 20.1 / 17.9 / 19.7, 128 rows 30.4 / 26.0 / 27.1;
    // fp32 D 64 16 rows 26 / 33, 32 rows 37 / 33, 128 rows 102 / 90.
    if (rows <= 16) return launch_blocks<T, D>(tree_attention_kernel<T, D, 1>, 16, a, stream);
    if constexpr (kF32) {
      // Heads of 128 with 32 rows leave a SIMD one wave: 11 sequences of 88 rows over up to
      // 8K keys 290 us, with 16 rows 168; where a few workgroups do not decide the time, 16 rows
      // lose to 32 (64 heads of 4096 keys: 32 rows 67 / 59 us, 128 rows 204 / 169).
      constexpr int RT = D == 128 ? 1 : 2;
      return launch_blocks<T, D>(tree_attention_kernel<T, D, RT>, 16 * RT, a, stream);
    } else {
      if (rows <= 32) return launch_blocks<T, D>(tree_attention_kernel<T, D, 2>, 32, a, stream);
      return launch_blocks<T, D>(tree_attention_kernel<T, D, 4>, 64, a, stream);
    }
  }
}

template <typename T, int D>
int launch_weights(TreeArgs& a, const uint8_t* counted, float* weights, hipStream_t stream) {
  // About four workgroups to a CU, whose waves keep a tile or two of loads in flight each.
  const int rounds = (a.cap + kTreeTile * kTreeWaves - 1) / (kTreeTile * kTreeWaves);
  a.splits = std::max(1, std::min(rounds, (1024 + a.groups - 1) / a.groups));
  if (long(a.groups) * a.splits >= kMostGroups) return set_error(SFL_ERR_UNSUPPORTED, "tree_weights: too many workgroups");
  // Rows held in registers, in tiles of 16: us with 1 / 2 / 4 tiles, 64 heads of 4096 keys of 128,
  // bf16 16 rows 17.2 / 16.9 / 17.9, 32 rows 29.6 / 19.2 / 20.4, 64 rows 50 / 33 / 26; fp32 16 rows
  // 30 / 39, 64 rows 96 / 93.
  const int rows = a.tokens << a.group_log2;
  constexpr int kMost = std::is_same<T, float>::value ? 2 : 4;
  const auto kernel = rows <= 16 ? tree_weights_kernel<T, D, 1> : rows <= 32 ? tree_weights_kernel<T, D, 2> : tree_weights_kernel<T, D, kMost>;
  hipLaunchKernelGGL(kernel, dim3(unsigned(a.groups * a.splits)), dim3(kTreeWaves * kWave), 0, stream, a, counted, weights);
  return check_launch("tree_weights");
}

template <typename T, typename F>
int tree_dims(int dim, F&& f) {
  switch (dim) {
    case 16: return f(T{}, std::integral_constant<int, 16>{});
    case 32: return f(T{}, std::integral_constant<int, 32>{});
    case 64: return f(T{}, std::integral_constant<int, 64>{});
    default: return f(T{}, std::integral_constant<int, 128>{});
  }
}
template <typename F>
int tree_types(int dtype, int dim, F&& f) {
  switch (dtype) {
    case SFL_DTYPE_F32: return tree_dims<float>(dim, f);
    case SFL_DTYPE_BF16: return tree_dims<bf16_t>(dim, f);
    default: return tree_dims<f16_t>(dim, f);
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// What both entry points check, and the arguments they share.
int fill(TreeArgs& a, const char* what, const void* q, const void* k, const int32_t* lengths, const uint8_t* mask,
         const int32_t* counts, float* lse, const long* strides, int batch, int q_heads, int kv_heads, int capacity,
         int tokens, int head_dim, float scale, int dtype) {
  if (!q || !k || !lengths || !mask || !lse || !strides) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (batch <= 0 || q_heads <= 0 || kv_heads <= 0 || capacity <= 0 || tokens <= 0)
    return set_error(SFL_ERR_INVALID, "%s: batch, heads, capacity and tokens must be positive", what);
  if (capacity > SFL_CACHE_MAX_SLOTS)  // slots are counted in 32 bits, up to a workgroup's round past the last
    return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d slots", what, SFL_CACHE_MAX_SLOTS);
  if (tokens > kMaxDrafts) return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d drafted tokens", what, kMaxDrafts);
  if (q_heads % kv_heads) return set_error(SFL_ERR_INVALID, "%s: query heads must be divisible by KV heads", what);
  const int group = q_heads / kv_heads;
  if (group != 1 && group != 2 && group != 4 && group != 8)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported GQA ratio %d", what, group);
  if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported head dim %d", what, head_dim);
  if (dtype != SFL_DTYPE_F32 && dtype != SFL_DTYPE_BF16 && dtype != SFL_DTYPE_F16)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: dtype must be F32, BF16 or F16", what);
  if (!(scale > 0.f) || !__builtin_isfinite(scale)) return set_error(SFL_ERR_INVALID, "%s: scale must be finite and positive", what);
  if (long(batch) * kv_heads > (1L << 24)) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many KV heads", what);
  const int piece = dtype == SFL_DTYPE_F32 ? 4 : 8;
  if (!aligned16(q) || !aligned16(k)) return set_error(SFL_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  for (int i = 0; i < 12; ++i)
    if (strides[i] % piece) return set_error(SFL_ERR_INVALID, "%s: strides must be multiples of 16 bytes", what);
  a.q = q, a.k = k, a.lengths = lengths, a.mask = mask, a.counts = counts, a.lse = lse;
  for (int i = 0; i < 3; ++i)
    a.qs[i] = strides[i], a.ks[i] = strides[3 + i], a.vs[i] = strides[6 + i], a.os[i] = strides[9 + i], a.ms[i] = strides[12 + i];
  a.kv_heads = kv_heads, a.cap = capacity, a.tokens = tokens, a.groups = batch * kv_heads;
  a.group_log2 = group == 8 ? 3 : group / 2;
  a.cs = scale * kLog2e;
  return SFL_OK;
}

}  // namespace
}  // namespace sfl

extern "C" int sfl_tree_attention(const void* q, const void* k, const void* v, const int32_t* lengths,
                                  const uint8_t* mask, const int32_t* counts, float* partial_max, float* partial_sum,
                                  float* partial_out, void* out, float* lse, const long* strides, int batch,
                                  int q_heads, int kv_heads, int capacity, int tokens, int head_dim, int splits,
                                  float scale, int dtype, void* stream) {
  using namespace sfl;
  const char* what = "tree_attention";
  TreeArgs a{};
  if (int rc = fill(a, what, q, k, lengths, mask, counts, lse, strides, batch, q_heads, kv_heads, capacity, tokens,
                    head_dim, scale, dtype))
    return rc;
  if (!v || !out) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (splits < 1 || splits > 1024) return set_error(SFL_ERR_INVALID, "%s: splits must be in [1, 1024]", what);
  if (splits > 1 && (!partial_max || !partial_sum || !partial_out))
    return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (!aligned16(v) || !aligned16(out)) return set_error(SFL_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  a.v = v, a.out = out, a.pmax = partial_max, a.psum = partial_sum, a.pout = partial_out, a.splits = splits;
  return tree_types(dtype, head_dim, [&](auto t, auto d) {
    return launch_tree<decltype(t), decltype(d)::value>(a, static_cast<hipStream_t>(stream));
  });
}

extern "C" int sfl_tree_weights(const void* q, const void* k, const float* lse, float* weights, const int32_t* lengths,
                                const uint8_t* mask, const int32_t* counts, const uint8_t* rows, const long* strides,
                                int batch, int q_heads, int kv_heads, int capacity, int tokens, int head_dim,
                                float scale, int dtype, void* stream) {
  using namespace sfl;
  TreeArgs a{};
  if (int rc = fill(a, "tree_weights", q, k, lengths, mask, counts, const_cast<float*>(lse), strides, batch, q_heads,
                    kv_heads, capacity, tokens, head_dim, scale, dtype))
    return rc;
  if (!weights) return set_error(SFL_ERR_INVALID, "tree_weights: null pointer argument");
  return tree_types(dtype, head_dim, [&](auto t, auto d) {
    return launch_weights<decltype(t), decltype(d)::value>(a, rows, weights, static_cast<hipStream_t>(stream));
  });
}
