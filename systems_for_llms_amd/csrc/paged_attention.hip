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
// bf16 pieces: q of fp16 as two, of fp32 as three, and the probabilities of 16-bit rows as two,
// of fp32 as three, so the only roundings are those of the probabilities to the sum of their
// pieces (2^-16 or 2^-24 of them) and of fp32 sums.
#include <algorithm>
#include <type_traits>

#include "attn_mfma.hpp"
#include "paged.hpp"

namespace sfl {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

constexpr int kPagedTile = 64;  // keys of a wave's tile
constexpr int kMaxTokens = 128;
constexpr int kRowWaves = 4;    // of the kernels for blocks of 32 and more rows
constexpr int kAtOnce = 256;    // workgroups that a call in need of more parts aims at
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
  int kv_heads, places, pages, page_log2, tokens, group_log2, row_blocks, groups;
  int splits, most;  // parts of a head's tiles: of sequences of the usual length, of long ones
  int more;          // workgroups (to a row block) for the latter's, where they may have more
  int batch;
  int window;   // slots before its own that a token sees; < 0: all
  float share;  // of the tiles of all sequences that a part is meant to have
  float cs;     // scale * log2(e): scores are kept in base 2
};

template <typename T> constexpr int pieces_of() { return std::is_same<T, bf16_t>::value ? 1 : std::is_same<T, f16_t>::value ? 2 : 3; }
// Of probabilities. With one piece for bf16 rows, off by 2^-8, results are 2.2e-3 from 64 bits, with
// two 1.7e-3, which is their own rounding. us with one and with two: 32 rows of up to 8191 tokens
// 54.9 / 55.6, one of 1024 12.0 / 12.0; where the matrix cores are busy, 64 query rows over 8 x
// 8000 keys 39.4 / 45.9, 108 over 8 of 1K to 8K 44.5 / 53.0, 512 over 32000 86.8 / 109.9.
template <typename T> constexpr int prob_pieces_of() { return std::is_same<T, float>::value ? 3 : 2; }

// What a sequence has: committed tokens, new ones in use, slots.
struct PagedRow {
  int len, count, cap;
};
template <typename P>
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& a, P lengths, P counts, int b) {
  PagedRow r;
  r.cap = a.places << a.page_log2;
  r.len = min(max(lengths[b], 0), r.cap);
  r.count = counts ? min(max(counts[b], 0), a.tokens) : a.tokens;
  r.count = min(r.count, r.cap - r.len);  // tokens that have a slot
  return r;
}
__device__ __forceinline__ PagedRow paged_row(const PagedArgs& a, int b) {
  typedef const __attribute__((address_space(4))) int32_t* Constant;  // read by scalar loads
  return paged_row(a, Constant(a.lengths), Constant(a.counts), __builtin_amdgcn_readfirstlane(b));
}

// Tiles that the tokens of a sequence see.
__device__ __forceinline__ int tiles_seen(const PagedArgs& a, const PagedRow& r) {
  if (r.count <= 0) return 0;
  return (r.len + r.count + kPagedTile - 1) / kPagedTile - (a.window >= 0 ? max(r.len - a.window, 0) / kPagedTile : 0);
}

// Into how many parts a head's tiles of a sequence go: `splits`, or, where the call has room
// for more, as many as it takes that none is more than the batch's tiles over kAtOnce. With
// `splits` by the number of heads only sequences far longer than the others get more: us
// without and with, 8 heads, 32 rows of 500 tokens but one of 131000 371 / 58 (78 where it is
// the last), 64 of 2000 743 / 94, 8 of 500 but one of 32000 with 108 query rows 92 / 55; for
// rows of one length the sum costs 1 to 4 of 170 to 320. More parts for every row by its
// share: rows of 1K to 8K 51.5 / 52.5, 108 query rows 44 / 52. Whole waves call it; it is one
// sum in one order, so all of them come to the same.
__device__ __forceinline__ int fair_part(const PagedArgs& a) {
  float total = 0.f;
  for (int b = threadIdx.x % kWave; b < a.batch; b += kWave) total += float(tiles_seen(a, paged_row(a, a.lengths, a.counts, b)));
  return int(fminf(wave_sum(total) * a.share, 0x1p24f)) + 1;
}
__device__ __forceinline__ int parts_of(const PagedArgs& a, const PagedRow& row, int fair) {
  const int tiles = tiles_seen(a, row);
  return (tiles + a.splits - 1) / a.splits > fair ? min((tiles + fair - 1) / fair, a.most) : a.splits;
}
__device__ __forceinline__ int parts_of(const PagedArgs& a, const PagedRow& row) {
  return __builtin_expect(a.most == a.splits, 1) ? a.splits : __builtin_amdgcn_readfirstlane(parts_of(a, row, fair_part(a)));
}

// The sequence that the x-th of the parts beyond `splits` belongs to, a head's parts behind each
// other, and the part's number there. No parts: there are not so many.
struct More {
  int b, parts, x;
};
__device__ __forceinline__ More find_more(const PagedArgs& a, int x) {
  const int fair = fair_part(a), lane = threadIdx.x % kWave;
  int of = 0, parts = 0, at_x = 0;
  for (int b0 = 0; b0 < a.batch && parts == 0; b0 += kWave) {
    const int mine = b0 + lane < a.batch ? parts_of(a, paged_row(a, a.lengths, a.counts, b0 + lane), fair) : a.splits;
    const int own = (mine - a.splits) * a.kv_heads;
    int sum = own;  // becomes that of the lanes up to this one
#pragma unroll
    for (int m = 1; m < kWave; m <<= 1) {
      const int other = __shfl_up(sum, m);
      sum += lane >= m ? other : 0;
    }
    const uint64_t past = __ballot(sum > x);
    const int at = past ? __builtin_ctzll(past) : kWave - 1;
    of = b0 + at, parts = past ? __builtin_amdgcn_readlane(mine, at) : 0, at_x = x - __builtin_amdgcn_readlane(sum - own, at);
    x -= __builtin_amdgcn_readlane(sum, kWave - 1);
  }
  return {of, parts, at_x};
}

// How many such parts the sequences before b have.
__device__ __forceinline__ int more_before(const PagedArgs& a, int b) {
  const int fair = fair_part(a);
  float sum = 0.f;
  for (int x = threadIdx.x % kWave; x < b; x += kWave)
    sum += float(parts_of(a, paged_row(a, a.lengths, a.counts, x), fair) - a.splits);
  return __builtin_amdgcn_readfirstlane(int(wave_sum(sum)) * a.kv_heads);
}

// A workgroup's work: some rows of a KV head of sequence b over a part of its tiles.
struct Work {
  int b, hk, group;        // group: the head among those of all sequences
  int part, parts, slot;   // slot: of the partial results of its head's rows
  int r0, rows;            // first row of the block; rows of a sequence
  int t0, t1;              // tokens of the block
  int start, end;          // slots that some row of the block sees
  int begin, count;        // its tiles
  PagedRow row;
};
__device__ __forceinline__ bool find_work(const PagedArgs& a, int block, Work& w) {
  // Row blocks of one unit run on one XCD, whose L2 then holds its pages.
  const int slice = int(blockIdx.x) / kXcds;
  const int unit = slice / a.row_blocks * kXcds + int(blockIdx.x) % kXcds;
  w.r0 = slice % a.row_blocks * block;
  const int usual = unit - a.more;  // the parts that only long sequences have come first
  if (usual >= a.groups * a.splits) return false;
  int group = usual / a.splits, more_parts = 0;
  w.part = usual - group * a.splits;
  if (__builtin_expect(usual < 0, 0)) {
    const More more = find_more(a, unit);
    if (more.parts == 0) return false;
    const int extra = more.parts - a.splits;
    group = more.b * a.kv_heads + more.x / extra, w.part = a.splits + more.x % extra, more_parts = more.parts;
  }
  w.group = __builtin_amdgcn_readfirstlane(group), w.part = __builtin_amdgcn_readfirstlane(w.part);
  w.b = __builtin_amdgcn_readfirstlane(w.group / a.kv_heads);
  w.hk = w.group - w.b * a.kv_heads;
  w.row = paged_row(a, w.b);
  w.parts = __builtin_amdgcn_readfirstlane(more_parts ? more_parts : parts_of(a, w.row));
  w.slot = usual < 0 ? a.groups * a.splits + unit : usual;
  w.rows = a.tokens << a.group_log2;
  w.t0 = w.r0 >> a.group_log2, w.t1 = min((min(w.r0 + block, w.rows) - 1) >> a.group_log2, w.row.count - 1);
  w.end = w.t1 >= w.t0 ? w.row.len + w.t1 + 1 : 0;
  w.start = a.window >= 0 ? max(w.row.len + w.t0 - a.window, 0) : 0;
  // The tiles from that of `start` on are shared out evenly.
  const int first = w.start / kPagedTile, tiles = max((w.end + kPagedTile - 1) / kPagedTile - first, 0);
  const int each = tiles / w.parts, more = tiles - each * w.parts;  // one more in the first ones
  w.begin = first + w.part * each + min(w.part, more);
  w.count = each + (w.part < more);
  return true;
}

// A part without tiles of a row that others share: the merge looks no further than its maximum.
template <int kRows, int kThreads>
__device__ __forceinline__ bool nothing_to_do(const PagedArgs& a, const Work& w) {
  if (w.parts == 1 || w.count > 0) return false;
  for (int i = threadIdx.x; i < min(kRows, w.rows - w.r0); i += kThreads)
    a.pmax[long(w.slot) * w.rows + w.r0 + i] = -INFINITY;
  return true;
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

// A scale as it is, or 1 for what a page that was never written may hold: the codes beside
// tokens in sight are zeros then, and zeros have to stay.
__device__ __forceinline__ float usable(float scale) { return fabsf(scale) < INFINITY ? scale : 1.f; }

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

  // Of the lane's part of a row of K.
  static __device__ __forceinline__ int part(int g) { return D >= 64 ? 16 * g : D == 32 ? 8 * g : 8 * (g & 1); }
  static __device__ __forceinline__ void load_k(const uint8_t* at, int g, uint32_t (&w)[kWords]) {
    if constexpr (D >= 64) {
#pragma unroll
      for (int e = 0; e < D / 64; ++e) {
        const u32x4 r = *reinterpret_cast<const u32x4*>(at + 64 * e);
#pragma unroll
        for (int x = 0; x < 4; ++x) w[4 * e + x] = r[x];
      }
    } else {
      const u32x2 r = *reinterpret_cast<const u32x2*>(at);
      w[0] = D == 16 && g > 1 ? 0u : r[0], w[1] = D == 16 && g > 1 ? 0u : r[1];
    }
  }
};

// Eight values of q as pieces, cut rather than rounded so that the pieces' sum is the value
// (zeros where not `on`).
template <typename T>
__device__ __forceinline__ void load_pieces(const T* at, bool on, u32x4 (&q)[pieces_of<T>()]) {
  constexpr int P = pieces_of<T>(), E = vec_elems<T>();
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
        q[p][e] = on ? (lo >> 16) | (hi & 0xffff0000u) : 0u;
        x[2 * e] -= __uint_as_float(lo & 0xffff0000u);
        x[2 * e + 1] -= __uint_as_float(hi & 0xffff0000u);
      }
  }
}

// Eight probabilities as pieces, each what the ones before it leave, rounded.
template <int P>
__device__ __forceinline__ void split_pieces(float (&x)[8], u32x4 (&prob)[P]) {
#pragma unroll
  for (int p = 0; p < P; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = pack2<bf16_t>(x[2 * e], x[2 * e + 1]);
      prob[p][e] = w;
      x[2 * e] -= bf16_lo(w), x[2 * e + 1] -= bf16_hi(w);
    }
}

// Ones in bf16 where eight codes are NaN, zeros elsewhere.
__device__ __forceinline__ u32x4 nan_ones(uint32_t lo, uint32_t hi) {
  const uint32_t m[2] = {nan_bytes(lo), nan_bytes(hi)};
  u32x4 r;
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    r[2 * x] = (m[x] & 0xff ? 0x3f80u : 0u) | (m[x] & 0xff00 ? 0x3f800000u : 0u);
    r[2 * x + 1] = (m[x] & 0xff0000 ? 0x3f80u : 0u) | (m[x] & 0xff000000u ? 0x3f800000u : 0u);
  }
  return r;
}

template <typename T>
__device__ __forceinline__ void store4(T* p, const float* v) {
  if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
  }
}

// Values are read once, past the caches, where a tile has whole lines of them. Pages of 128
// tokens have two tiles to a line.
template <int kPage>
__device__ __forceinline__ u32x4 load_v(const uint8_t* at) {
  const u32x4* p = reinterpret_cast<const u32x4*>(at);
  return kPage == 128 ? *p : __builtin_nontemporal_load(p);
}

// A workgroup has up to 16 NC query rows (the G heads of a KV head times the tokens, row
// r = t G + g) and a split of the keys; its waves take the split's tiles in turn and are
// joined through LDS at the end. Codes go from memory to registers: a tile's values are asked
// for before or among its products with K, the next tile's keys before its softmax. Nothing
// stays under way from one tile to the next: keys are asked for on one of two paths (not on
// the last tile's), so the waits before the products with V, which have to hold on both, let
// the keys arrive, too; the other seven waves are what fills the time. Bound by HBM: 32 rows of
// 8000 tokens of 8 heads of 128 84 us (537 MB, 6.4 TB/s), of 1K to 8K 52 (314 MB, 6.0, the matrix
// cores busy for 13% of it, vector instructions for 28%), one of 131072 48 (274 MB, 5.6); a CU alone
// reads 35 GB/s, so a head wants about 30 workgroups. Both ways measured, us at those two: values past the caches 58, 57 and through them 63, 52
// (pages of 64, pages of 128); both tiles' values ahead 58, 57; 4, 6, 8 and 12 waves 57, 56,
// 56, 56 at their best splits, 8 for one short row (11 us for 1024 keys, where two splits and
// their merge take 13.5); three waves a SIMD instead of two 60.
template <typename T, int D, int NC, int kPage, int W>
__global__ __launch_bounds__(W * kWave, D == 128 && NC == 2 ? 1 : 2) void paged_attention_kernel(const PagedArgs a) {
  using L = Tile<D>;
  constexpr bool kWide = kPage >= kPagedTile;
  constexpr int P = pieces_of<T>(), BT = kPagedTile, kRows = 16 * NC, kLine = D + 4;
  constexpr int kProb = prob_pieces_of<T>();
  __shared__ float merged[W][kRows][kLine];
  __shared__ float tops[W][kRows], sums[W][kRows];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave, g = lane / 16, n = lane % 16;
  Work work;
  if (!find_work(a, kRows, work) || nothing_to_do<kRows, W * kWave>(a, work)) return;
  const int b = work.b, hk = work.hk, r0 = work.r0, rows = work.rows, G = 1 << a.group_log2;
  const PagedRow row = work.row;
  const int t0 = work.t0, t1 = work.t1, start = work.start, end = work.end;
  const int begin = work.begin, stop = work.begin + work.count;

  u32x4 q[NC][L::kSteps][P];
  int seen_from[NC], seen_to[NC];  // first and last slot of the lane's query row
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int r = min(r0 + 16 * c + n, rows - 1), t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
    const T* at = static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[1] + t * a.qs[2];
#pragma unroll
    for (int s = 0; s < L::kSteps; ++s) load_pieces<T>(at + L::dim(s, D > 16 ? g : g & 1), D > 16 || g < 2, q[c][s]);
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

  // The pages of the wave's next tiles, one or (pages of less than a tile) four to a tile, and
  // their scales, a lane each: nothing in the loop below waits for a page before it can ask
  // for its rows.
  constexpr int kSpots = kWide ? 1 : 4, kBatch = kWave / kSpots;
  const int32_t* table = a.tables + long(b) * a.places;
  const int page_mask = (1 << a.page_log2) - 1;
  const int count = stop - begin - wave > 0 ? (stop - begin - wave + W - 1) / W : 0;  // the wave's tiles
  const auto tile_of = [&](int i) { return begin + wave + W * i; };
  int spots = -1;  // -1: no page
  float spots_ks = 0.f, spots_vs = 0.f;
  const auto look_up = [&](int i) {
    const int slot = tile_of(min(i + lane / kSpots, count - 1)) * BT + lane % kSpots * 16;
    const int page = table[min(slot >> a.page_log2, a.places - 1)];
    spots = slot < row.cap && page >= 0 && page < a.pages ? page : -1;
    const long block = long(max(spots, 0)) * a.kv_heads + hk;
    spots_ks = usable(a.k_scale[block]), spots_vs = usable(a.v_scale[block]);
  };
  const auto pick = [&](auto x, int i, int sub) {  // of tile i's keys from 16 sub on
    const uint32_t bits = __builtin_bit_cast(uint32_t, x);
    const uint32_t got = kWide ? __builtin_amdgcn_readlane(bits, i % kBatch) : uint32_t(__shfl(int(bits), i % kBatch * kSpots + sub));
    return __builtin_bit_cast(decltype(x), got);
  };

  const int off_k = n / 4 * 16, off_v = g * 16;  // of the lane's keys in a tile
  const int sub_k = kWide ? 0 : off_k, sub_v = kWide ? 0 : off_v;
  uint32_t kw[4][L::kWords];
  float ks = 0.f;
  const auto fetch_k = [&](int i) {
    const long block = long(max(pick(spots, i, n / 4), 0)) * a.kv_heads + hk;
    ks = pick(spots_ks, i, n / 4);
    const uint8_t* base = a.k + ((block << a.page_log2) + ((tile_of(i) * BT + sub_k) & page_mask)) * D;
    const unsigned lane_at = unsigned(((kWide ? off_k : 0) + n % 4) * D + L::part(g));
#pragma unroll
    for (int t = 0; t < 4; ++t) L::load_k(base + lane_at + 4 * t * D, g, kw[t]);
  };
  // Tiles that some row does not see whole.
  const auto partly_seen = [&](int slot0, int spot) {
    return slot0 + BT - 1 > row.len + t0 || (a.window >= 0 && slot0 < row.len + t1 - a.window) || __any(spot < 0);
  };
  const auto sees = [&](int c, int slot, int spot) { return spot >= 0 && slot <= seen_to[c] && slot >= seen_from[c]; };
  bool found = false;  // NaN among the values of such a tile

  if (count > 0) {
    look_up(0);
    fetch_k(0);
  }
  for (int i = 0; i < count; ++i) {
    const int slot0 = tile_of(i) * BT, spot = pick(spots, i, g);
    u32x4 vw[L::kDims];
    const float vs = pick(spots_vs, i, g);
    const uint8_t* base = a.v + (((long(max(spot, 0)) * a.kv_heads + hk) * D) << a.page_log2) + ((slot0 + sub_v) & page_mask);
    const unsigned lane_at = unsigned((n << a.page_log2) + (kWide ? off_v : 0));
#pragma unroll
    for (int d = 0; d < L::kDims; ++d)
      vw[d] = load_v<kPage>(base + (d * 16 << a.page_log2) + lane_at);

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
    if (i + 1 < count) {
      if ((i + 1) % kBatch == 0) look_up(i + 1);
      fetch_k(i + 1);
    }

    const bool masked = partly_seen(slot0, spot);
    if (masked) {
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[c][e / 4][e % 4] = sees(c, slot0 + off_v + e, spot) ? s[c][e / 4][e % 4] : -INFINITY;
    }
    u32x4 prob[NC][2][kProb];
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
#pragma unroll
      for (int y = 0; y < 2; ++y) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_amdgcn_exp2f(fmaf(s[c][2 * y + e / 4][e % 4], a.cs, -base));
          sum[c] += x[e];
        }
        split_pieces(x, prob[c][y]);
      }
    }
    if (masked) {
      // Values of slots that nobody sees become zeros: old codes there may be NaN. NaN in slots
      // that some rows see and some do not is zero here, too, and put into its rows below.
      const int from = start - (slot0 + off_v), to = spot >= 0 ? end - (slot0 + off_v) : 0;
      uint32_t bad = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const uint32_t keep = first_bytes(to - 4 * x) & ~first_bytes(from - 4 * x);
#pragma unroll
        for (int d = 0; d < L::kDims; ++d) {
          const uint32_t w = vw[d][x] & keep, is_nan = nan_bytes(w);
          vw[d][x] = w & ~is_nan;
          bad |= is_nan;
        }
      }
      found |= __any(bad != 0);
    }
#pragma unroll
    for (int d = 0; d < L::kDims; ++d)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const u32x4 value = from_codes(vw[d][2 * h], vw[d][2 * h + 1], vs);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int p = kProb - 1; p >= 0; --p) o[c][d] = mfma16(value, prob[c][h][p], o[c][d]);
      }
  }
  if (found) {
    // Which rows see a NaN, as products of what is NaN with what is seen.
    for (int i = 0; i < count; ++i) {
      if (i % kBatch == 0) look_up(i);
      const int slot0 = tile_of(i) * BT, spot = pick(spots, i, g);
      if (!partly_seen(slot0, spot)) continue;
      u32x4 on[NC][2];
#pragma unroll
      for (int c = 0; c < NC; ++c)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          on[c][e / 4][e % 4] = (sees(c, slot0 + off_v + 2 * e, spot) ? 0x3f80u : 0u) |
                                (sees(c, slot0 + off_v + 2 * e + 1, spot) ? 0x3f800000u : 0u);
      const uint8_t* at = a.v + (((long(max(spot, 0)) * a.kv_heads + hk) * D + n) << a.page_log2) + ((slot0 + off_v) & page_mask);
#pragma unroll
      for (int d = 0; d < L::kDims; ++d) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(at + (d * 16 << a.page_log2));
#pragma unroll
        for (int c = 0; c < NC; ++c) {
          f32x4 hits = mfma16(nan_ones(w[0], w[1]), on[c][0], f32x4{0.f, 0.f, 0.f, 0.f});
          hits = mfma16(nan_ones(w[2], w[3]), on[c][1], hits);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[c][d][e] = hits[e] > 0.f ? NAN : o[c][d][e];
        }
        __builtin_amdgcn_sched_barrier(0);  // few registers rather than many loads at once
      }
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
    if (work.parts > 1) {
      const long to = long(work.slot) * rows + r;
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

// The same for more rows: W waves with 32 query rows each, and tiles of 64 keys that they
// share. A tile's codes are read once into LDS as they are (K [key][dim], V [dim][key],
// 16-byte slots swizzled by row) and become bf16 operands of 32 x 32 x 16 MFMAs on their way
// out of it, the next tile's codes under way meanwhile. A lane's 16 codes are its k-slots in
// two products: in those with K dims 32 x + 16 h .. + 15 of a key, in those with V keys
// 32 x + 16 h .. + 15 of a dim (lane = 32 h + n). So that lane (h, n) holds the scores of the
// latter, row m of S^T takes the key 16 (m / 4 % 2) + 8 (m / 16) + 4 (m / 8 % 2) + m % 4 of its 32.
// Bound by a wave's chain, its products and its vector instructions (48 products of 32 cycles
// beside 128 conversions, 32 exponentials and their pieces, some 400 in all, to a tile of 32 rows
// of 128 in bf16): 512 rows over 32000 keys of 8 heads 110 us with the merge (610 TFLOP/s), 27
// tokens of 4 heads over 8 rows of 1K to 8K 46 (350), the matrix cores busy for 42% of it, vector
// instructions for 57%. Measured with the probabilities as one piece, where those two took 87
// and 37: tiles staged as bf16 (a conversion for four waves, twice the LDS bytes) 89; two buffers
// and one barrier a tile 90; the products of the tile before between this tile's exponentials
// 89 to 95; two teams of four waves to a workgroup 86 at half the splits, but 51 where 37 + 7
// stand for rows of different length.
template <typename T, int D, int kPage>
__global__ __launch_bounds__(kRowWaves * kWave, 2) void paged_rows_kernel(const PagedArgs a) {
  constexpr bool kWide = kPage >= kPagedTile;
  constexpr int P = pieces_of<T>(), BT = kPagedTile, kRows = 32 * kRowWaves, kThreads = kRowWaves * kWave;
  constexpr int kProb = prob_pieces_of<T>();
  constexpr int kSteps = D / 16, kTiles = D / 32;          // of the products with K, of dims of V
  constexpr int kPieces = BT * D / 16 / kThreads;          // of 16 codes of a tile's keys a thread stages
  constexpr int kSpots = kWide ? 1 : 4, kBatch = kWave / kSpots;
  __shared__ u32x4 keys[BT * D / 16], values[D * BT / 16];
  __shared__ int found;
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave);
  const int lane = threadIdx.x % kWave, h = lane / 32, n = lane % 32;
  Work work;
  if (!find_work(a, kRows, work) || nothing_to_do<kRows, kThreads>(a, work)) return;
  const int b = work.b, hk = work.hk, r0 = work.r0, rows = work.rows, G = 1 << a.group_log2;
  const PagedRow row = work.row;
  const int t0 = work.t0, t1 = work.t1, start = work.start, end = work.end, begin = work.begin, count = work.count;

  const bool active = r0 + 32 * wave < rows;
  const int r = min(r0 + 32 * wave + n, rows - 1), t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
  const int seen_to = t < row.count ? row.len + t : -1, seen_from = a.window >= 0 ? row.len + t - a.window : 0;
  u32x4 q[kSteps][P];
  {
    const T* at = static_cast<const T*>(a.q) + b * a.qs[0] + head * a.qs[1] + t * a.qs[2] + 16 * h;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) load_pieces<T>(at + s / 2 * 32 + s % 2 * 8, true, q[s]);
  }
  f32x16 o[kTiles];
#pragma unroll
  for (int d = 0; d < kTiles; ++d)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[d][e] = 0.f;
  float top = -INFINITY, sum = 0.f;

  const int32_t* table = a.tables + long(b) * a.places;
  const int page_mask = (1 << a.page_log2) - 1;
  int spots = -1;
  float spots_ks = 0.f, spots_vs = 0.f;
  const auto look_up = [&](int i) {
    const int slot = (begin + min(i + lane / kSpots, count - 1)) * BT + lane % kSpots * 16;
    const int page = table[min(slot >> a.page_log2, a.places - 1)];
    spots = slot < row.cap && page >= 0 && page < a.pages ? page : -1;
    const long block = long(max(spots, 0)) * a.kv_heads + hk;
    spots_ks = usable(a.k_scale[block]), spots_vs = usable(a.v_scale[block]);
  };
  const auto pick = [&](auto x, int i, int sub) {
    const uint32_t bits = __builtin_bit_cast(uint32_t, x);
    const uint32_t got = kWide ? __builtin_amdgcn_readlane(bits, i % kBatch) : uint32_t(__shfl(int(bits), i % kBatch * kSpots + sub));
    return __builtin_bit_cast(decltype(x), got);
  };
  // A thread's pieces: 16 dims of a key, 16 keys of a dim.
  u32x4 kw[kPieces], vw[kPieces];
  bool kept[kPieces];
  const auto fetch = [&](int i) {
    const int slot0 = (begin + i) * BT;
#pragma unroll
    for (int e = 0; e < kPieces; ++e) {
      const int x = int(threadIdx.x) + kThreads * e, key = x / (D / 16), dim = x / 4;
      const int page_k = pick(spots, i, key / 16), page_v = pick(spots, i, x % 4);
      kept[e] = page_v >= 0;
      const long block_k = long(max(page_k, 0)) * a.kv_heads + hk, block_v = long(max(page_v, 0)) * a.kv_heads + hk;
      kw[e] = *reinterpret_cast<const u32x4*>(a.k + ((block_k << a.page_log2) + ((slot0 + key) & page_mask)) * D + x % (D / 16) * 16);
      vw[e] = *reinterpret_cast<const u32x4*>(a.v + ((block_v * D + dim) << a.page_log2) + ((slot0 + x % 4 * 16) & page_mask));
    }
  };
  const auto partly_seen = [&](int slot0, bool whole) {
    return slot0 + BT - 1 > row.len + t0 || (a.window >= 0 && slot0 < row.len + t1 - a.window) || !whole;
  };
  // Whether all of tile i's keys have a page.
  const auto whole_tile = [&](int i) { return kWide ? pick(spots, i, 0) >= 0 : !__any(pick(spots, i, lane % 4) < 0); };
  const int key_row = 16 * (n / 4 % 2) + 8 * (n / 16) + 4 * (n / 8 % 2) + n % 4;
  const auto key_slot = [](int key, int x) { return key * (D / 16) + (x ^ (D == 128 ? key / 2 % 8 : key / 4 % 4)); };
  const auto value_slot = [](int dim, int x) { return dim * 4 + (x ^ dim / 4 % 4); };

  if (threadIdx.x == 0) found = 0;
  __syncthreads();  // before a wave that is ahead finds something
  if (count > 0) {
    look_up(0);
    fetch(0);
  }
  for (int i = 0; i < count; ++i) {
    const int slot0 = (begin + i) * BT;
    const bool masked = partly_seen(slot0, whole_tile(i));
    const int missing = masked ? (kWide ? (pick(spots, i, 0) < 0 ? 15 : 0) : int(__ballot(pick(spots, i, lane % 4) < 0) & 15)) : 0;
    if (masked) {
      // Values that nobody sees become zeros, and so does NaN, which goes to its rows at the end.
      uint32_t bad = 0;
#pragma unroll
      for (int e = 0; e < kPieces; ++e) {
        const int at = slot0 + (int(threadIdx.x) + kThreads * e) % 4 * 16;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const uint32_t keep = kept[e] ? first_bytes(end - at - 4 * x) & ~first_bytes(start - at - 4 * x) : 0u;
          const uint32_t w = vw[e][x] & keep, is_nan = nan_bytes(w);
          vw[e][x] = w & ~is_nan;
          bad |= is_nan;
        }
      }
      if (bad) found = 1;
    }
    __syncthreads();  // the last tile's operands are read
#pragma unroll
    for (int e = 0; e < kPieces; ++e) {
      const int x = int(threadIdx.x) + kThreads * e;
      keys[key_slot(x / (D / 16), x % (D / 16))] = kw[e];
      values[value_slot(x / 4, x % 4)] = vw[e];
    }
    float ks[2], vs[2];  // of the lane's keys in the two halves of the tile
#pragma unroll
    for (int half = 0; half < 2; ++half)
      ks[half] = pick(spots_ks, i, 2 * half + key_row / 16), vs[half] = pick(spots_vs, i, 2 * half + h);
    __syncthreads();
    if (i + 1 < count) {
      if ((i + 1) % kBatch == 0) look_up(i + 1);
      fetch(i + 1);
    }
    if (!active) continue;

    f32x16 s[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[half][e] = 0.f;
      const int key = 32 * half + key_row;
#pragma unroll
      for (int st = 0; st < kSteps; st += 2) {
        const u32x4 w = keys[key_slot(key, st + h)];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const u32x4 x = from_codes(w[2 * y], w[2 * y + 1], ks[half]);
#pragma unroll
          for (int p = P - 1; p >= 0; --p) s[half] = mfma32<bf16_t>(x, q[st + y][p], s[half]);
        }
      }
    }
    if (masked) {
#pragma unroll
      for (int half = 0; half < 2; ++half)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int at = 32 * half + 16 * h + e;
          const bool on = slot0 + at <= seen_to && slot0 + at >= seen_from && !(missing >> (2 * half + h) & 1);
          s[half][e] = on ? s[half][e] : -INFINITY;
        }
    }
    float high = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) high = fmaxf(high, s[e / 16][e % 16]);
    high = fmaxf(high, lane_xor(high, 32)) * a.cs;
    const bool raise = high > top + kLazyMax;
    if (__any(raise)) {
      const float now = raise ? high : top;
      const float keep = raise ? __builtin_amdgcn_exp2f(top - now) : 1.f;
      top = now;
      sum *= keep;
#pragma unroll
      for (int d = 0; d < kTiles; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] *= keep;
    }
    const float base = top == -INFINITY ? 0.f : top;
    u32x4 prob[4][kProb];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        y[e] = __builtin_amdgcn_exp2f(fmaf(s[x / 2][x % 2 * 8 + e], a.cs, -base));
        sum += y[e];
      }
      split_pieces(y, prob[x]);
    }
#pragma unroll
    for (int d = 0; d < kTiles; ++d)
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const u32x4 w = values[value_slot(32 * d + n, 2 * x + h)];
#pragma unroll
        for (int y = 0; y < 2; ++y) {
          const u32x4 v = from_codes(w[2 * y], w[2 * y + 1], vs[x]);
#pragma unroll
          for (int p = kProb - 1; p >= 0; --p) o[d] = mfma32<bf16_t>(v, prob[2 * x + y][p], o[d]);
        }
      }
  }
  __syncthreads();
  if (!active) return;
  if (found) {
    for (int i = 0; i < count; ++i) {
      if (i % kBatch == 0) look_up(i);
      const int slot0 = (begin + i) * BT;
      if (!partly_seen(slot0, whole_tile(i))) continue;
#pragma unroll 1
      for (int x = 0; x < 4; ++x) {
        const int spot = pick(spots, i, x / 2 * 2 + h), slot = slot0 + x / 2 * 32 + 16 * h + x % 2 * 8;
        u32x4 on;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const auto sees = [&](int at) { return spot >= 0 && at <= seen_to && at >= seen_from; };
          on[e] = (sees(slot + 2 * e) ? 0x3f80u : 0u) | (sees(slot + 2 * e + 1) ? 0x3f800000u : 0u);
        }
        const uint8_t* at = a.v + (((long(max(spot, 0)) * a.kv_heads + hk) * D + n) << a.page_log2) + (slot & page_mask);
#pragma unroll
        for (int d = 0; d < kTiles; ++d) {
          const u32x2 w = *reinterpret_cast<const u32x2*>(at + (d * 32 << a.page_log2));
          f32x16 hits;
#pragma unroll
          for (int e = 0; e < 16; ++e) hits[e] = 0.f;
          hits = mfma32<bf16_t>(nan_ones(w[0], w[1]), on, hits);
#pragma unroll
          for (int e = 0; e < 16; ++e) o[d][e] = hits[e] > 0.f ? NAN : o[d][e];
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
  }
  sum += lane_xor(sum, 32);
  if (top == -INFINITY && sum != sum) top = 0.f;  // as above
  if (r0 + 32 * wave + n >= rows) return;
  const bool empty = top == -INFINITY || t >= row.count;
  const long to = long(work.slot) * rows + r;
  if (h == 0) {
    if (work.parts > 1)
      a.pmax[to] = top, a.psum[to] = sum;
    else
      a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (top + __builtin_log2f(sum)) * kLn2;
  }
  T* out = static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
  const float share = work.parts > 1 ? 1.f : empty ? 0.f : 1.f / sum;
#pragma unroll
  for (int d = 0; d < kTiles; ++d)
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      float num[4];
      const int dim = 32 * d + 8 * x + 4 * h;
#pragma unroll
      for (int e = 0; e < 4; ++e) num[e] = empty && work.parts == 1 ? 0.f : o[d][4 * x + e] * share;
      if (work.parts > 1)
        store4<float>(a.pout + to * D + dim, num);
      else
        store4<T>(out + dim, num);
    }
}

// The splits of a row joined. A wave has a row, or with `kShared` a workgroup has one and
// its four waves every fourth round of splits; kRound splits' loads go out together. A
// chain of latencies for few rows (1024 of 2 splits 4.8 us; 32 of 32 splits 4.8, with a wave to
// a row 6.0), memory for many (6912 of 8 splits, 32 MB read, 8.3).
template <typename T, int D, bool kShared>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedArgs a) {
  constexpr int DPL = (D + kWave - 1) / kWave, kRound = 8, W = kShared ? 4 : 1;
  __shared__ float nums[kShared ? 4 : 1][D], tops[4], dens[4];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int rows = a.tokens << a.group_log2, G = 1 << a.group_log2;
  const long at = kShared ? long(blockIdx.x) : long(blockIdx.x) * 4 + wave;
  if (at >= long(a.groups) * rows) return;
  const int group = __builtin_amdgcn_readfirstlane(int(at / rows)), r = int(at - long(group) * rows);
  const int b = group / a.kv_heads, hk = group - b * a.kv_heads;
  const PagedRow row = paged_row(a, b);
  const int parts = parts_of(a, row);
  if (parts == 1) return;  // written already
  int more = 0;  // slot of the row's first part beyond `splits`, less that part's number
  if (parts > a.splits)
    more = a.groups * a.splits + min(more_before(a, b) + hk * (parts - a.splits), a.more - (parts - a.splits)) - a.splits;
  const int t = r >> a.group_log2, head = (hk << a.group_log2) + (r & (G - 1));
  float top = -INFINITY, den = 0.f, num[DPL] = {};
  for (int s0 = kShared ? wave * kRound : 0; s0 < parts; s0 += kRound * W) {
    const auto part = [&](int s) {
      const int x = min(s0 + s, parts - 1);
      return long(x < a.splits ? group * a.splits + x : more + x) * rows + r;
    };
    const bool on = lane < kRound && s0 + lane < parts;
    const float high = a.pmax[part(lane % kRound)], sum = a.psum[part(lane % kRound)];
    float x[kRound][DPL];
#pragma unroll
    for (int s = 0; s < kRound; ++s)
#pragma unroll
      for (int i = 0; i < DPL; ++i) x[s][i] = a.pout[part(s) * D + min(lane + i * kWave, D - 1)];
    const float mine = on ? high : -INFINITY;
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
  if constexpr (kShared) {
#pragma unroll
    for (int i = 0; i < DPL; ++i)
      if (lane + i * kWave < D) nums[wave][lane + i * kWave] = num[i];
    if (lane == 0) tops[wave] = top, dens[wave] = den;
    __syncthreads();
    if (wave) return;
    top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
    den = 0.f;
#pragma unroll
    for (int i = 0; i < DPL; ++i) num[i] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const bool on = tops[w] != -INFINITY;
      const float weight = on ? __builtin_amdgcn_exp2f(tops[w] - top) : 0.f;
      den = on ? fmaf(weight, dens[w], den) : den;
#pragma unroll
      for (int i = 0; i < DPL; ++i) num[i] = on ? fmaf(weight, nums[w][min(lane + i * kWave, D - 1)], num[i]) : num[i];
    }
  }
  const bool empty = top == -INFINITY || t >= row.count;
  T* o = static_cast<T*>(a.out) + b * a.os[0] + head * a.os[1] + t * a.os[2];
#pragma unroll
  for (int i = 0; i < DPL; ++i)
    if (lane + i * kWave < D) store_scalar<T>(o + lane + i * kWave, empty ? 0.f : num[i] / den);
  if (lane == 0)
    a.lse[(long(b) * a.kv_heads * G + head) * a.tokens + t] = empty ? -INFINITY : (top + __builtin_log2f(den)) * kLn2;
}

constexpr long kMostThreads = 1L << 32;  // a launch holds fewer

template <typename T, int D>
int launch_paged(PagedArgs& a, hipStream_t stream) {
  const char* what = "page_attention";
  const int rows = a.tokens << a.group_log2;
  // By rows, us at the best number of splits with blocks of 16 / 32 rows / 128 that share
  // tiles: bf16 D 128 2 x 8000 keys of 8 heads 32 rows 15.6 / 16.7 / 21.5, 8 x 4000 of 16
  // heads 40 rows 52.9 / 39.9 / 51.2, 8 x 8000 of 8 heads 64 rows 51.8 / 43.0 / 53.3, 8 of 1K
  // to 8K 108 rows 67.5 / 56.7 / 49.6, 4 x 8000 128 rows 57.9 / 41.4 / 40.6, 16 x 4000 128 rows
  // 104.8 / 72.6 / 67.7, 32000 keys 512 rows 190 / 128 / 107; fp16, whose pieces leave blocks of 32 rows too few registers, 8 x up to 8000 40
  // rows 37.3 / 43.6 / 59, D 64 8 x 8000 128 rows - / 49.9 / 48; fp32 4 x 4000 128 rows 32.3 /
  // 39.4, D 64 8 x 4000 128 rows 34.1 / 37.2; D 32 8 x 4000 128 rows 17.7 / 21.1.
  constexpr bool kPairs = pieces_of<T>() == 1 && D >= 64, kShares = pieces_of<T>() < 3 && D >= 64;
  const int block = rows > 64 && kShares ? 128 : rows > 32 && kPairs ? 32 : 16;
  const int threads = (block == 16 ? 8 : kRowWaves) * kWave;  // kernels below
  a.row_blocks = (rows + block - 1) / block;
  a.share = float(a.kv_heads) * a.row_blocks / kAtOnce;
  // Sequences of more than `splits` parts have together fewer parts than kAtOnce / row_blocks.
  a.more = a.most > a.splits ? kAtOnce / a.row_blocks + 1 : 0;
  const long units = (long(a.groups) * a.splits + a.more + kXcds - 1) / kXcds * kXcds;
  const long merged = long(a.groups) * rows;
  if (units * a.row_blocks * threads >= kMostThreads || (merged + 3) * 256 >= kMostThreads)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: too many workgroups", what);
  const auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(unsigned(units * a.row_blocks)), dim3(unsigned(threads)), 0, stream, a);
  };
  const auto run = [&](auto page) {
    constexpr int kPage = decltype(page)::value;
    if constexpr (kShares)
      if (block == 128) return launch(paged_rows_kernel<T, D, kPage>);
    if constexpr (kPairs)
      if (block == 32) return launch(paged_attention_kernel<T, D, 2, kPage, kRowWaves>);
    launch(paged_attention_kernel<T, D, 1, kPage, 8>);
  };
  if (a.page_log2 == 7) run(std::integral_constant<int, 128>{});
  else if (a.page_log2 == 6) run(std::integral_constant<int, 64>{});
  else run(std::integral_constant<int, 16>{});  // pages of less than a tile
  if (int rc = check_launch(what)) return rc;
  if (a.most == 1) return SFL_OK;
  if (a.splits > 8 || (a.most > 8 && merged <= 2048))
    hipLaunchKernelGGL((paged_merge_kernel<T, D, true>), dim3(unsigned(merged)), dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_merge_kernel<T, D, false>), dim3(unsigned((merged + 3) / 4)), dim3(256), 0, stream, a);
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
                                  int splits, int most_splits, float scale, int dtype, void* stream) {
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
  if (splits < 1 || most_splits < splits || most_splits > 1024)
    return set_error(SFL_ERR_INVALID, "%s: splits must be in [1, 1024], most_splits in [splits, 1024]", what);
  if (most_splits > 1 && (!partial_max || !partial_sum || !partial_out))
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
  a.group_log2 = ratio == 8 ? 3 : ratio / 2, a.groups = batch * kv_heads;
  a.splits = splits, a.most = most_splits, a.batch = batch;
  a.window = std::max(window_left, -1);
  a.cs = scale * kLog2e;
  return paged_types(dtype, head_dim, [&](auto t, auto d) {
    return launch_paged<decltype(t), decltype(d)::value>(a, static_cast<hipStream_t>(stream));
  });
}
