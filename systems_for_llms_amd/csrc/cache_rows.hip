// Rows of a KV cache: new tokens' q, k and v normed, rotated and written into it,
// an accepted path moved behind the committed rows, and the rows of an eviction's
// kept slots moved into the places that become free. All of it moves bytes: the
// bound is memory, and below a few hundred KB the launch.
#include <limits.h>

#include <algorithm>
#include <type_traits>

#include "attn_mfma.hpp"

namespace sfl {
namespace {

struct RotateArgs {
  const void *q, *k, *v;
  const int32_t* positions;
  const float *cos, *sin;
  const void *q_gain, *k_gain;
  const int32_t *start, *counts;
  void *q_out, *k_out, *v_out;
  long st[6][3];  // strides in elements (batch, head, token) of q, k, v, q_out, k_out, v_out
  int batch, tokens, q_heads, kv_heads, half, table, slots, gain_f32;
  float eps;
};

// One row of the launch: token t of sequence b, head h of q, then k, then v.
struct RotateRow {
  const void* in;
  void* out;
  const void* gain;
  bool turn;   // q and k; v is copied
  bool store;  // whether the row has a place
  bool zero;   // padding of an output that is not a cache
};
template <typename T>
__device__ __forceinline__ RotateRow rotate_row(const RotateArgs& a, int b, int t, int h) {
  const int which = h < a.q_heads ? 0 : h < a.q_heads + a.kv_heads ? 1 : 2;
  const int head = which == 0 ? h : which == 1 ? h - a.q_heads : h - a.q_heads - a.kv_heads;
  const bool used = !a.counts || t < a.counts[b];
  // q goes to token t of its output; k and v to slot start + t of the cache, where it has that slot.
  const long slot = which && a.start ? long(a.start[b]) + t : t;
  RotateRow r;
  // Strides by selection: an index that is not a constant would put the arguments into scratch memory.
  const auto at = [&](int first, long row, int i) {
    return b * a.st[first + i][0] + head * a.st[first + i][1] + row * a.st[first + i][2];
  };
  r.in = which == 0 ? static_cast<const T*>(a.q) + at(0, t, 0)
         : which == 1 ? static_cast<const T*>(a.k) + at(0, t, 1) : static_cast<const T*>(a.v) + at(0, t, 2);
  r.out = which == 0 ? static_cast<T*>(a.q_out) + at(3, slot, 0)
          : which == 1 ? static_cast<T*>(a.k_out) + at(3, slot, 1) : static_cast<T*>(a.v_out) + at(3, slot, 2);
  r.gain = which == 0 ? a.q_gain : which == 1 ? a.k_gain : nullptr;
  r.turn = which < 2;
  r.zero = !used;
  r.store = which == 0 || !a.start || (used && slot >= 0 && slot < a.slots);
  return r;
}

__device__ __forceinline__ float gain_at(const RotateArgs& a, const void* gain, int d, float) {
  return static_cast<const float*>(gain)[d];
}
template <typename T>
__device__ __forceinline__ float gain_at(const RotateArgs& a, const void* gain, int d, T) {
  return a.gain_f32 ? static_cast<const float*>(gain)[d] : load_scalar<T>(static_cast<const T*>(gain) + d);
}

// One wave per row, a row staged in LDS as fp32: any layout, rotated part and alignment.
// Bound by its scalar accesses: 4 x 4001 tokens of 48 fp16 heads of 128 390 us, in
// 16-byte pieces (below) 82.
template <typename T, bool kHalfLayout>
__global__ __launch_bounds__(256) void rotate_any_kernel(const RotateArgs a, int dim, unsigned rows, unsigned heads) {
  __shared__ float stage[4][128];
  const int wave = __builtin_amdgcn_readfirstlane(int(threadIdx.x) / kWave), lane = threadIdx.x % kWave;
  for (unsigned row0 = blockIdx.x * 4; row0 < rows; row0 += gridDim.x * 4) {
    const unsigned at = min(row0 + unsigned(wave), rows - 1);  // the last workgroup's missing rows repeat the last one
    const unsigned token = at / heads;
    const int h = int(at - token * heads), b = int(token / unsigned(a.tokens)), t = int(token - unsigned(b) * unsigned(a.tokens));
    const RotateRow r = rotate_row<T>(a, b, t, h);
    float x[2], sq = 0.f;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = lane + kWave * e;
      x[e] = d < dim ? load_scalar<T>(static_cast<const T*>(r.in) + d) : 0.f;
      sq = fmaf(x[e], x[e], sq);
    }
    if (r.gain) {
      const float scale = 1.f / sqrtf(wave_sum(sq) / float(dim) + a.eps);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        if (lane + kWave * e < dim) x[e] *= scale * gain_at(a, r.gain, lane + kWave * e, T{});
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + kWave * e < dim) stage[wave][lane + kWave * e] = x[e];
    __syncthreads();
    const int pos = a.positions[long(b) * a.tokens + t];
    const bool known = pos >= 0 && pos < a.table;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int d = lane + kWave * e;
      if (d >= dim || !r.store) continue;
      float y = x[e];
      if (r.turn && d < 2 * a.half) {
        const int i = kHalfLayout ? d % a.half : d / 2;
        const bool second = kHalfLayout ? d >= a.half : d & 1;
        const float other = stage[wave][kHalfLayout ? (second ? d - a.half : d + a.half) : d ^ 1];
        const float c = known ? a.cos[long(pos) * a.half + i] : NAN, s = known ? a.sin[long(pos) * a.half + i] : NAN;
        y = second ? fmaf(other, s, y * c) : fmaf(-other, s, y * c);
      }
      store_scalar<T>(static_cast<T*>(r.out) + d, r.zero ? 0.f : y);
    }
    __syncthreads();  // before the next rows' values
  }
}

// N values (8, 16 or 32 bytes) as fp32.
template <typename T, int N>
__device__ __forceinline__ void load_values(const T* p, float (&v)[N]) {
  if constexpr (std::is_same<T, float>::value && N == 2) {
    const float2 r = *reinterpret_cast<const float2*>(p);
    v[0] = r.x, v[1] = r.y;
  } else {
    constexpr int E = vec_elems<T>();
#pragma unroll
    for (int i = 0; i < N / E; ++i) unpack16<T>(load16(p + i * E), &v[i * E]);
  }
}

// The same for rows of 16-byte pieces: a lane holds one piece, LPR lanes a row. A
// group of LPR lanes walks tokens, every GH-th head of each: the gains are loaded once,
// a token's angles once, and the rows of kRows heads before the first is used. In the
// half layout a lane also loads the piece its own is paired with (from the cache, as
// its neighbour just did), which costs no exchange between lanes. Bound by memory: 4 x
// 4001 tokens of 48 heads of 128 (348 MB read and written) 84 us, 4.1 TB/s, where a copy
// reaches 5.1; 32 tokens 5 us, one chain of position, angle and store.
template <typename T, int D, bool kHalfLayout>
__global__ __launch_bounds__(256) void rotate_rows_kernel(const RotateArgs a, int heads, int gh_log2, bool norm) {
  constexpr int VEC = vec_elems<T>(), LPR = D / VEC, kRows = 3;
  constexpr int ANGLES = kHalfLayout ? VEC : VEC / 2;
  const int group = int(threadIdx.x) / LPR, piece = int(threadIdx.x) % LPR;
  const int gh = 1 << gh_log2, per_block = (256 / LPR) >> gh_log2;
  const int d0 = piece * VEC;
  const bool turned = d0 < 2 * a.half;
  const bool second = kHalfLayout && d0 >= a.half;
  const int d1 = !kHalfLayout || !turned ? d0 : second ? d0 - a.half : d0 + a.half;  // the paired piece
  const int i0 = !turned ? 0 : kHalfLayout ? (second ? d1 : d0) : d0 / 2;            // the first angle

  const auto gains = [&](const void* gain, int d, float (&g)[VEC]) {
    if (!gain) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) g[e] = 1.f;
    } else if (a.gain_f32) {
      load_values<float, VEC>(static_cast<const float*>(gain) + d, g);
    } else {
      load_values<T, VEC>(static_cast<const T*>(gain) + d, g);
    }
  };
  float gq[VEC], gk[VEC], pq[VEC], pk[VEC];
  gains(a.q_gain, d0, gq);
  gains(a.k_gain, d0, gk);
  if constexpr (kHalfLayout) {
    gains(a.q_gain, d1, pq);
    gains(a.k_gain, d1, pk);
  }

  const unsigned tokens = unsigned(a.batch) * unsigned(a.tokens), stride = gridDim.x * unsigned(per_block);
  const int step = gh * int(gridDim.y), first = int(blockIdx.y) * gh;
  // What a token's rows depend on, loaded a token ahead.
  struct Token {
    int b, t, pos, start, count;
  };
  const auto look = [&](unsigned token) {
    const unsigned at = min(token, tokens - 1);  // the lanes of missing tokens repeat the last one
    Token k;
    k.b = int(at / unsigned(a.tokens));
    k.t = int(at - unsigned(k.b) * unsigned(a.tokens));
    k.pos = a.positions[at];
    k.start = a.start ? a.start[k.b] : 0;
    k.count = a.counts ? a.counts[k.b] : a.tokens;
    return k;
  };
  const unsigned lead = unsigned(group >> gh_log2);
  Token next = look(blockIdx.x * unsigned(per_block) + lead);
  for (unsigned tok0 = blockIdx.x * unsigned(per_block); tok0 < tokens; tok0 += stride) {
    const bool on = tok0 + lead < tokens;
    const int b = next.b, t = next.t, pos = next.pos;
    const bool used = t < next.count;
    const long slot = long(next.start) + t;
    const bool kv_store = on && (!a.start || (used && slot >= 0 && slot < a.slots));
    const bool known = pos >= 0 && pos < a.table;
    // Where head 0 of the launch's order (q, k, v) would be in each tensor.
    const int k0 = a.q_heads, v0 = a.q_heads + a.kv_heads;
    const auto from = [&](const void* p, int w, int h0) {
      return static_cast<const T*>(p) + b * a.st[w][0] + t * a.st[w][2] - h0 * a.st[w][1];
    };
    const auto into = [&](void* p, int w, int h0, long row) {
      return static_cast<T*>(p) + b * a.st[w][0] + row * a.st[w][2] - h0 * a.st[w][1];
    };
    const T *qi = from(a.q, 0, 0), *ki = from(a.k, 1, k0), *vi = from(a.v, 2, v0);
    T *qo = into(a.q_out, 3, 0, t), *ko = into(a.k_out, 4, k0, slot), *vo = into(a.v_out, 5, v0, slot);
    uint4 x[kRows], xp[kRows];
    const auto load = [&](int h0) {
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int h = min(h0 + r * step + (group & (gh - 1)), heads - 1);
        const T* p = h < k0 ? qi + h * a.st[0][1] : h < v0 ? ki + h * a.st[1][1] : vi + h * a.st[2][1];
        x[r] = load16(p + d0);
        if constexpr (kHalfLayout) xp[r] = load16(p + d1);
      }
    };
    // All of a token's loads before the first use: its rows, its angles, the next token's place.
    float c[ANGLES], sn[ANGLES];
    const long angle = long(known ? pos : 0) * a.half + i0;
    load_values<float, ANGLES>(a.cos + angle, c);
    load_values<float, ANGLES>(a.sin + angle, sn);
    load(first);
    next = look(tok0 + stride + lead);
#pragma unroll
    for (int i = 0; i < ANGLES; ++i) {
      c[i] = known ? c[i] : NAN;
      sn[i] = known ? sn[i] : NAN;
    }

    for (int h0 = first; h0 < heads; h0 += kRows * step) {  // uniform over the workgroup
      if (h0 > first) load(h0);
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const int h = h0 + r * step + (group & (gh - 1));
        const int w = h < k0 ? 0 : h < v0 ? 1 : 2;
        float v[VEC], o[VEC];
        unpack16<T>(x[r], v);
        if constexpr (kHalfLayout) unpack16<T>(xp[r], o);
        const bool is_q = w == 0;
        if (norm) {
          float sq = 0.f;
#pragma unroll
          for (int e = 0; e < VEC; ++e) sq = fmaf(v[e], v[e], sq);
          const float rms = 1.f / sqrtf(group_sum<LPR>(sq) / float(D) + a.eps);
          const float scale = (is_q ? a.q_gain : a.k_gain) ? rms : 1.f;
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            v[e] *= scale * (is_q ? gq[e] : gk[e]);
            if constexpr (kHalfLayout) o[e] *= scale * (is_q ? pq[e] : pk[e]);
          }
        }
        if constexpr (kHalfLayout) {
          if (turned) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = fmaf(second ? o[e] : -o[e], sn[e], v[e] * c[e]);
          }
        } else if (turned) {
#pragma unroll
          for (int e = 0; e < VEC; e += 2) {
            const float u = v[e], n = v[e + 1];
            v[e] = fmaf(-n, sn[e / 2], u * c[e / 2]);
            v[e + 1] = fmaf(u, sn[e / 2], n * c[e / 2]);
          }
        }
        uint4 y;
        if constexpr (std::is_same<T, float>::value)
          y = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        else
          y = make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
        if (w == 2) y = x[r];
        if (!used) y = make_uint4(0u, 0u, 0u, 0u);
        if (h < heads && (w == 0 ? on : kv_store)) {
          T* p = w == 0 ? qo + h * a.st[3][1] : w == 1 ? ko + h * a.st[4][1] : vo + h * a.st[5][1];
          *reinterpret_cast<uint4*>(p + d0) = y;
        }
      }
    }
  }
}

// Whether the rows come in 16-byte pieces, the paired ones, the angles and the gains too.
bool rotate_in_pieces(const RotateArgs& a, int es, bool half_layout) {
  const void* p[6] = {a.q, a.k, a.v, a.q_out, a.k_out, a.v_out};
  for (int i = 0; i < 6; ++i) {
    if (reinterpret_cast<uintptr_t>(p[i]) % 16) return false;
    for (int j = 0; j < 3; ++j)
      if (p[i] && a.st[i][j] * es % 16) return false;
  }
  const void* f[4] = {a.cos, a.sin, a.q_gain, a.k_gain};
  for (const void* g : f)
    if (reinterpret_cast<uintptr_t>(g) % 16) return false;
  return (half_layout ? a.half : 2 * a.half) * es % 16 == 0;
}

template <typename T, int D>
int launch_rotate_rows(const RotateArgs& a, int heads, bool half_layout, hipStream_t stream) {
  constexpr int kGroups = 256 / (D / vec_elems<T>());
  int gh_log2 = 0;
  while ((1 << gh_log2) < heads && (1 << gh_log2) < kGroups) ++gh_log2;
  const int per_block = kGroups >> gh_log2;
  const long blocks = (long(a.batch) * a.tokens + per_block - 1) / per_block;
  // Few tokens: their heads on several workgroups, until there are about two for each CU.
  const int rounds = (heads + (1 << gh_log2) - 1) >> gh_log2;
  const int share = int(std::max(1L, std::min(long(rounds), 512 / blocks)));
  // Many tokens: as many workgroups as the CUs hold at once, which walk them.
  const dim3 grid{unsigned(std::min(blocks, 1024L)), unsigned(share), 1u};
  const bool norm = a.q_gain || a.k_gain;
  if (half_layout)
    hipLaunchKernelGGL((rotate_rows_kernel<T, D, true>), grid, dim3(256), 0, stream, a, heads, gh_log2, norm);
  else
    hipLaunchKernelGGL((rotate_rows_kernel<T, D, false>), grid, dim3(256), 0, stream, a, heads, gh_log2, norm);
  return check_launch("rotate");
}

// ---- accepted path --------------------------------------------------------------

constexpr int kMaxPath = 128;

// Row len + j of a sequence's cache takes what row len + path[j] held, j < accepted.
// One workgroup has all the rows of a (sequence, KV head) in one tensor and reads
// every one before it writes any, so chains of rows that move are safe. Blocks in
// y: k, v, the slot values (which also lose the rejected drafts' weights); where k and
// v are one tensor its rows move once. Bound by
// latency: path, rows, stores (64 sequences, 9 MB: 6.5 us).
struct AcceptArgs {
  void *k, *v;
  float* weights;
  int32_t* positions;
  const int32_t *lengths, *path, *accepted;
  int32_t* new_lengths;
  long ks[3], vs[3];
  int kv_heads, cap, tokens, row_pieces;  // 16-byte pieces of a row
  int elem_bytes;
};
__global__ __launch_bounds__(256) void accept_kernel(const AcceptArgs a) {
  const int b = int(blockIdx.x) / a.kv_heads, hk = int(blockIdx.x) - b * a.kv_heads;
  const int len = a.lengths[b];
  const int count = len < 0 || len > a.cap ? 0 : min(min(max(a.accepted[b], 0), a.tokens), a.cap - len);
  const int32_t* path = a.path + long(b) * a.tokens;
  const auto source = [&](int j) {  // the slot that moves to len + j, -1 for none
    const int from = path[j];
    return from >= 0 && from < a.tokens && len + from < a.cap ? len + from : -1;
  };
  if (blockIdx.y == 2) {
    const int j = threadIdx.x;
    const long base = (long(b) * a.kv_heads + hk) * a.cap;
    if (hk == 0 && j == 0) a.new_lengths[b] = len + count;
    const int from = j < count ? source(j) : -1;
    float w = 0.f;
    int32_t p = 0;
    if (from >= 0 && a.weights) w = a.weights[base + from];
    if (from >= 0 && a.positions) p = a.positions[base + from];
    __syncthreads();
    // No sum with a length that may be any number: near 2^31 it would wrap into range.
    if (len < 0 || len >= a.cap || j >= a.tokens || j >= a.cap - len) return;
    if (a.weights && (from >= 0 || j >= count)) a.weights[base + len + j] = w;
    if (a.positions && from >= 0) a.positions[base + len + j] = p;
    return;
  }
  if (blockIdx.y == 1 && a.v == a.k) return;
  unsigned char* rows = static_cast<unsigned char*>(blockIdx.y ? a.v : a.k);
  const long stride = (blockIdx.y ? a.vs[2] : a.ks[2]) * a.elem_bytes;
  rows += (blockIdx.y ? b * a.vs[0] + hk * a.vs[1] : b * a.ks[0] + hk * a.ks[1]) * a.elem_bytes;
  constexpr int kPieces = kMaxPath * 32 / 256;  // of 16 bytes, per thread: 128 rows of 512 bytes
  uint4 held[kPieces];
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int at = int(threadIdx.x) + 256 * i, j = at / a.row_pieces;
    const int from = j < count ? source(j) : -1;
    if (from >= 0) held[i] = load16(rows + from * stride + 16 * (at - j * a.row_pieces));
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPieces; ++i) {
    const int at = int(threadIdx.x) + 256 * i, j = at / a.row_pieces;
    if (j < count && source(j) >= 0)
      *reinterpret_cast<uint4*>(rows + (len + j) * stride + 16 * (at - j * a.row_pieces)) = held[i];
  }
}

// ---- eviction -------------------------------------------------------------------

// Weights as unsigned numbers in the same order: -0 as 0, NaN below every number,
// and above them all the slots that stay because they are recent.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0u;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}

struct SelectArgs {
  const float* weights;
  const int32_t *lengths, *positions;
  int32_t *kept, *new_lengths;
  int kv_heads, cap, keep, recent;
};

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / kWave;
constexpr int kBins = 2048;          // 11 bits of a key
constexpr int kMoverList = 4096;     // movers placed at a time

// Sum over the workgroup of what the threads before this one have; *total: all of them.
__device__ __forceinline__ int block_exclusive(int v, int* scratch, int* total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int incl = v;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const int up = __shfl_up(incl, d);
    if (lane >= d) incl += up;
  }
  __syncthreads();  // scratch may still be read
  if (lane == kWave - 1) scratch[wave] = incl;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectWaves; ++w) {
    const int c = scratch[w];
    before += w < wave ? c : 0;
    all += c;
  }
  *total = all;
  return before + incl - v;
}

// kept[b, h, i]: the slot whose rows belong into slot i; one workgroup for a head. A
// radix selection, 11 bits of the keys at a time, finds the key of the last slot that
// stays; slots with that very key stay from the lowest on. (Weights share few
// exponents: with 8 bits at a time most of a wave counted in the same few bins, one
// lane after another.) The slots that stay are then counted by words of 64, the r-th
// of them from keep on goes through a list in LDS, and the r-th hole below keep takes
// it. Bound by its chain of some 20 barriers and by one CU's LDS: 32 heads of 20011
// slots 26 us (of 21 between the first and the last barrier the loads took 3, counting
// 11 and 11 bits 5 and 3, who stays 6, the list 4), 128 heads of 4160 slots with
// positions 18.6. kHeld: the keys stay in LDS; else they are formed again in every pass.
template <bool kHeld>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(const SelectArgs a) {
  extern __shared__ __align__(16) unsigned char dynamic[];  // [words] bits that stay, [words] counts before, [n] keys
  __shared__ int bins[kMoverList > kBins ? kMoverList : kBins];  // of the radix passes, then the movers
  __shared__ int scratch[kSelectWaves];
  __shared__ int found[3];  // the digit, how many of its keys are needed, how many there are
  const int b = int(blockIdx.x) / a.kv_heads, hk = int(blockIdx.x) - b * a.kv_heads;
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int n = min(max(a.lengths[b], 0), a.cap);
  int32_t* kept = a.kept + long(blockIdx.x) * a.keep;
  if (hk == 0 && tid == 0) a.new_lengths[b] = min(n, a.keep);
  if (n <= a.keep) {
    for (int i = tid; i < a.keep; i += kSelectThreads) kept[i] = i < n ? i : -1;
    return;
  }
  const float* weights = a.weights + long(blockIdx.x) * a.cap;
  const int32_t* positions = a.positions ? a.positions + long(blockIdx.x) * a.cap : nullptr;

  const int words = (n + 63) / 64;
  uint64_t* stays = reinterpret_cast<uint64_t*>(dynamic);
  int* before = reinterpret_cast<int*>(stays + words);
  uint32_t* keys = reinterpret_cast<uint32_t*>(before + words);

  // f(slot, values of kBatch rounds' slots): the loads of kBatch rounds go out together.
  constexpr int kBatch = 8;
  const auto positions_of = [&](int i0, int (&p)[kBatch]) {
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int i = min(i0 + u * kSelectThreads, n - 1);
      p[u] = positions ? positions[i] : i;
    }
  };
  int newest = n - 1;
  if (positions) {
    newest = INT_MIN;
    for (int i0 = tid; i0 < n; i0 += kBatch * kSelectThreads) {
      int p[kBatch];
      positions_of(i0, p);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) newest = max(newest, p[u]);
    }
    for (int m = 32; m >= 1; m >>= 1) newest = max(newest, lane_xor(newest, m));
    if (lane == 0) scratch[wave] = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectWaves; ++w) newest = max(newest, scratch[w]);
  }
  const long since = long(newest) - a.recent;
  const auto keys_of = [&](int i0, uint32_t (&k)[kBatch]) {
    int p[kBatch];
    positions_of(i0, p);
#pragma unroll
    for (int u = 0; u < kBatch; ++u) k[u] = weight_key(weights[min(i0 + u * kSelectThreads, n - 1)]);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (long(p[u]) > since) k[u] = 0xffffffffu;
  };
  if constexpr (kHeld) {
    for (int i0 = tid; i0 < n; i0 += kBatch * kSelectThreads) {
      uint32_t k[kBatch];
      keys_of(i0, k);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (i0 + u * kSelectThreads < n) keys[i0 + u * kSelectThreads] = k[u];  // its own thread's alone, in every pass
    }
  }
  // Round r of the workgroup: slots 1024 r .. 1024 r + 1023. f(round, slot, key), for all
  // threads of a round (slots from n on have some key).
  const int rounds = (n + kSelectThreads - 1) / kSelectThreads;
  const auto each = [&](auto&& f) {
    for (int r0 = 0; r0 < rounds; r0 += kBatch) {
      uint32_t k[kBatch];
      if constexpr (kHeld) {
#pragma unroll
        for (int u = 0; u < kBatch; ++u) k[u] = keys[min((r0 + u) * kSelectThreads + tid, n - 1)];
      } else {
        keys_of(r0 * kSelectThreads + tid, k);
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (r0 + u < rounds) f(r0 + u, (r0 + u) * kSelectThreads + tid, k[u]);
    }
  };

  uint32_t last = 0;  // the key of the last slot that stays, as far as it is known
  int need = a.keep, equal = n, shift = 32;
  while (shift > 0 && need < equal) {  // done as soon as every key that begins like this stays
    const int top = shift, width = shift > 10 ? 11 : 10;
    shift -= width;
    for (int i = tid; i < kBins; i += kSelectThreads) bins[i] = 0;
    __syncthreads();
    each([&](int, int i, uint32_t key) {
      if (i < n && (top == 32 || key >> top == last >> top)) atomicAdd(&bins[key >> shift & ((1u << width) - 1)], 1);
    });
    __syncthreads();
    // Thread t has bins 2 t' and 2 t' + 1 counted from the highest.
    const int high = (1 << width) - 1 - 2 * tid;
    const int c0 = high >= 0 ? bins[high] : 0, c1 = high >= 1 ? bins[high - 1] : 0;
    int all;
    const int above = block_exclusive(c0 + c1, scratch, &all);
    if (above < need && need <= above + c0 + c1) {
      const bool first = need <= above + c0;
      found[0] = first ? high : high - 1;
      found[1] = need - above - (first ? 0 : c0);
      found[2] = first ? c0 : c1;
    }
    __syncthreads();
    last |= uint32_t(found[0]) << shift;
    need = found[1];
    equal = found[2];
  }
  // Stays: a key above the last one's known bits, or with those bits and among the first `need` of them.
  const auto above_last = [&](uint32_t key) { return shift < 32 && key >> shift > last >> shift; };
  const auto like_last = [&](uint32_t key) { return shift == 32 || key >> shift == last >> shift; };
  const bool ties = need < equal;

  const int per = (words + kSelectThreads - 1) / kSelectThreads;
  const int first = min(tid * per, words), end = min(first + per, words);
  const auto scan = [&]() {  // counts of words to the counts before them
    __syncthreads();
    int sum = 0, total;
    for (int w = first; w < end; ++w) sum += before[w];
    int run = block_exclusive(sum, scratch, &total);
    for (int w = first; w < end; ++w) {
      const int c = before[w];
      before[w] = run;
      run += c;
    }
    __syncthreads();
  };
  if (ties) {
    each([&](int r, int i, uint32_t key) {
      const uint64_t bits = __ballot(i < n && like_last(key));
      if (lane == 0 && r * kSelectWaves + wave < words) before[r * kSelectWaves + wave] = __builtin_popcountll(bits);
    });
    scan();
  }
  each([&](int r, int i, uint32_t key) {
    const int w = r * kSelectWaves + wave;
    const bool like = i < n && like_last(key);
    bool in = like;
    if (ties) {
      const uint64_t bits = __ballot(like);
      in = like && before[min(w, words - 1)] + __builtin_popcountll(bits & ((1ull << lane) - 1)) < need;
    }
    const uint64_t bits = __ballot(in || (i < n && above_last(key)));
    if (lane == 0 && w < words) {
      stays[w] = bits;
      before[w] = __builtin_popcountll(bits);  // this wave alone reads and writes the word's entry
    }
  });
  scan();

  const int edge = a.keep / 64;
  const int below = before[edge] + __builtin_popcountll(stays[edge] & ((1ull << (a.keep % 64)) - 1));
  const int movers = a.keep - below;
  for (int base = 0; base == 0 || base < movers; base += kMoverList) {
    for (int r0 = a.keep / kSelectThreads; r0 < rounds; r0 += kBatch) {
      uint64_t bits[kBatch];
      int rank[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int w = min((r0 + u) * kSelectWaves + wave, words - 1);
        bits[u] = stays[w];
        rank[u] = before[w] + __builtin_popcountll(bits[u] & ((1ull << lane) - 1)) - below - base;
      }
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        const int i = (r0 + u) * kSelectThreads + tid;
        if (i >= a.keep && i < n && (bits[u] >> lane & 1) && rank[u] >= 0 && rank[u] < kMoverList) bins[rank[u]] = i;
      }
    }
    __syncthreads();
    for (int i = tid; i < a.keep; i += kSelectThreads) {
      const int w = i / 64;
      const int holes = i - before[w] - __builtin_popcountll(stays[w] & ((1ull << lane) - 1)) - base;  // below slot i
      if (stays[w] >> lane & 1) {
        if (base == 0) kept[i] = i;
      } else if (holes >= 0 && holes < kMoverList) {
        kept[i] = bins[holes];
      }
    }
    __syncthreads();
  }
}

// Slot i takes what slot kept[i] held where that lies at or above keep: what is read is
// never written, so nothing has to wait. A workgroup looks at 256 places, lists those
// that take another slot's rows, and moves the pieces of k and v of all of them
// together, kPieces loads of a thread in flight: few or many, the threads stay busy.
// Bound by memory where many move (3300 of 4096 rows of 32 heads, 100 MB, 22 us), by the
// launch and the list where few do (63 rows of 128 heads 8 us; without the list 12).
struct CompactArgs {
  void *k, *v;
  float* weights;
  int32_t* positions;
  const int32_t* kept;
  long ks[3], vs[3];
  int kv_heads, cap, keep, pieces_log2, elem_bytes, blocks;
};
__global__ __launch_bounds__(256) void compact_rows_kernel(const CompactArgs a) {
  constexpr int kPieces = 8;
  __shared__ int2 moves[256];
  __shared__ int counts[4];
  const int group = int(blockIdx.x) / a.blocks, part = int(blockIdx.x) - group * a.blocks;
  const int b = group / a.kv_heads, hk = group - b * a.kv_heads;
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int i = part * 256 + int(threadIdx.x);
  const int from = i < a.keep ? a.kept[long(group) * a.keep + i] : -1;
  const bool move = from >= a.keep && from < a.cap;
  const uint64_t bits = __ballot(move);
  if (lane == 0) counts[wave] = __builtin_popcountll(bits);
  __syncthreads();
  int before = 0, total = 0;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    before += w < wave ? counts[w] : 0;
    total += counts[w];
  }
  if (move) moves[before + __builtin_popcountll(bits & ((1ull << lane) - 1))] = make_int2(i, from);
  __syncthreads();

  unsigned char* k = static_cast<unsigned char*>(a.k) + (b * a.ks[0] + hk * a.ks[1]) * a.elem_bytes;
  unsigned char* v = static_cast<unsigned char*>(a.v) + (b * a.vs[0] + hk * a.vs[1]) * a.elem_bytes;
  const long kstride = a.ks[2] * a.elem_bytes, vstride = a.vs[2] * a.elem_bytes;
  const int items = total << (a.pieces_log2 + 1);  // (row, k or v, piece)
  for (int x0 = threadIdx.x; x0 < items; x0 += 256 * kPieces) {
    uint4 held[kPieces];
    unsigned char* to[kPieces];
#pragma unroll
    for (int e = 0; e < kPieces; ++e) {
      const int x = min(x0 + 256 * e, items - 1), y = x >> a.pieces_log2;
      const int2 m = moves[y >> 1];
      const int piece = x & ((1 << a.pieces_log2) - 1);
      unsigned char* rows = (y & 1 ? v : k) + 16 * piece;
      const long stride = y & 1 ? vstride : kstride;
      to[e] = rows + m.x * stride;
      held[e] = load16(rows + m.y * stride);
    }
#pragma unroll
    for (int e = 0; e < kPieces; ++e)
      if (x0 + 256 * e < items) *reinterpret_cast<uint4*>(to[e]) = held[e];
  }
}
// Weights and positions by slot; the weights of slots from keep on are cleared once all have moved.
__global__ __launch_bounds__(1024) void compact_values_kernel(const CompactArgs a) {
  const long base = long(blockIdx.x) * a.cap;
  for (int i = threadIdx.x; i < a.keep; i += 1024) {
    const int from = a.kept[long(blockIdx.x) * a.keep + i];
    if (from < a.keep || from >= a.cap) continue;
    if (a.weights) a.weights[base + i] = a.weights[base + from];
    if (a.positions) a.positions[base + i] = a.positions[base + from];
  }
  if (!a.weights) return;
  __syncthreads();
  for (int i = a.keep + int(threadIdx.x); i < a.cap; i += 1024) a.weights[base + i] = 0.f;
}

constexpr long kMostHeads = 1L << 22;  // a launch holds fewer than 2^32 threads

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int elem_size(int dtype) { return dtype == SFL_DTYPE_F32 ? 4 : dtype == SFL_DTYPE_BF16 || dtype == SFL_DTYPE_F16 ? 2 : 0; }

// Cache rows that are moved in 16-byte pieces.
int check_rows(const char* what, const void* k, const void* v, const long* strides, int batch, int kv_heads, int capacity,
               int head_dim, int dtype) {
  if (!k || !v || !strides) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (batch <= 0 || kv_heads <= 0 || capacity <= 0)
    return set_error(SFL_ERR_INVALID, "%s: batch, heads and capacity must be positive", what);
  if (long(batch) * kv_heads >= kMostHeads) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many KV heads", what);
  if (capacity > SFL_CACHE_MAX_SLOTS)  // slots are counted in 32 bits, up to a workgroup's step past the last
    return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d slots", what, SFL_CACHE_MAX_SLOTS);
  const int es = elem_size(dtype);
  if (!es) return set_error(SFL_ERR_UNSUPPORTED, "%s: dtype must be F32, BF16 or F16", what);
  if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported head dim %d", what, head_dim);
  if (!aligned16(k) || !aligned16(v)) return set_error(SFL_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  for (int i = 0; i < 6; ++i)
    if (strides[i] * es % 16) return set_error(SFL_ERR_INVALID, "%s: strides must be multiples of 16 bytes", what);
  return SFL_OK;
}

}  // namespace
}  // namespace sfl

extern "C" int sfl_rotate(const void* q, const void* k, const void* v, const int32_t* positions, const float* cos,
                          const float* sin, const void* q_gain, const void* k_gain, const int32_t* start,
                          const int32_t* counts, void* q_out, void* k_out, void* v_out, const long* strides, int batch,
                          int tokens, int q_heads, int kv_heads, int head_dim, int rotary_dim, int table, int slots,
                          int half_layout, int gain_dtype, float eps, int dtype, void* stream) {
  using namespace sfl;
  const char* what = "rotate";
  if (!q || !k || !positions || !cos || !sin || !q_out || !k_out || !strides || (v && !v_out))
    return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (batch <= 0 || tokens <= 0 || q_heads <= 0 || kv_heads <= 0 || table <= 0 || slots <= 0)
    return set_error(SFL_ERR_INVALID, "%s: batch, tokens, heads, table and slots must be positive", what);
  if (slots > SFL_CACHE_MAX_SLOTS)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d slots", what, SFL_CACHE_MAX_SLOTS);
  const int es = elem_size(dtype);
  if (!es) return set_error(SFL_ERR_UNSUPPORTED, "%s: dtype must be F32, BF16 or F16", what);
  if (head_dim != 16 && head_dim != 32 && head_dim != 64 && head_dim != 128)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: unsupported head dim %d", what, head_dim);
  if (rotary_dim < 2 || rotary_dim > head_dim || rotary_dim % 2)
    return set_error(SFL_ERR_INVALID, "%s: rotary dim must be even and in [2, head dim]", what);
  if (gain_dtype != dtype && gain_dtype != SFL_DTYPE_F32)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: gains must have the dtype of q or F32", what);
  if (!(eps >= 0.f) || !__builtin_isfinite(eps)) return set_error(SFL_ERR_INVALID, "%s: eps must be finite and not negative", what);
  if (v && k_out == v_out) return set_error(SFL_ERR_INVALID, "%s: k_out and v_out must not be the same memory", what);
  RotateArgs a{q, k, v, positions, cos, sin, q_gain, k_gain, start, counts, q_out, k_out, v_out};
  for (int i = 0; i < 18; ++i) a.st[i / 3][i % 3] = strides[i];
  a.batch = batch, a.tokens = tokens, a.q_heads = q_heads, a.kv_heads = kv_heads, a.half = rotary_dim / 2;
  a.table = table, a.slots = slots, a.gain_f32 = gain_dtype == SFL_DTYPE_F32, a.eps = eps;
  const int heads = q_heads + kv_heads * (v ? 2 : 1);
  const long rows = long(batch) * tokens * heads;
  if (rows >= (1L << 31)) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many rows", what);
  const auto run = [&](auto t) {
    using T = decltype(t);
    if (rotate_in_pieces(a, es, half_layout)) {
      const hipStream_t on = static_cast<hipStream_t>(stream);
      switch (head_dim) {
        case 16: return launch_rotate_rows<T, 16>(a, heads, half_layout, on);
        case 32: return launch_rotate_rows<T, 32>(a, heads, half_layout, on);
        case 64: return launch_rotate_rows<T, 64>(a, heads, half_layout, on);
        default: return launch_rotate_rows<T, 128>(a, heads, half_layout, on);
      }
    }
    const dim3 grid(unsigned(std::min((rows + 3) / 4, 1L << 20)));
    if (half_layout)
      hipLaunchKernelGGL((rotate_any_kernel<T, true>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a, head_dim, unsigned(rows), unsigned(heads));
    else
      hipLaunchKernelGGL((rotate_any_kernel<T, false>), grid, dim3(256), 0, static_cast<hipStream_t>(stream), a, head_dim, unsigned(rows), unsigned(heads));
    return check_launch(what);
  };
  if (dtype == SFL_DTYPE_F32) return run(float{});
  return dtype == SFL_DTYPE_BF16 ? run(bf16_t{}) : run(f16_t{});
}

extern "C" int sfl_accept_path(void* k, void* v, float* weights, int32_t* positions, const int32_t* lengths,
                               const int32_t* path, const int32_t* accepted, int32_t* new_lengths, const long* strides,
                               int batch, int kv_heads, int capacity, int tokens, int head_dim, int dtype, void* stream) {
  using namespace sfl;
  const char* what = "accept_path";
  if (int rc = check_rows(what, k, v, strides, batch, kv_heads, capacity, head_dim, dtype)) return rc;
  if (!lengths || !path || !accepted || !new_lengths) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (tokens < 1 || tokens > kMaxPath)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: between 1 and %d drafted tokens", what, kMaxPath);
  AcceptArgs a{k, v, weights, positions, lengths, path, accepted, new_lengths};
  for (int i = 0; i < 3; ++i) a.ks[i] = strides[i], a.vs[i] = strides[3 + i];
  a.kv_heads = kv_heads, a.cap = capacity, a.tokens = tokens, a.elem_bytes = elem_size(dtype);
  a.row_pieces = head_dim * a.elem_bytes / 16;
  hipLaunchKernelGGL(accept_kernel, dim3(unsigned(batch * kv_heads), 3), dim3(256), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(what);
}

extern "C" int sfl_select_slots(const float* weights, const int32_t* lengths, const int32_t* positions, int32_t* kept,
                                int32_t* new_lengths, int batch, int kv_heads, int capacity, int keep, int recent,
                                void* stream) {
  using namespace sfl;
  const char* what = "select_slots";
  if (!weights || !lengths || !kept || !new_lengths) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (batch <= 0 || kv_heads <= 0 || capacity <= 0)
    return set_error(SFL_ERR_INVALID, "%s: batch, heads and capacity must be positive", what);
  if (capacity > SFL_SELECT_MAX_SLOTS)
    return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d slots", what, SFL_SELECT_MAX_SLOTS);
  if (keep < 1 || keep > capacity || recent < 0 || recent > keep)
    return set_error(SFL_ERR_INVALID, "%s: keep must be in [1, capacity] and recent in [0, keep]", what);
  if (long(batch) * kv_heads >= kMostHeads) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many KV heads", what);
  const SelectArgs a{weights, lengths, positions, kept, new_lengths, kv_heads, capacity, keep, recent};
  // By the capacity, as the slots in use are known on the device only. Keys held / formed again,
  // us with 8 and 32 heads: 24573 slots 23.7, 26.8 / 29.7, 30.2; 5000 slots in use 12.7 either way.
  // Past that: 32768 slots 37, 131072 141 (32 heads 169), 262144 273.
  const bool held = capacity <= 24 * kSelectThreads;  // 96 KB of keys
  const unsigned bytes = unsigned((capacity + 63) / 64) * 12u + (held ? 4u * unsigned(capacity) : 0u);
  const auto kernel = held ? select_kernel<true> : select_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3(unsigned(batch * kv_heads)), dim3(kSelectThreads), bytes, static_cast<hipStream_t>(stream), a);
  return check_launch(what);
}

extern "C" int sfl_compact_slots(void* k, void* v, float* weights, int32_t* positions, const int32_t* kept,
                                 const long* strides, int batch, int kv_heads, int capacity, int keep, int head_dim,
                                 int dtype, void* stream) {
  using namespace sfl;
  const char* what = "compact_slots";
  if (int rc = check_rows(what, k, v, strides, batch, kv_heads, capacity, head_dim, dtype)) return rc;
  if (!kept) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (keep < 1 || keep > capacity) return set_error(SFL_ERR_INVALID, "%s: keep must be in [1, capacity]", what);
  CompactArgs a{k, v, weights, positions, kept};
  for (int i = 0; i < 3; ++i) a.ks[i] = strides[i], a.vs[i] = strides[3 + i];
  a.kv_heads = kv_heads, a.cap = capacity, a.keep = keep, a.elem_bytes = elem_size(dtype);
  while ((16 << a.pieces_log2) < head_dim * a.elem_bytes) ++a.pieces_log2;
  a.blocks = (keep + 255) / 256;
  if (long(batch) * kv_heads * a.blocks >= (1L << 24)) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many workgroups", what);
  hipLaunchKernelGGL(compact_rows_kernel, dim3(unsigned(batch * kv_heads * a.blocks)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), a);
  if (int rc = check_launch(what)) return rc;
  if (!weights && !positions) return SFL_OK;
  hipLaunchKernelGGL(compact_values_kernel, dim3(unsigned(batch * kv_heads)), dim3(1024), 0, static_cast<hipStream_t>(stream), a);
  return check_launch(what);
}
