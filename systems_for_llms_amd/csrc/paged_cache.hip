// A KV cache in pages of 8-bit codes: new tokens quantised into their sequences' pages,
// and the books of the pages (who holds which): forks, reservations with copies of
// shared pages, compaction.
//
// A page holds `page` tokens of every KV head of every layer. Its keys are e4m3 codes
// [page, D] with one scale for the head, its values codes [D, page] with another; a value is
// code * scale. Scales are powers of two: a floating-point code has the same relative
// precision under any scale, so nothing is lost, a page whose scale grows is re-scaled
// exactly (but for its smallest codes), and code * scale is exact in bf16.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "paged.hpp"

namespace sfl {
namespace {

// ---- append -----------------------------------------------------------------------

struct AppendArgs {
  const void *k, *v;
  uint8_t *k_codes, *v_codes;
  float *k_scale, *v_scale;
  const int32_t *tables, *lengths, *counts, *refs;
  long st[2][3];  // strides in elements (batch, head, token) of k and v
  int kv_heads, places, pages, page_log2, tokens, reach;  // reach: pages of a row that the tokens may touch
};

// The least e in [kLeastExponent, 120] with amax <= 448 * 2^e (448 = 1.75 * 2^8 is the
// largest code); amax is finite and below 2^127.
__device__ __forceinline__ int scale_exponent(uint32_t amax_bits) {
  const int e = int(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7fffffu) > 0x600000u);
  return max(e, kLeastExponent);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(uint32_t(max(e, -126) + 127) << 23); }

// Infinities, and what lies so near to them that its code's value could be one, have no code
// but NaN.
__device__ __forceinline__ bool has_code(float x) { return fabsf(x) < 0x1p127f; }

// One workgroup has one page of one row, one head, keys or values. A thread holds pieces of
// 16 bytes of four consecutive tokens: a piece of K is rounded along its dims, of V along
// the tokens, so both come out as whole words; V's words are turned through LDS into rows of
// the page's [D, page]. A row that starts inside a page first re-scales the tokens there
// when the scale grows. Bound by memory for prompts (4 x up to 4001 fp16 tokens of 8 heads of
// 128, 86 MB, 19 us, 4.5 TB/s, where a copy reaches 4.9), by its chain of loads for single
// tokens (32 of them 5.3 us).
template <typename T, int D>
__global__ __launch_bounds__(1024) void append_kernel(const AppendArgs a) {
  constexpr int VEC = vec_elems<T>(), PIECES = D / VEC;
  extern __shared__ uint32_t turned[];  // V: [D][page / 4 + 1] words of four tokens
  __shared__ float wave_amax[16];
  const int page = 1 << a.page_log2;
  unsigned u = blockIdx.x;
  const bool values = u & 1;
  u >>= 1;
  const unsigned row = u / unsigned(a.kv_heads), h = u - row * unsigned(a.kv_heads);
  const unsigned b = row / unsigned(a.reach), s = row - b * unsigned(a.reach);
  // What is the same for the workgroup comes by scalar loads, whose chain (length, page,
  // holders) then runs beside the tokens' own.
  typedef const __attribute__((address_space(4))) int32_t* Constant;
  typedef const __attribute__((address_space(4))) float* ConstantF;
  const int cap = a.places << a.page_log2;
  const int len = min(max(Constant(a.lengths)[b], 0), cap);
  const int count = min(a.counts ? min(max(Constant(a.counts)[b], 0), a.tokens) : a.tokens, cap - len);
  const int place = (len >> a.page_log2) + int(s);
  const int first = place << a.page_log2;  // the page's first slot
  const int lo = max(len - first, 0), hi = min(len + count - first, page);
  if (lo >= hi) return;
  const int at = Constant(a.tables)[long(b) * a.places + place];

  const int i = int(threadIdx.x) / PIECES, j = int(threadIdx.x) % PIECES;  // tokens 4 i .. 4 i + 3, piece j
  const long step = values ? a.st[1][2] : a.st[0][2];
  const T* x = static_cast<const T*>(values ? a.v : a.k) + b * (values ? a.st[1][0] : a.st[0][0]) +
               h * (values ? a.st[1][1] : a.st[0][1]) + VEC * j;
  const bool some = 4 * i + 3 >= lo && 4 * i < hi;
  uint4 raw[4] = {};
  if (some) {
#pragma unroll
    for (int c = 0; c < 4; ++c) raw[c] = load16(x + long(first + min(max(4 * i + c, lo), hi - 1) - len) * step);
  }
  if (at < 0 || at >= a.pages || Constant(a.refs)[at] != 1) return;
  const long block = long(at) * a.kv_heads + h;
  uint8_t* codes = (values ? a.v_codes : a.k_codes) + (block << a.page_log2) * D;
  float* scale = (values ? a.v_scale : a.k_scale) + block;
  const int held = int(__float_as_uint(ConstantF(scale)[0]) >> 23) - 127;

  float v[4][VEC] = {};
  float amax = 0.f;
  if (some) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      unpack16<T>(raw[c], v[c]);
      const bool on = 4 * i + c >= lo && 4 * i + c < hi;
#pragma unroll
      for (int f = 0; f < VEC; ++f) {
        v[c][f] = on ? v[c][f] : 0.f;
        amax = fmaxf(amax, has_code(v[c][f]) ? fabsf(v[c][f]) : 0.f);
      }
    }
  }
  amax = wave_max(amax);
  const int waves = (int(blockDim.x) + kWave - 1) / kWave;
  if (threadIdx.x % kWave == 0) wave_amax[threadIdx.x / kWave] = amax;
  __syncthreads();
  for (int w = 0; w < waves; ++w) amax = fmaxf(amax, wave_amax[w]);
  int e = scale_exponent(__float_as_uint(amax));
  if (lo > 0) {
    const int before = min(max(held, kLeastExponent), 120);
    if (before < e) {  // the committed tokens' codes under the new scale
      const float down = power_of_two(before - e);
      const int words = (page * D) / 4;
      uint32_t* w = reinterpret_cast<uint32_t*>(codes);
      for (int y = threadIdx.x; y < words; y += blockDim.x) {
        // A word is four dims of token 4 y / D, or four tokens from 4 y % page on of one dim.
        const int token = values ? (4 * y) & (page - 1) : 4 * y / D;
        if (token >= lo) continue;
        const uint32_t old = w[y];
        const auto p = __builtin_amdgcn_cvt_pk_f32_fp8(old, false), q = __builtin_amdgcn_cvt_pk_f32_fp8(old, true);
        uint32_t now = __builtin_amdgcn_cvt_pk_fp8_f32(p[0] * down, p[1] * down, 0, false);
        now = __builtin_amdgcn_cvt_pk_fp8_f32(q[0] * down, q[1] * down, now, true);
        const uint32_t mask = values && lo - token < 4 ? (1u << (8 * (lo - token))) - 1 : ~0u;
        w[y] = (now & mask) | (old & ~mask);
      }
    }
    e = max(e, before);
  }
  asm volatile("" : "+v"(e));  // from the held scale, which is read before it is replaced
  settle();  // the words above are written before the new tokens' bytes beside them
  if (threadIdx.x == 0) *scale = power_of_two(e);
  const float up = power_of_two(-e);
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int f = 0; f < VEC; ++f) v[c][f] = has_code(v[c][f]) ? v[c][f] * up : NAN;
  if (!values) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int slot = 4 * i + c;
      if (slot < lo || slot >= hi) continue;
#pragma unroll
      for (int f = 0; f < VEC; f += 4) {
        uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(v[c][f], v[c][f + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(v[c][f + 2], v[c][f + 3], w, true);
        *reinterpret_cast<uint32_t*>(codes + slot * D + VEC * j + f) = w;
      }
    }
    return;
  }
  const int quads = page / 4, stride = quads + 1;
  if (i < quads) {
#pragma unroll
    for (int f = 0; f < VEC; ++f) {
      uint32_t w = __builtin_amdgcn_cvt_pk_fp8_f32(v[0][f], v[1][f], 0, false);
      w = __builtin_amdgcn_cvt_pk_fp8_f32(v[2][f], v[3][f], w, true);
      turned[(VEC * j + f) * stride + i] = w;
    }
  }
  __syncthreads();
  // Pieces of 16 tokens of one dim: whole where the new tokens cover them, else byte by byte.
  const int pieces_log2 = a.page_log2 - 4;
  for (int y = threadIdx.x; y < D << pieces_log2; y += blockDim.x) {
    const int d = y >> pieces_log2, t0 = (y & ((1 << pieces_log2) - 1)) * 16;
    const uint32_t* w = turned + d * stride + t0 / 4;
    uint8_t* to = codes + (d << a.page_log2) + t0;
    if (lo <= t0 && t0 + 16 <= hi) {
      *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
      for (int t = max(lo - t0, 0); t < min(hi - t0, 16); ++t) to[t] = uint8_t(w[t / 4] >> (8 * (t % 4)));
    }
  }
}

// Bytes from the first to past the last one of a tensor.
struct Extent {
  uintptr_t from, to;
};
Extent extent_of(const void* p, long bytes, long before = 0) {
  const uintptr_t at = reinterpret_cast<uintptr_t>(p);
  return {at - uintptr_t(before), at + uintptr_t(bytes)};
}

// Whether what is read while pages are written lies apart from them.
bool apart(const AppendArgs& a, int batch, int dim, int element) {
  const int sizes[3] = {batch, a.kv_heads, a.tokens};
  Extent read[3] = {{}, {}, extent_of(a.counts, a.counts ? 4L * batch : 0)};
  for (int x = 0; x < 2; ++x) {
    long high = dim, low = 0;
    for (int i = 0; i < 3; ++i) {
      const long step = (sizes[i] - 1) * a.st[x][i];
      high += std::max(step, 0L), low -= std::min(step, 0L);
    }
    read[x] = extent_of(x ? a.v : a.k, high * element, low * element);
  }
  const long heads = long(a.pages) * a.kv_heads, pool = (heads << a.page_log2) * dim;
  for (const Extent& y : {extent_of(a.k_codes, pool), extent_of(a.v_codes, pool), extent_of(a.k_scale, 4 * heads),
                          extent_of(a.v_scale, 4 * heads)})
    for (const Extent& x : read)
      if (x.from < y.to && y.from < x.to) return false;
  return true;
}

template <typename T, int D>
int launch_append(const AppendArgs& a, int batch, hipStream_t stream) {
  const long blocks = 2L * batch * a.reach * a.kv_heads;
  const int page = 1 << a.page_log2;
  const int threads = std::max(kWave, page / 4 * (D / vec_elems<T>()));  // at most 1024
  if (blocks * threads >= (1L << 32)) return set_error(SFL_ERR_UNSUPPORTED, "page_append: too many workgroups");
  if (!apart(a, batch, D, sizeof(T)))
    return set_error(SFL_ERR_INVALID, "page_append: k, v and counts must not share memory with the layer's pages");
  hipLaunchKernelGGL((append_kernel<T, D>), dim3(unsigned(blocks)), dim3(unsigned(threads)), unsigned(D * (page + 4)), stream, a);
  return check_launch("page_append");
}

// ---- books ------------------------------------------------------------------------

constexpr int kBookThreads = 1024;
constexpr int kMostRows = kBookThreads;  // sequences: a thread each
constexpr int kForkWords = 16384;        // of LDS for the columns of a fork's workgroup

struct BookArgs {
  int32_t *tables, *lengths, *refs;
  int batch, places, pages, page_log2;
};

__device__ __forceinline__ bool is_page(const BookArgs& a, int x) { return x >= 0 && x < a.pages; }

// A row's parent: itself where the entry is no row and not -1.
__device__ __forceinline__ int parent_of(const int32_t* parents, int b, int batch) {
  const int p = parents[b];
  return p < -1 || p >= batch ? b : p;
}

// Every row takes the filled pages of its parent, all at once: a workgroup has some columns
// of the tables, of all rows, and holds them in LDS before it writes the first. `alone`: the
// grid is this workgroup, which then writes the lengths too (64 rows of 17 places 3.6 us;
// other grids have another launch for them).
__global__ __launch_bounds__(kBookThreads) void fork_kernel(const BookArgs a, const int32_t* parents, int columns, int alone) {
  extern __shared__ int32_t held[];  // [batch][columns], then [batch] filled pages
  int32_t* filled = held + a.batch * columns;
  const int c0 = int(blockIdx.x) * columns, n = min(columns, a.places - c0);
  const int cap = a.places << a.page_log2;
  for (int y = threadIdx.x; y < a.batch * n; y += kBookThreads) held[y] = a.tables[long(y / n) * a.places + c0 + y % n];
  int length = 0, parent = 0;  // of this thread's row
  if (int(threadIdx.x) < a.batch) {
    const int b = threadIdx.x;
    length = min(max(a.lengths[b], 0), cap);
    filled[b] = (length + (1 << a.page_log2) - 1) >> a.page_log2;
    parent = parent_of(parents, b, a.batch);
    if (alone && parent >= 0) length = min(max(a.lengths[parent], 0), cap);
    if (parent < 0) length = 0;
  }
  __syncthreads();
  if (alone && int(threadIdx.x) < a.batch && parent != int(threadIdx.x)) a.lengths[threadIdx.x] = length;
  for (int y = threadIdx.x; y < a.batch * n; y += kBookThreads) {
    const int b = y / n, c = y % n, p = parent_of(parents, b, a.batch);
    if (p == b) continue;
    const int was = held[y];
    int now = p >= 0 && c0 + c < filled[p] ? held[p * n + c] : -1;
    if (!is_page(a, now)) now = -1;
    if (now == was) continue;
    if (is_page(a, was)) atomicSub(&a.refs[was], 1);
    if (now >= 0) atomicAdd(&a.refs[now], 1);
    a.tables[long(b) * a.places + c0 + c] = now;
  }
}
__global__ __launch_bounds__(kBookThreads) void fork_lengths_kernel(const BookArgs a, const int32_t* parents) {
  const int b = threadIdx.x;
  int p = 0, length = 0;
  if (b < a.batch) {
    p = parent_of(parents, b, a.batch);
    if (p >= 0) length = min(max(a.lengths[p], 0), a.places << a.page_log2);
  }
  __syncthreads();
  if (b < a.batch && p != b) a.lengths[b] = length;
}

// The sum of `x` over the threads before this one, and over all (in `total`). Every thread
// of the workgroup calls it; `sums` is LDS of 16 words, free again after the next barrier.
__device__ __forceinline__ int scan(int x, int* sums, int& total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  int mine = x;
#pragma unroll
  for (int m = 1; m < kWave; m <<= 1) {
    const int other = __shfl_up(mine, m);
    mine += lane >= m ? other : 0;
  }
  __syncthreads();
  if (lane == kWave - 1) sums[wave] = mine;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kBookThreads / kWave; ++w) {
    before += w < wave ? sums[w] : 0;
    total += sums[w];
  }
  return before + mine - x;
}

__device__ __forceinline__ int32_t load_now(const int32_t* p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The lowest free pages from page `from` on, up to `most` of them into `found`; returns how
// many there are. Every thread of the workgroup calls it.
__device__ __forceinline__ int find_free(const BookArgs& a, int from, int most, int* found, int* sums) {
  constexpr int kScan = 8;  // pages looked at by a thread at a time
  int have = 0;
  for (int base = from & ~(kBookThreads * kScan - 1); have < most && base < a.pages; base += kBookThreads * kScan) {
    const int page = base + int(threadIdx.x) * kScan;
    int refs[kScan];
#pragma unroll
    for (int e = 0; e < kScan; ++e) refs[e] = a.refs[min(page + e, a.pages - 1)];
    unsigned free = 0;
#pragma unroll
    for (int e = 0; e < kScan; ++e) free |= unsigned(refs[e] == 0 && page + e >= from && page + e < a.pages) << e;
    int frees;
    int k = have + scan(__builtin_popcount(free), sums, frees);
#pragma unroll
    for (int e = 0; e < kScan; ++e)
      if (free >> e & 1) {
        if (k < most) found[k] = page + e;
        ++k;
      }
    have = min(have + frees, most);
  }
  __syncthreads();
  return have;
}

// One workgroup serves the rows one after another, place by place: a place that its row
// will write and that has no page, or one that others hold too, gets the lowest free page.
// 1024 places at a time are looked at together. What the rows before it in the same round
// do to a place's page is found from the pages they hold: of r holders, the first r - 1 that
// write it leave it, and the last then has it alone. (Those of earlier rounds have left, or
// there are no free pages any more.) Bound by its chain of loads and barriers: 64 rows, 16 of
// them with 6 new places and 16 that share a page, of 1600 pages 11 to 12 us.
__global__ __launch_bounds__(kBookThreads) void reserve_kernel(const BookArgs a, const int32_t* counts, int32_t* granted,
                                                               int2* copies, int* copied) {
  __shared__ int sums[kBookThreads / kWave];
  __shared__ int lens[kMostRows], ends[kMostRows], starts[kMostRows + 1], failed[kMostRows];
  __shared__ int rank_of[kBookThreads], found[kBookThreads];
  __shared__ __align__(16) int shared_page[kBookThreads];  // of places whose page others hold too, else -1
  __shared__ int made, position;
  const int tid = threadIdx.x, cap = a.places << a.page_log2;
  int wanted = 0;  // places of this thread's row
  if (tid < a.batch) {
    const int len = min(max(a.lengths[tid], 0), cap);
    // No row gets more places than there are pages: one more shows what fails.
    const long most = ((long(len) >> a.page_log2) + a.pages + 1) << a.page_log2;
    const int end = int(min(long(len) + min(max(counts[tid], 0), cap - len), most));
    lens[tid] = len, ends[tid] = end, failed[tid] = a.places;
    wanted = end > len ? ((end - 1) >> a.page_log2) - (len >> a.page_log2) + 1 : 0;
  }
  int items;
  const int start = scan(wanted, sums, items);
  if (tid <= a.batch) starts[tid] = start;  // [batch] is the total, as wanted is 0 there
  if (a.batch == kMostRows && tid == 0) starts[kMostRows] = items;
  if (tid == 0) made = 0, position = 0;
  __syncthreads();
  for (int base = 0; base < items; base += kBookThreads) {
    const int item = base + tid;
    int b = 0, place = 0, held = -1, holders = 0;
    if (item < items) {
      int hi = a.batch - 1;  // the last row whose places start at or before the item
      while (b < hi) {
        const int mid = (b + hi + 1) / 2;
        if (starts[mid] <= item) b = mid; else hi = mid - 1;
      }
      place = (lens[b] >> a.page_log2) + item - starts[b];
      held = load_now(&a.tables[long(b) * a.places + place]);
      if (!is_page(a, held)) held = -1;
      if (held >= 0) holders = load_now(&a.refs[held]);
    }
    shared_page[tid] = holders > 1 ? held : -1;
    __syncthreads();
    bool lacks = item < items && held < 0, stays = false;
    int last = -1;  // the place before it with the same page
    if (holders > 1) {
      int before = 0;
      for (int j = 0; j < tid; j += 4) {
        const int4 x = *reinterpret_cast<const int4*>(shared_page + j);
        const int pages[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (pages[e] == held && j + e < tid) ++before, last = j + e;
      }
      lacks = before < holders - 1;
      stays = !lacks;
    }
    int lacking;
    const int rank = scan(lacks, sums, lacking);
    rank_of[tid] = rank;
    const int have = find_free(a, position, lacking, found, sums);
    const bool got = lacks && rank < have;
    if (got) {
      const int now = found[rank];
      a.tables[long(b) * a.places + place] = now;
      atomicExch(&a.refs[now], 1);
      if (held >= 0) {
        atomicSub(&a.refs[held], 1);
        if (place << a.page_log2 < lens[b]) copies[atomicAdd(&made, 1)] = make_int2(held, now);
      }
    }
    // A row has a shared page alone only once the one before it has left.
    if ((lacks && !got) || (stays && last >= 0 && rank_of[last] >= have)) atomicMin(&failed[b], place);
    __syncthreads();
    if (tid == 0) position = have < lacking ? a.pages : have > 0 ? found[have - 1] + 1 : position;
    settle();
  }
  if (tid < a.batch) {
    const long reach = (long(failed[tid]) << a.page_log2) - lens[tid];
    granted[tid] = int(min(long(ends[tid] - lens[tid]), max(reach, 0L)));
  }
  if (tid == 0) *copied = made;
}

// Which pages move where: the k-th page in use past the first `used` to the k-th free one
// among them. 2048 pages 6.5 us, a chain of loads and barriers.
__global__ __launch_bounds__(kBookThreads) void compact_plan_kernel(const BookArgs a, int2* moves, int32_t* target, int* moved,
                                                                    int32_t* used) {
  constexpr int kScan = 8;
  __shared__ int sums[kBookThreads / kWave];
  const int tid = threadIdx.x;
  int live = 0;
  for (int p = tid; p < a.pages; p += kBookThreads) live += a.refs[p] > 0;
  int total;
  scan(live, sums, total);
  int movers = 0, holes = 0;
  for (int base = 0; base < a.pages; base += kBookThreads * kScan) {
    const int page0 = base + tid * kScan;
    unsigned move = 0, hole = 0;
#pragma unroll
    for (int e = 0; e < kScan; ++e) {
      const int p = page0 + e;
      if (p >= a.pages) continue;
      const bool in_use = a.refs[p] > 0;
      if (in_use && p >= total) move |= 1u << e;
      if (!in_use && p < total) hole |= 1u << e;
      if (p >= total) target[p] = -1;
    }
    // Both counts in one scan: at most 8192 of each in a round.
    int sum;
    const int before = scan(__builtin_popcount(move) << 16 | __builtin_popcount(hole), sums, sum);
    int m = movers + (before >> 16), h = holes + (before & 0xffff);
#pragma unroll
    for (int e = 0; e < kScan; ++e) {
      if (move >> e & 1) moves[m++].x = page0 + e;
      if (hole >> e & 1) moves[h++].y = page0 + e;
    }
    movers += sum >> 16, holes += sum & 0xffff;
  }
  settle();
  for (int k = tid; k < movers; k += kBookThreads) target[load_now(&moves[k].x)] = load_now(&moves[k].y);
  if (tid == 0) *moved = movers, *used = total;
}

struct CopyArgs {
  uint8_t *k, *v;
  float *k_scale, *v_scale;
  const int2* moves;
  const int* moved;
  long page_bytes, pool_bytes;  // of one page's keys (and of its values) in one layer; of a layer's pool
  int layers, kv_heads, pages, parts;
};

constexpr int kCopyPieces = 4, kCopyPart = 256 * 16 * kCopyPieces;

// Pages copied, all layers: workgroups walk (move, layer, keys or values, 16 KB of it), as a
// plan made on the device is not known to the launch. Bound by memory: 491 pages of 8 layers,
// 1.03 GB read and written, 209 us (4.9 TB/s); 94 MB 20 (4.7).
__device__ __forceinline__ void copy_pages(const CopyArgs& c) {
  const long items = long(*c.moved) * c.layers * 2 * c.parts;
  for (long y = blockIdx.x; y < items; y += gridDim.x) {
    long x = y;
    const int part = int(x % c.parts);
    x /= c.parts;
    const bool values = x & 1;
    x >>= 1;
    const int layer = int(x % c.layers);
    const int2 m = c.moves[x / c.layers];
    uint8_t* pool = (values ? c.v : c.k) + layer * c.pool_bytes;
    const uint8_t* from = pool + m.x * c.page_bytes;
    uint8_t* to = pool + m.y * c.page_bytes;
    uint4 held[kCopyPieces];
    const long at = long(part) * kCopyPart + threadIdx.x * 16;
#pragma unroll
    for (int e = 0; e < kCopyPieces; ++e)
      if (at + e * 4096 < c.page_bytes) held[e] = load16(from + at + e * 4096);
#pragma unroll
    for (int e = 0; e < kCopyPieces; ++e)
      if (at + e * 4096 < c.page_bytes) *reinterpret_cast<uint4*>(to + at + e * 4096) = held[e];
    if (part == 0) {
      float* scales = (values ? c.v_scale : c.k_scale) + long(layer) * c.pages * c.kv_heads;
      for (int h = threadIdx.x; h < c.kv_heads; h += 256) scales[long(m.y) * c.kv_heads + h] = scales[long(m.x) * c.kv_heads + h];
    }
  }
}

__global__ __launch_bounds__(256) void copy_kernel(const CopyArgs c) { copy_pages(c); }

__global__ __launch_bounds__(256) void compact_kernel(const CopyArgs c, const BookArgs a, const int32_t* target,
                                                      const int32_t* used) {
  copy_pages(c);
  const long first = long(blockIdx.x) * 256 + threadIdx.x, step = long(gridDim.x) * 256;
  const int total = *used;
  for (long y = first; y < long(a.batch) * a.places; y += step) {
    const int x = a.tables[y];
    if (x >= total && x < a.pages) a.tables[y] = target[x];
  }
  for (long k = first; k < *c.moved; k += step) {
    const int2 m = c.moves[k];
    a.refs[m.y] = a.refs[m.x];
    a.refs[m.x] = 0;
  }
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int fill_books(BookArgs& a, const char* what, int32_t* tables, int32_t* lengths, int32_t* refs, int batch, int places,
               int pages, int page_size) {
  if (!tables || !refs) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (int rc = check_paged(what, batch, places, pages, page_size)) return rc;
  if (batch > kMostRows) return set_error(SFL_ERR_UNSUPPORTED, "%s: at most %d sequences", what, kMostRows);
  a = BookArgs{tables, lengths, refs, batch, places, pages, log2_of(page_size)};
  return SFL_OK;
}

int fill_copy(CopyArgs& c, const char* what, void* k, void* v, float* k_scale, float* v_scale, int layers, int pages,
              int kv_heads, int page_size, int head_dim) {
  if (!k || !v || !k_scale || !v_scale) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (!aligned16(k) || !aligned16(v)) return set_error(SFL_ERR_INVALID, "%s: pools must be 16-byte aligned", what);
  if (layers <= 0 || kv_heads <= 0) return set_error(SFL_ERR_INVALID, "%s: layers and heads must be positive", what);
  if (int rc = check_head_dim(what, head_dim)) return rc;
  c = CopyArgs{static_cast<uint8_t*>(k), static_cast<uint8_t*>(v), k_scale, v_scale};
  c.page_bytes = long(kv_heads) * page_size * head_dim, c.pool_bytes = c.page_bytes * pages;
  c.layers = layers, c.kv_heads = kv_heads, c.pages = pages;
  c.parts = int((c.page_bytes + kCopyPart - 1) / kCopyPart);
  return SFL_OK;
}

constexpr long kCopyGrid = 2048;  // about eight workgroups to a CU

}  // namespace
}  // namespace sfl

extern "C" int sfl_page_append(const void* k, const void* v, void* k_codes, void* v_codes, float* k_scale, float* v_scale,
                               const int32_t* tables, const int32_t* lengths, const int32_t* counts, const int32_t* refs,
                               const long* strides, int batch, int kv_heads, int tokens, int places, int pages,
                               int page_size, int head_dim, int dtype, void* stream) {
  using namespace sfl;
  const char* what = "page_append";
  if (!k || !v || !k_codes || !v_codes || !k_scale || !v_scale || !tables || !lengths || !refs || !strides)
    return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  if (kv_heads <= 0 || tokens <= 0) return set_error(SFL_ERR_INVALID, "%s: heads and tokens must be positive", what);
  if (int rc = check_paged(what, batch, places, pages, page_size)) return rc;
  if (int rc = check_head_dim(what, head_dim)) return rc;
  const int es = dtype == SFL_DTYPE_F32 ? 4 : dtype == SFL_DTYPE_BF16 || dtype == SFL_DTYPE_F16 ? 2 : 0;
  if (!es) return set_error(SFL_ERR_UNSUPPORTED, "%s: dtype must be F32, BF16 or F16", what);
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_codes) || !aligned16(v_codes))
    return set_error(SFL_ERR_INVALID, "%s: tensors must be 16-byte aligned", what);
  for (int i = 0; i < 6; ++i)
    if (strides[i] * es % 16) return set_error(SFL_ERR_INVALID, "%s: strides must be multiples of 16 bytes", what);
  AppendArgs a{k, v, static_cast<uint8_t*>(k_codes), static_cast<uint8_t*>(v_codes), k_scale, v_scale, tables, lengths, counts, refs};
  for (int i = 0; i < 6; ++i) a.st[i / 3][i % 3] = strides[i];
  a.kv_heads = kv_heads, a.places = places, a.pages = pages, a.page_log2 = log2_of(page_size), a.tokens = tokens;
  a.reach = std::min(places, (tokens - 1) / page_size + (tokens > 1 ? 2 : 1));
  return paged_types(dtype, head_dim, [&](auto t, auto d) {
    return launch_append<decltype(t), decltype(d)::value>(a, batch, static_cast<hipStream_t>(stream));
  });
}

extern "C" int sfl_page_fork(int32_t* tables, int32_t* lengths, int32_t* refs, const int32_t* parents, int batch,
                             int places, int pages, int page_size, void* stream) {
  using namespace sfl;
  const char* what = "page_fork";
  BookArgs a;
  if (int rc = fill_books(a, what, tables, lengths, refs, batch, places, pages, page_size)) return rc;
  if (!lengths || !parents) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  const int columns = std::min(places, std::max(1, (kForkWords - batch) / batch));
  const int blocks = (places + columns - 1) / columns;
  hipLaunchKernelGGL(fork_kernel, dim3(unsigned(blocks)), dim3(kBookThreads), unsigned(4 * batch * (columns + 1)), on, a, parents,
                     columns, int(blocks == 1));
  if (int rc = check_launch(what)) return rc;
  if (blocks == 1) return SFL_OK;
  hipLaunchKernelGGL(fork_lengths_kernel, dim3(1), dim3(kBookThreads), 0, on, a, parents);
  return check_launch(what);
}

extern "C" int sfl_page_reserve(void* k, void* v, float* k_scale, float* v_scale, int32_t* tables, const int32_t* lengths,
                                int32_t* refs, const int32_t* counts, int32_t* granted, int32_t* scratch, int batch,
                                int places, int pages, int layers, int kv_heads, int page_size, int head_dim,
                                void* stream) {
  using namespace sfl;
  const char* what = "page_reserve";
  BookArgs a;
  CopyArgs c;
  if (int rc = fill_books(a, what, tables, const_cast<int32_t*>(lengths), refs, batch, places, pages, page_size)) return rc;
  if (int rc = fill_copy(c, what, k, v, k_scale, v_scale, layers, pages, kv_heads, page_size, head_dim)) return rc;
  if (!lengths || !counts || !granted || !scratch) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  if (long(batch) * std::min(places, pages + 1) >= (1L << 31)) return set_error(SFL_ERR_UNSUPPORTED, "%s: too many places", what);
  int2* copies = reinterpret_cast<int2*>(scratch + 2);
  hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kBookThreads), 0, on, a, counts, granted, copies, scratch);
  if (int rc = check_launch(what)) return rc;
  c.moves = copies, c.moved = scratch;
  const long most = long(batch) * layers * 2 * c.parts;
  hipLaunchKernelGGL(copy_kernel, dim3(unsigned(std::min(most, kCopyGrid))), dim3(256), 0, on, c);
  return check_launch(what);
}

extern "C" int sfl_page_compact(void* k, void* v, float* k_scale, float* v_scale, int32_t* tables, int32_t* refs,
                                int32_t* used, int32_t* scratch, int batch, int places, int pages, int layers, int kv_heads,
                                int page_size, int head_dim, void* stream) {
  using namespace sfl;
  const char* what = "page_compact";
  BookArgs a;
  CopyArgs c;
  if (int rc = fill_books(a, what, tables, nullptr, refs, batch, places, pages, page_size)) return rc;
  if (int rc = fill_copy(c, what, k, v, k_scale, v_scale, layers, pages, kv_heads, page_size, head_dim)) return rc;
  if (!used || !scratch) return set_error(SFL_ERR_INVALID, "%s: null pointer argument", what);
  const hipStream_t on = static_cast<hipStream_t>(stream);
  int2* moves = reinterpret_cast<int2*>(scratch + 2);  // pages / 2 + 1 of them
  int32_t* target = scratch + 4 + pages;
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kBookThreads), 0, on, a, moves, target, scratch, used);
  if (int rc = check_launch(what)) return rc;
  c.moves = moves, c.moved = scratch;
  const long most = std::max(long(pages) / 2 * layers * 2 * c.parts, 1L);
  hipLaunchKernelGGL(compact_kernel, dim3(unsigned(std::min(most, kCopyGrid))), dim3(256), 0, on, c, a, target, used);
  return check_launch(what);
}
