// dgi/csrc/longctx/select_pages.hip — which pages of its context a row's group of heads is to read.
//
// With P_d = sum over the group of max(q_d, 0) and N_d = sum of min(q_d, 0), a page scores P . hi + N . lo: the sum over the group of
// the largest q . k that a key within the page's bounds can have.  Kept are the first and last pages (as many as the caller says) and the
// best of the others, ties to the lowest.
//
// Scores are summed in 64 bits: which page is kept is a whole number, and may not depend on the order in which a sum was taken.
// They go as integers of the same order into a workspace [T, n_kv, pages]; a second launch chooses by digits of these integers
// taken from the top.
//
// Decode rows each have bounds of their own, which is what bounds them (a lane multiplies what it loads).  Rows of a prompt share
// their sequence's: 16 of them are the rows of matrix instructions in 64 bits, whose rate is the bound.
#include "../common.h"

using namespace dgi;

namespace {

typedef unsigned long long u64;
typedef double d4 __attribute__((ext_vector_type(4)));

// Integers of the order of the doubles; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ u64 key_of(double x) {
  if (x != x) x = -__builtin_inf();
  const u64 b = __double_as_longlong(x + 0.0);
  return b >> 63 ? ~b : b | (1ull << 63);
}

struct Args {
  const uint16_t* q;
  long long q_stride;
  const uint16_t* bounds;
  const int* tables;
  int table_stride, table_cols, n_seqs, num_blocks;
  const int* ctx;
  const int* row_seq;
  int T, nh, nkv, page, count, first, recent;
  u64* keys;
  int key_stride;
  int* out;
  int chunk;      // pages of a workgroup
};

__device__ __forceinline__ int pages_of(const Args& a, int t) {
  const int c = a.ctx[t];
  return c <= 0 ? 0 : min((c - 1) / a.page + 1, a.table_cols);
}

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kRows = 16, kRuns = 4;      // rows of an aligned group; it goes together if they are of so many sequences at most

__device__ __forceinline__ bool together(unsigned begins) { return __popc(begins & ((1u << kRows) - 1)) <= kRuns; }

// The aligned group of row t: bit i says that row i begins another sequence than the row before it (or is behind the last row).
__device__ __forceinline__ unsigned begins_of(const Args& a, int t, int lane) {
  const int row = t / kRows * kRows + lane;
  const int seq = lane < kRows && row < a.T ? a.row_seq[row] : -1;
  const int prev = __shfl_up(seq, 1, 64);
  return (unsigned)__ballot(lane < kRows && (lane == 0 || row == a.T || (row < a.T && seq != prev))) | 1u << kRows;
}

// up += max(q, 0), down += min(q, 0) of eight channels over a group's G heads, HD apart; four of them under way at a time.
template <int HD>
__device__ __forceinline__ void add_heads(double* up, double* down, const uint16_t* q, int G) {
  for (int g0 = 0; g0 < G; g0 += 4) {
    u32x4 v[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) v[g] = *reinterpret_cast<const u32x4*>(q + min(g0 + g, G - 1) * HD);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      float x[8];
      unpack8(v[g], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (g0 + g >= G) x[j] = 0.f;
        up[j] += x[j] < 0.f ? 0.f : x[j];        // no number stays none
        down[j] += x[j] > 0.f ? 0.f : x[j];
      }
    }
  }
}

// Row by row.  Four 16-byte chunks of a page's [lo | hi] a lane, HD / 16 lanes a page; the next pages' bounds are under way
// while these are multiplied.  GROUPS: not the rows that page_scores_tiles_kernel takes.
template <int HD, bool GROUPS>
__global__ __launch_bounds__(kThreads) void page_scores_kernel(Args a) {
  constexpr int LP = HD / 16, PW = 64 / LP, STEP = kWaves * PW;      // lanes a page, pages a wave and a workgroup at a time
  const int t = blockIdx.x / a.nkv, h = blockIdx.x - t * a.nkv;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane % LP, p0 = lane / LP;
  if (GROUPS && together(begins_of(a, t, lane))) return;
  const int n = pages_of(a, t);
  const int begin = a.first + blockIdx.y * a.chunk, end = min(begin + a.chunk, n - a.recent);
  if (n <= a.count || begin >= end) return;
  const int G = a.nh / a.nkv;
  __shared__ double wgt_s[2 * HD];      // of lo, of hi
  if (threadIdx.x < HD / 8) {
    double up[8] = {}, down[8] = {};
    add_heads<HD>(up, down, a.q + t * a.q_stride + h * G * HD + threadIdx.x * 8, G);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wgt_s[threadIdx.x * 8 + j] = down[j];
      wgt_s[HD + threadIdx.x * 8 + j] = up[j];
    }
  }
  const int seq = a.row_seq ? a.row_seq[t] : t;
  const bool known = seq >= 0 && seq < a.n_seqs;
  const int* table = a.tables + (size_t)(known ? seq : 0) * a.table_stride;
  u64* keys = a.keys + ((size_t)t * a.nkv + h) * a.key_stride;
  auto id_of = [&](int base) {
    const int p = base + p0, id = known && p < end ? table[p] : -1;
    return id >= 0 && id < a.num_blocks ? id : -1;
  };
  u32x4 v[2][4];
  auto load = [&](u32x4* to, int id) {
    const uint16_t* bp = a.bounds + ((size_t)max(id, 0) * a.nkv + h) * 2 * HD + l * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = *reinterpret_cast<const u32x4*>(bp + LP * i * 8);
  };
  int base = begin + w * PW, id = id_of(base), id_next = id_of(base + STEP);
  load(v[0], id);
  __syncthreads();
  // chunk l + LP i: the lo half for i < 2, the hi half behind it
  double wgt[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) wgt[i][j] = wgt_s[(l + LP * i) * 8 + j];
  auto score = [&](const u32x4* x4, int base, int id) {
    double sum[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float x[8];
      unpack8(x4[i], x);
#pragma unroll
      for (int j = 0; j < 8; ++j) sum[i] = fma(wgt[i][j], (double)x[j], sum[i]);
    }
    double s = (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
    for (int o = 1; o < LP; o <<= 1) s += __shfl_xor(s, o, 64);
    if (l == 0 && base + p0 < end) keys[base + p0] = key_of(id >= 0 ? s : -__builtin_inf());
  };
  for (; base < end; base += 2 * STEP) {
    int id2 = id_of(base + 2 * STEP);
    load(v[1], id_next);
    score(v[0], base, id);
    if (base + STEP >= end) break;
    id = id2;
    load(v[0], id);
    id2 = id_of(base + 3 * STEP);
    score(v[1], base + STEP, id_next);
    id_next = id2;
  }
}

// Rows that go together: 16 x 16 (rows, pages) at a time, four channels an instruction.  A lane has row lane % 16's weights and page
// lane % 16's bounds of the chunks 4 j + lane / 16 of [lo | hi], eight values each.
template <int HD>
__global__ __launch_bounds__(kThreads, 2) void page_scores_tiles_kernel(Args a) {
  constexpr int CH = HD / 4, J = CH / 4;      // chunks of a row of bounds, of them a lane's
  constexpr int LD = 2 * HD + 2;              // doubles between rows in LDS: reads of 16 rows hit other banks
  __shared__ __attribute__((aligned(16))) double wgt_s[kRows * LD];
  const int group = blockIdx.x / a.nkv, h = blockIdx.x - group * a.nkv, t0 = group * kRows;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n16 = lane & 15, kq = lane >> 4;
  const unsigned begins = begins_of(a, t0, lane);
  if (!together(begins)) return;
  const int G = a.nh / a.nkv;
  // the workgroup's run: rows r0 .. r1 of the group
  const int chunks = gridDim.y / kRuns, run = blockIdx.y / chunks;
  unsigned rest = begins;
  for (int i = 0; i < run; ++i) rest &= rest - 1;
  const int r0 = __ffs(rest) - 1, r1 = __ffs(begins >> (r0 + 1)) + r0;
  if (r0 >= kRows || t0 + r0 >= a.T) return;
  // weights of the group's rows
  for (int i = tid; i < kRows * (HD / 8); i += kThreads) {
    const int row = i / (HD / 8), c = i - row * (HD / 8), t = min(t0 + row, a.T - 1);
    double up[8] = {}, down[8] = {};
    add_heads<HD>(up, down, a.q + t * a.q_stride + h * G * HD + c * 8, G);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      wgt_s[row * LD + c * 8 + j] = down[j];
      wgt_s[row * LD + HD + c * 8 + j] = up[j];
    }
  }
  int stop = 0;      // pages that row n16 needs scores of end here
  if (n16 >= r0 && n16 < r1) {
    const int n = pages_of(a, t0 + n16);
    stop = n > a.count ? n - a.recent : 0;
  }
  int last = stop;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
  const int begin = a.first + (blockIdx.y - run * chunks) * a.chunk, end = __builtin_amdgcn_readfirstlane(min(begin + a.chunk, last));
  if (begin >= end) return;
  const int seq = a.row_seq[t0 + r0];
  const bool known = seq >= 0 && seq < a.n_seqs;
  const int* table = a.tables + (size_t)(known ? seq : 0) * a.table_stride;
  auto id_of = [&](int base) {
    const int p = base + n16, id = known && p < end ? table[p] : -1;
    return id >= 0 && id < a.num_blocks ? id : -1;
  };
  u32x4 v[J];
  auto load = [&](int id) {
    const uint16_t* bp = a.bounds + ((size_t)max(id, 0) * a.nkv + h) * 2 * HD + kq * 8;
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = *reinterpret_cast<const u32x4*>(bp + j * 32);
  };
  constexpr int STEP = kWaves * 16;
  int base = begin + 16 * w, id = id_of(base), id_next = id_of(base + STEP);
  load(id);
  __syncthreads();
  double wgt[J][8];
#pragma unroll
  for (int j = 0; j < J; ++j)
#pragma unroll
    for (int s = 0; s < 8; ++s) wgt[j][s] = wgt_s[n16 * LD + (4 * j + kq) * 8 + s];
  for (; base < end; base += STEP) {
    d4 acc[2] = {};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      float x[8];
      unpack8(v[j], x);
#pragma unroll
      for (int s = 0; s < 8; ++s) acc[s & 1] = __builtin_amdgcn_mfma_f64_16x16x4f64(wgt[j][s], (double)x[s], acc[s & 1], 0, 0, 0);
    }
    const int now = id;
    id = id_next;
    load(id);
    id_next = id_of(base + 2 * STEP);
    // the lane has page n16 of rows 4 i + lane / 16
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * i + kq, p = base + n16;
      if (p < __shfl(stop, row, 64)) a.keys[((size_t)(t0 + row) * a.nkv + h) * a.key_stride + p] = key_of(now >= 0 ? acc[0][i] + acc[1][i] : -__builtin_inf());
    }
  }
}

// A workgroup per (row, kv head).  The threshold is found by digits of 8 bits within the window that still holds it, the first one
// cut from the range of the keys; then the kept pages are written in order.  R > 0: a thread has R of the keys in registers.
struct Shared {
  u64 lo[kWaves], hi[kWaves];
  int hist[3][256];
  int eq[32][kWaves], kept[32][kWaves];
};

template <int R>
__device__ __forceinline__ void pick(const Args& a, const u64* keys, int begin, int end, int need, int* out, Shared& sh) {
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  u64 k[R];
  u64 lo = ~0ull, hi = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = begin + r * kThreads + tid;
    k[r] = i < end ? keys[i] : 0;
    if (i < end) {
      lo = min(lo, k[r]);
      hi = max(hi, k[r]);
    }
  }
  auto there = [&](int r) { return begin + r * kThreads + tid < end; };
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, (u64)__shfl_xor(lo, o, 64));
    hi = max(hi, (u64)__shfl_xor(hi, o, 64));
  }
  if (lane == 0) {
    sh.lo[w] = lo;
    sh.hi[w] = hi;
  }
  sh.hist[0][tid] = 0;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    lo = min(lo, sh.lo[v]);
    hi = max(hi, sh.hi[v]);
  }
  // the window [lo, hi] holds the threshold; above it all are kept, `need` of it
  bool whole = false;      // the window's keys are all kept
  for (int turn = 0; lo < hi && !whole; ++turn) {
    int* hist = sh.hist[turn % 3];
    const int shift = max(64 - __clzll(hi - lo) - 8, 0);
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (there(r) && k[r] >= lo && k[r] <= hi) atomicAdd(&hist[(int)((k[r] - lo) >> shift)], 1);
    sh.hist[(turn + 1) % 3][tid] = 0;      // its last readers are before the last barrier
    __syncthreads();
    // every wave: lane's digits are 4 lane .. 4 lane + 3; how many keys lie above each
    const int4 c = reinterpret_cast<const int4*>(hist)[lane];
    int above = c.x + c.y + c.z + c.w;
    const int own = above;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int x = __shfl_down(above, o, 64);
      if (lane + o < 64) above += x;
    }
    above -= own;
    int digit = -1, over = 0, in = 0;
    const int cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int j = 3; j >= 0; --j) {
      if (above < need && above + cs[j] >= need) {
        digit = 4 * lane + j;
        over = above;
        in = cs[j];
      }
      above += cs[j];
    }
    const int src = __ffsll((u64)__ballot(digit >= 0)) - 1;      // one lane has it
    digit = __shfl(digit, src, 64);
    need -= __shfl(over, src, 64);
    whole = __shfl(in, src, 64) == need;
    lo += (u64)digit << shift;
    hi = lo + min(hi - lo, (u64)((1ull << shift) - 1));      // lo + 2^shift may not fit
  }
  // kept: keys > hi, and of those in [lo, hi] all, or (then lo == hi) the first `need`
  u64 kept[R];
  if (whole) {
#pragma unroll
    for (int r = 0; r < R; ++r) kept[r] = __ballot(there(r) && k[r] >= lo);
  } else {
    u64 eq[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      eq[r] = __ballot(there(r) && k[r] == lo);
      if (lane == 0) sh.eq[r][w] = __popcll(eq[r]);
    }
    __syncthreads();
    int before = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
      int mine = before;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        if (v < w) mine += sh.eq[r][v];
        before += sh.eq[r][v];
      }
      kept[r] = __ballot(there(r) && (k[r] > hi || (k[r] == lo && mine + __popcll(eq[r] & ((1ull << lane) - 1)) < need)));
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane == 0) sh.kept[r][w] = __popcll(kept[r]);
  __syncthreads();
  int at = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    int mine = at;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) {
      if (v < w) mine += sh.kept[r][v];
      at += sh.kept[r][v];
    }
    if (kept[r] >> lane & 1) out[mine + __popcll(kept[r] & ((1ull << lane) - 1))] = begin + r * kThreads + tid;
  }
}

// MOST: keys of a thread in registers at most (their number is the kernel's registers, and so how many workgroups share a compute unit)
template <int MOST>
__global__ __launch_bounds__(kThreads) void pick_pages_kernel(Args a) {
  const int t = blockIdx.x / a.nkv, h = blockIdx.x - t * a.nkv, tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int n = pages_of(a, t);
  int* out = a.out + ((size_t)t * a.nkv + h) * a.count;
  if (n <= a.count) {
    for (int i = tid; i < a.count; i += kThreads) out[i] = i < n ? i : -1;
    return;
  }
  const u64* keys = a.keys + ((size_t)t * a.nkv + h) * a.key_stride;
  const int begin = a.first, end = n - a.recent;
  int need = a.count - a.first - a.recent;
  for (int i = tid; i < a.first; i += kThreads) out[i] = i;
  for (int i = tid; i < a.recent; i += kThreads) out[a.count - a.recent + i] = n - a.recent + i;
  if (need == 0) return;
  __shared__ __attribute__((aligned(16))) Shared sh;
  out += a.first;
  if (end - begin <= 2 * kThreads) return pick<2>(a, keys, begin, end, need, out, sh);
  if (end - begin <= 4 * kThreads) return pick<4>(a, keys, begin, end, need, out, sh);
  if constexpr (MOST > 4) {
    if (end - begin <= 8 * kThreads) return pick<8>(a, keys, begin, end, need, out, sh);
    if (end - begin <= 16 * kThreads) return pick<16>(a, keys, begin, end, need, out, sh);
    if (end - begin <= 32 * kThreads) return pick<32>(a, keys, begin, end, need, out, sh);
  }

  // longer ones read their keys anew each time: the same in loops
  u64 lo = ~0ull, hi = 0;
  for (int i = begin + tid; i < end; i += kThreads) {
    lo = min(lo, keys[i]);
    hi = max(hi, keys[i]);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, (u64)__shfl_xor(lo, o, 64));
    hi = max(hi, (u64)__shfl_xor(hi, o, 64));
  }
  if (lane == 0) {
    sh.lo[w] = lo;
    sh.hi[w] = hi;
  }
  __syncthreads();
  for (int v = 0; v < kWaves; ++v) {
    lo = min(lo, sh.lo[v]);
    hi = max(hi, sh.hi[v]);
  }
  __shared__ int s_digit, s_above, s_in;
  bool whole = false;
  while (lo < hi) {
    int* hist = sh.hist[0];
    const int shift = max(64 - __clzll(hi - lo) - 8, 0);
    hist[tid] = 0;
    __syncthreads();
    for (int i = begin + tid; i < end; i += kThreads) {
      const u64 k = keys[i];
      if (k >= lo && k <= hi) atomicAdd(&hist[(int)((k - lo) >> shift)], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int above = 0, d = 255;
      for (; above + hist[d] < need; --d) above += hist[d];
      s_digit = d;
      s_above = above;
      s_in = hist[d];
    }
    __syncthreads();
    need -= s_above;
    lo += (u64)s_digit << shift;
    hi = lo + min(hi - lo, (u64)((1ull << shift) - 1));
    if (s_in == need) {
      whole = true;
      break;
    }
    __syncthreads();
  }
  int done = 0, ties = 0;
  for (int base = begin; base < end; base += kThreads) {
    const int i = base + tid;
    const u64 k = i < end ? keys[i] : 0;
    const bool in = i < end && k >= lo && k <= hi;
    const u64 eq = __ballot(in);
    __syncthreads();
    if (lane == 0) sh.eq[0][w] = __popcll(eq);
    __syncthreads();
    int before = ties;
    for (int v = 0; v < kWaves; ++v) {
      if (v < w) before += sh.eq[0][v];
      ties += sh.eq[0][v];
    }
    const bool kept = i < end && (k > hi || (in && (whole || before + __popcll(eq & ((1ull << lane) - 1)) < need)));
    const u64 b = __ballot(kept);
    if (lane == 0) sh.kept[0][w] = __popcll(b);
    __syncthreads();
    int at = done;
    for (int v = 0; v < kWaves; ++v) {
      if (v < w) at += sh.kept[0][v];
      done += sh.kept[0][v];
    }
    if (kept) out[at + __popcll(b & ((1ull << lane) - 1))] = i;
  }
}

template <int HD>
int scores(Args a, bool groups, hipStream_t s) {
  const int span = a.table_cols - a.first - a.recent, tiles = (a.T + kRows - 1) / kRows * a.nkv;
  // pages of a workgroup, a multiple of `unit`, so that there are about `want` workgroups
  auto chunk = [&](long long items, int unit, int want, int most) {
    return (int)min(max((items * span / want + unit - 1) / unit * unit, (long long)unit), (long long)most);
  };
  Args rows = a;
  rows.chunk = chunk((long long)a.nkv * a.T, 32, 2048, 1024);
  const dim3 grid(a.nkv * a.T, (span + rows.chunk - 1) / rows.chunk);
  if constexpr (HD <= 128) {      // 256 dims: a row's weights do not fit a lane's registers
    if (groups) {
      a.chunk = chunk(tiles, 64, 1024, 1 << 20);
      page_scores_tiles_kernel<HD><<<dim3(tiles, (span + a.chunk - 1) / a.chunk * kRuns), kThreads, 0, s>>>(a);
      DGI_CHECK_LAUNCH();
      page_scores_kernel<HD, true><<<grid, kThreads, 0, s>>>(rows);
      DGI_CHECK_LAUNCH();
      return 0;
    }
  }
  page_scores_kernel<HD, false><<<grid, kThreads, 0, s>>>(rows);
  DGI_CHECK_LAUNCH();
  return 0;
}

}  // namespace

extern "C" int dgi_select_pages(const void* q, long long q_stride, const void* bounds, const int* tables, int table_stride, int table_cols,
                                int n_seqs, int num_blocks, const int* ctx, const int* row_seq, int T, int nh, int nkv, int hd, int page,
                                int count, int first, int recent, void* keys, int key_stride, int* out, hipStream_t s) {
  if (T == 0) return 0;
  const Args a{(const uint16_t*)q, q_stride, (const uint16_t*)bounds, tables, table_stride, table_cols, n_seqs, num_blocks, ctx, row_seq,
               T, nh, nkv, page, count, first, recent, (u64*)keys, key_stride, out, 0};
  if (table_cols > count) {
    const bool groups = row_seq && T > n_seqs;      // else hardly two rows of one sequence
    int rc = -5;
    if (hd == 64) rc = scores<64>(a, groups, s);
    else if (hd == 128) rc = scores<128>(a, groups, s);
    else if (hd == 256) rc = scores<256>(a, groups, s);
    if (rc) return rc;
  }
  if (table_cols - first - recent <= 4 * kThreads) pick_pages_kernel<4><<<nkv * T, kThreads, 0, s>>>(a);
  else pick_pages_kernel<32><<<nkv * T, kThreads, 0, s>>>(a);
  DGI_CHECK_LAUNCH();
  return 0;
}
