// dgi/csrc/longctx/select_pages.hip — which pages of its context a row's group of heads is to read.
//
// With P_d = sum over the group of max(q_d, 0) and N_d = sum of min(q_d, 0), a page scores P . hi + N . lo: the sum over the group of
// the largest q . k that a key within the page's bounds can have.  Kept are the first and last pages (as many as the caller says) and the
// best of the others, ties to the lowest.
//
// Which page is kept is a whole number, and may not depend on the order in which a sum was taken: pages are compared by sums in 64 bits.
// What they are compared by goes into a workspace [T, n_kv, pages], and another launch chooses.
//
// Decode rows each have bounds of their own: the scores in 64 bits as a lane multiplies what it loads, as integers of the same order, whose
// digits from the top are counted until the threshold is found.  What bounds this are the loads of the bounds (64 rows over 4000 to 32000 keys,
// 8 kv heads of 128, 303 MB: 71 us at 4.3 TB/s, where a kernel that only reads reaches 6.3, and 7 us for the choice).
//
// Rows of a prompt share their sequence's bounds: 16 of them are the rows of bf16 matrix instructions, which give each score in 32 bits and
// a bound for its error; pages that the error leaves open are scored in 64 bits (1018 rows of 28 heads over 730 to 1000 pages of 4 kv heads
// of 128: 53 us, of which scores 30, looking for rows that do not go together 4, the choice 21; with the products in 64 bits on the matrix
// cores, whose rate alone is 24 us, 88 us).  What bounds this is latency: of the weights ahead of 4 steps of 64 pages, and of the choice.
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
  int T, nh, nkv, hd, page, count, first, recent;
  u64* keys;
  int key_stride;
  int* out;
  int chunk;      // pages of a workgroup
  int row_chunk;  // of one that scores a single row
};

__device__ __forceinline__ int pages_of(const Args& a, int t) {
  const int c = a.ctx[t];
  return c <= 0 ? 0 : min((c - 1) / a.page + 1, a.table_cols);
}

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLeast = 0x1p-110f;      // the least error: products too small for 32 bits
constexpr int kRows = 16, kRuns = 4;      // rows of an aligned group; it goes together if they are of so many sequences at most

__device__ __forceinline__ bool together(unsigned begins) { return __popc(begins & ((1u << kRows) - 1)) <= kRuns; }

// The aligned group of row t: bit i says that row i begins another sequence than the row before it (or is behind the last row).
__device__ __forceinline__ unsigned begins_of(const Args& a, int t, int lane, int& seq) {
  const int row = t / kRows * kRows + lane;
  seq = lane < kRows && row < a.T ? a.row_seq[row] : -1;
  const int prev = __shfl_up(seq, 1, 64);
  return (unsigned)__ballot(lane < kRows && (lane == 0 || row == a.T || (row < a.T && seq != prev))) | 1u << kRows;
}

// Eight channels of eight of a group's G heads, hd apart.
__device__ __forceinline__ void load_heads(u32x4* v, const uint16_t* q, int hd, int g0, int G) {
#pragma unroll
  for (int g = 0; g < 8; ++g) v[g] = *reinterpret_cast<const u32x4*>(q + min(g0 + g, G - 1) * hd);
}

// P and N of a group in 64 bits by N threads, [N | P] into LDS.
template <int N>
__device__ __forceinline__ void weigh(double* wgt, const uint16_t* q, int hd, int G) {
  for (int d = threadIdx.x % N; d < hd; d += N) {
    double up = 0., down = 0.;
    for (int g0 = 0; g0 < G; g0 += 8) {
      float x[8];
#pragma unroll
      for (int g = 0; g < 8; ++g) x[g] = bf16_to_f32(q[min(g0 + g, G - 1) * hd + d]);
#pragma unroll
      for (int g = 0; g < 8; ++g) {
        if (g0 + g >= G) x[g] = 0.f;
        up += x[g] < 0.f ? 0.f : x[g];        // no number stays none
        down += x[g] > 0.f ? 0.f : x[g];
      }
    }
    wgt[d] = down;
    wgt[hd + d] = up;
  }
}

__device__ __forceinline__ unsigned begins_of(const Args& a, int t, int lane) {
  int seq;
  return begins_of(a, t, lane, seq);
}

// A row's pages from `begin` on, `pages` of them.  Four 16-byte chunks of a page's [lo | hi] a lane, HD / 16 lanes a page; the next pages'
// bounds are under way while these are multiplied.  GROUPS: scores rounded to 32 bits, as page_screen_kernel leaves them.
template <int HD, bool GROUPS>
__device__ __forceinline__ void score_pages(const Args& a, double* wgt_s, int t, int h, int begin, int pages) {
  constexpr int LP = HD / 16, PW = 64 / LP, STEP = kWaves * PW;      // lanes a page, pages a wave and a workgroup at a time
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane % LP, p0 = lane / LP;
  // the first ids beside the context
  const int seq = a.row_seq ? a.row_seq[t] : t;
  const bool known = seq >= 0 && seq < a.n_seqs;
  const int* table = a.tables + (size_t)(known ? seq : 0) * a.table_stride;
  int base = begin + w * PW, id = known && base + p0 < a.table_cols ? table[base + p0] : -1;
  int id_next = known && base + STEP + p0 < a.table_cols ? table[base + STEP + p0] : -1;
  const int n = pages_of(a, t), end = min(begin + pages, n - a.recent);
  if (n <= a.count || begin >= end) return;
  const int G = a.nh / a.nkv;
  u64* keys = a.keys + ((size_t)t * a.nkv + h) * a.key_stride;
  auto valid = [&](int base, int id) { return base + p0 < end && id >= 0 && id < a.num_blocks ? id : -1; };
  auto id_of = [&](int base) { return valid(base, known && base + p0 < end ? table[base + p0] : -1); };
  u32x4 v[2][4];
  auto load = [&](u32x4* to, int id) {
    const uint16_t* bp = a.bounds + ((size_t)max(id, 0) * a.nkv + h) * 2 * HD + l * 8;
#pragma unroll
    for (int i = 0; i < 4; ++i) to[i] = *reinterpret_cast<const u32x4*>(bp + LP * i * 8);
  };
  id = valid(base, id);
  id_next = valid(base + STEP, id_next);
  load(v[0], id);
  weigh<kThreads>(wgt_s, a.q + t * a.q_stride + h * G * HD, HD, G);
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
    if (l != 0 || base + p0 >= end) return;
    if constexpr (GROUPS) {
      reinterpret_cast<float*>(keys)[base + p0] = id < 0 ? -__builtin_inff() : fabs(s) <= 0x1p126 ? (float)s : __builtin_nanf("");
    } else {
      keys[base + p0] = key_of(id >= 0 ? s : -__builtin_inf());
    }
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

// Row by row.
template <int HD>
__global__ __launch_bounds__(kThreads) void page_scores_kernel(Args a) {
  __shared__ double wgt_s[2 * HD];      // of lo, of hi
  const int t = blockIdx.x / a.nkv;
  score_pages<HD, false>(a, wgt_s, t, blockIdx.x - t * a.nkv, a.first + blockIdx.y * a.row_chunk, a.row_chunk);
}

// The rows that page_screen_kernel does not take.  Which groups of 16 these are each workgroup finds out by itself, 256 groups at a time, and
// takes every gridDim-th of their (group, pages, row, head); pages of a unit are such that there are some 2048 units.  (A workgroup for every
// row and head, most of which end at once: 4.6 us where there is no such row, and 24 for 12 rows over 1000 pages beside 500 of a prompt,
// which take 4.7 and 15.)
template <int HD>
__global__ __launch_bounds__(kThreads) void page_scores_alone_kernel(Args a) {
  __shared__ double wgt_s[2 * HD];
  __shared__ u64 alone_s[kWaves];
  const int tid = threadIdx.x, groups = (a.T + kRows - 1) / kRows, span = a.table_cols - a.first - a.recent;
  for (int g0 = 0; g0 < groups; g0 += kThreads) {
    const int row0 = (g0 + tid) * kRows;
    int runs = row0 < a.T, seqs[kRows];      // as begins_of has them
#pragma unroll
    for (int i = 0; i < kRows; ++i) seqs[i] = row0 + i < a.T ? a.row_seq[row0 + i] : 0;
#pragma unroll
    for (int i = 1; i < kRows; ++i) runs += row0 + i < a.T ? seqs[i] != seqs[i - 1] : row0 + i == a.T;
    const u64 mine = __ballot(runs > kRuns);
    __syncthreads();
    if ((tid & 63) == 0) alone_s[tid >> 6] = mine;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int v = 0; v < kWaves; ++v) n += __popcll(alone_s[v]);
    const int each = (int)min(max(((long long)n * kRows * a.nkv * span / 2048 + 31) / 32 * 32, 128ll), 1024ll), chunks = (span + each - 1) / each;
    for (long long unit = blockIdx.x; unit < (long long)n * chunks * kRows * a.nkv; unit += gridDim.x) {
      const int h = unit % a.nkv, row = unit / a.nkv % kRows;
      const long long place = unit / a.nkv / kRows;
      int rank = place / chunks, v = 0;
      u64 word = alone_s[0];
      while (rank >= __popcll(word)) {
        rank -= __popcll(word);
        word = alone_s[++v];
      }
      for (; rank > 0; --rank) word &= word - 1;
      const int t = (g0 + 64 * v + __ffsll(word) - 1) * kRows + row;
      __syncthreads();      // the unit before has read its weights
      if (t < a.T) score_pages<HD, true>(a, wgt_s, t, h, a.first + (int)(place % chunks) * each, each);
    }
  }
}

// Rows that go together: 16 x 16 (rows, pages) at a time, 32 channels an instruction, in fewer bits than the choice needs: a weight w
// is the sum of two bf16 numbers to |w| 2^-16, their products with the bounds are exact in 32 bits, and each of the 4 HD additions is
// off by no more than two steps of the last place, 2^-22 of S = sum |w| |bound| (all 256 of a chain together: 2^-20.8 of S at the worst, of half a
// million with exponents spread over 2 to 40); G heads are added up for a weight, each to 2^-24.  Small weights lose no more: queries are
// multiples of 2^-133, the last place of subnormal bf16 numbers, and so are their sums and what is left of them, so that a second number
// below 2^-126 is exact, and the matrix cores take subnormal numbers as they are.  A third
// product gives S (of the weights' first numbers, no less than 1 - 2^-8 of it).  Written are the score and, for a wave's pages of a
// row, the largest error; what no such bound holds for (infinite or no numbers) is written as none.
// A lane has row lane % 16's weights and page lane % 16's bounds of the chunks 4 j + lane / 16 of [lo | hi], eight values each.
template <int HD>
__global__ __launch_bounds__(kThreads, HD <= 128 ? 2 : 1) void page_screen_kernel(Args a) {
  constexpr int CH = HD / 4, J = CH / 4;      // chunks of a row of bounds, of them a lane's
  constexpr int LD = 2 * HD + 8;              // numbers between rows in LDS: reads of 16 rows hit other banks
  __shared__ __attribute__((aligned(16))) uint16_t wgt_s[2][kRows * LD];
  const int group = blockIdx.x / a.nkv, h = blockIdx.x - group * a.nkv, t0 = group * kRows;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, n16 = lane & 15, kq = lane >> 4;
  int seqs;
  const unsigned begins = begins_of(a, t0, lane, seqs);
  if (!together(begins)) return;
  const int G = a.nh / a.nkv;
  const float error = 1.02f * (HD * 0x1p-20f + 0x1p-16f + G * 0x1p-24f);
  // contexts, the first run's ids and queries are loaded together
  constexpr int STEP = kWaves * 16, TASKS = kRows * (HD / 8);
  const int begin = a.first + blockIdx.y * a.chunk, begin_w = begin + 16 * w;
  const int ctx = t0 + n16 < a.T ? a.ctx[t0 + n16] : 0;
  const int* table = nullptr;
  auto id_of = [&](int base, int end) {
    const int p = base + n16, id = table && p < end ? table[p] : -1;
    return id >= 0 && id < a.num_blocks ? id : -1;
  };
  auto table_of = [&](int r) {
    const int seq = __builtin_amdgcn_readlane(seqs, r);
    return seq >= 0 && seq < a.n_seqs ? a.tables + (size_t)seq * a.table_stride : nullptr;
  };
  table = table_of(0);
  int id = id_of(begin_w, a.table_cols), id_next = id_of(begin_w + STEP, a.table_cols);
  u32x4 qv[8];
  auto q_of = [&](int i) { return a.q + min(t0 + i / (HD / 8), a.T - 1) * a.q_stride + h * G * HD + i % (HD / 8) * 8; };
  load_heads(qv, q_of(tid % TASKS), HD, 0, G);
  const int n = ctx <= 0 ? 0 : min((ctx - 1) / a.page + 1, a.table_cols);
  const int stop_n16 = n > a.count ? n - a.recent : 0;      // pages that row n16 needs scores of end here
  u32x4 v[2][J];
  auto load = [&](u32x4* v, int id) {
    const uint16_t* bp = a.bounds + ((size_t)max(id, 0) * a.nkv + h) * 2 * HD + kq * 8;
#pragma unroll
    for (int j = 0; j < J; ++j) v[j] = *reinterpret_cast<const u32x4*>(bp + j * 32);
  };
  bf16x8 wgt[2][J];
  bool ready = false;
  // the runs of rows of one sequence
  for (int r0 = 0; r0 < kRows && t0 + r0 < a.T;) {
    const int r1 = __ffs(begins >> (r0 + 1)) + r0;
    const int stop = n16 >= r0 && n16 < r1 ? stop_n16 : 0;
    int last = stop;
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) last = max(last, __shfl_xor(last, o, 64));
    const int end = __builtin_amdgcn_readfirstlane(min(begin + a.chunk, last));
    if (begin >= end) {
      r0 = r1;
      continue;
    }
    if (r0 > 0) {
      table = table_of(r0);
      id = id_of(begin_w, end);
      id_next = id_of(begin_w + STEP, end);
    }
    load(v[0], id);
    if (!ready) {
      // weights of the group's rows
      for (int i = tid; i < TASKS; i += kThreads) {
        const int row = i / (HD / 8), c = i - row * (HD / 8);
        if (i > tid) load_heads(qv, q_of(i), HD, 0, G);
        float both[2][8] = {};
        for (int g0 = 0; g0 < G; g0 += 8) {
          if (g0 > 0) load_heads(qv, q_of(i), HD, g0, G);
#pragma unroll
          for (int g = 0; g < 8; ++g) {
            if (g0 + g >= G) break;
            float x[8];
            unpack8(qv[g], x);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              both[0][j] += x[j] - fabsf(x[j]);      // twice the smaller of x and 0
              both[1][j] += x[j] + fabsf(x[j]);
            }
          }
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          float x[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) both[half][j] *= 0.5f;
          const u32x4 high = pack8(both[half]);
          unpack8(high, x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] = both[half][j] - x[j];
          *reinterpret_cast<u32x4*>(&wgt_s[0][row * LD + half * HD + c * 8]) = high;
          *reinterpret_cast<u32x4*>(&wgt_s[1][row * LD + half * HD + c * 8]) = pack8(x);
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int s = 0; s < 2; ++s) wgt[s][j] = *reinterpret_cast<const bf16x8*>(&wgt_s[s][n16 * LD + (4 * j + kq) * 8]);
      ready = true;
    }
    // the lane has page n16 of rows 4 kq + i
    int stops[4];
    float largest[4] = {}, *to[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      stops[i] = __shfl(stop, 4 * kq + i, 64);
      to[i] = reinterpret_cast<float*>(a.keys + ((size_t)(t0 + 4 * kq + i) * a.nkv + h) * a.key_stride);
    }
    auto score = [&](const u32x4* v, int base, int id) {
      f32x4 acc[2] = {}, sum = {};
#pragma unroll
      for (int j = 0; j < J; ++j) {
        acc[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wgt[0][j], as_bf16x8(v[j]), acc[0], 0, 0, 0);
        acc[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wgt[1][j], as_bf16x8(v[j]), acc[1], 0, 0, 0);
        // the weights of lo are none above zero, those of hi none below it
        const u32x4 size = j < J / 2 ? v[j] | 0x80008000u : v[j] & 0x7fff7fffu;
        sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wgt[0][j], as_bf16x8(size), sum, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = base + n16;
        if (p >= stops[i]) continue;
        float x = acc[0][i] + acc[1][i];
        if (!(fabsf(x) <= 0x1p126f && sum[i] <= 0x1p126f)) x = __builtin_nanf("");
        if (id < 0) x = -__builtin_inff();
        else largest[i] = fmaxf(largest[i], sum[i]);
        to[i][p] = x;
      }
    };
    for (int base = begin_w; base < end; base += 2 * STEP) {
      int id2 = id_of(base + 2 * STEP, end);
      load(v[1], id_next);
      score(v[0], base, id);
      if (base + STEP >= end) break;
      id = id2;
      load(v[0], id);
      id2 = id_of(base + 3 * STEP, end);
      score(v[1], base + STEP, id_next);
      id_next = id2;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) largest[i] = fmaxf(largest[i], __shfl_xor(largest[i], o, 64));
      if (n16 == 0 && begin_w < stops[i]) to[i][a.key_stride + blockIdx.y * kWaves + w] = largest[i] * error + kLeast;
    }
    r0 = r1;
  }
}

// A workgroup per (row, kv head).  The threshold is found by digits of 8 bits within the window that still holds it, the first one
// cut from the range of the keys; then the kept pages are written in order.  A thread has R of the keys in registers, the first two of
// them from `ahead`.
struct Long {
  u64 lo[kWaves], hi[kWaves];
  alignas(16) int hist[256];      // read four at a time
  int eq[kWaves], kept[kWaves], digit, above, in;
};

struct Shared {
  u64 lo[kWaves], hi[kWaves];
  alignas(16) int hist[3][256];
  int eq[32][kWaves], kept[32][kWaves];
  Long any;
};

// The digit of the need-th largest; `need` becomes what is needed of it and `in` what has it.  Every wave does this for itself.
__device__ __forceinline__ int digit_of(const int* hist, int lane, int& need, int& in) {
  // a lane's digits are 4 lane .. 4 lane + 3; how many keys lie above each
  const int4 c = reinterpret_cast<const int4*>(hist)[lane];
  const int own = c.x + c.y + c.z + c.w;
  int above = own;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_down(above, o, 64);
    if (lane + o < 64) above += x;
  }
  above -= own;
  int digit = -1, over = 0, has = 0;
  const int cs[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
  for (int j = 3; j >= 0; --j) {
    if (above < need && above + cs[j] >= need) {
      digit = 4 * lane + j;
      over = above;
      has = cs[j];
    }
    above += cs[j];
  }
  const int src = __ffsll((u64)__ballot(digit >= 0)) - 1;      // one lane has it
  need -= __shfl(over, src, 64);
  in = __shfl(has, src, 64);
  return __shfl(digit, src, 64);
}

// The kept of R * 256 in order; sh.kept has their numbers by turn and wave.
template <int R>
__device__ __forceinline__ void write_kept(const u64* kept, int begin, int* out, const Shared& sh) {
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
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

template <int R>
__device__ __forceinline__ void pick(const u64* keys, const u64* ahead, int begin, int end, int need, int* out, Shared& sh) {
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  u64 k[R];
  u64 lo = ~0ull, hi = 0;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = begin + r * kThreads + tid;
    k[r] = i < end ? r < 2 ? ahead[r] : keys[i] : 0;
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
    int in;
    const int digit = digit_of(hist, lane, need, in);
    whole = in == need;
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
  write_kept<R>(kept, begin, out, sh);
}

// W waves together: all of a workgroup's, or one by itself.
template <int W>
__device__ __forceinline__ void sync() {
  if constexpr (W > 1) {
    __syncthreads();
  } else {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// The same for any number of keys, read anew each time, by W waves.
template <int W>
__device__ void pick_long(const u64* keys, int begin, int end, int need, int* out, Long& sh) {
  constexpr int N = 64 * W;
  const int tid = threadIdx.x % N, w = tid >> 6, lane = tid & 63;
  u64 lo = ~0ull, hi = 0;
  for (int i = begin + tid; i < end; i += N) {
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
  sync<W>();
  for (int v = 0; v < W; ++v) {
    lo = min(lo, sh.lo[v]);
    hi = max(hi, sh.hi[v]);
  }
  bool whole = false;
  while (lo < hi) {
    const int shift = max(64 - __clzll(hi - lo) - 8, 0);
    for (int i = tid; i < 256; i += N) sh.hist[i] = 0;
    sync<W>();
    for (int i = begin + tid; i < end; i += N) {
      const u64 k = keys[i];
      if (k >= lo && k <= hi) atomicAdd(&sh.hist[(int)((k - lo) >> shift)], 1);
    }
    sync<W>();
    if (tid == 0) {
      int above = 0, d = 255;
      for (; above + sh.hist[d] < need; --d) above += sh.hist[d];
      sh.digit = d;
      sh.above = above;
      sh.in = sh.hist[d];
    }
    sync<W>();
    need -= sh.above;
    lo += (u64)sh.digit << shift;
    hi = lo + min(hi - lo, (u64)((1ull << shift) - 1));
    if (sh.in == need) {
      whole = true;
      break;
    }
    sync<W>();
  }
  int done = 0, ties = 0;
  for (int base = begin; base < end; base += N) {
    const int i = base + tid;
    const u64 k = i < end ? keys[i] : 0;
    const bool in = i < end && k >= lo && k <= hi;
    const u64 eq = __ballot(in);
    sync<W>();
    if (lane == 0) sh.eq[w] = __popcll(eq);
    sync<W>();
    int before = ties;
    for (int v = 0; v < W; ++v) {
      if (v < w) before += sh.eq[v];
      ties += sh.eq[v];
    }
    const bool kept = i < end && (k > hi || (in && (whole || before + __popcll(eq & ((1ull << lane) - 1)) < need)));
    const u64 b = __ballot(kept);
    if (lane == 0) sh.kept[w] = __popcll(b);
    sync<W>();
    int at = done;
    for (int v = 0; v < W; ++v) {
      if (v < w) at += sh.kept[v];
      done += sh.kept[v];
    }
    if (kept) out[at + __popcll(b & ((1ull << lane) - 1))] = i;
  }
}

// 32-bit integers of the order of the floats; no number is the largest.
__device__ __forceinline__ unsigned key_of(float x) {
  const unsigned b = __float_as_uint(x + 0.f);
  return x != x ? ~0u : b >> 31 ? ~b : b | 1u << 31;
}
__device__ __forceinline__ float float_of(unsigned k) { return __uint_as_float(k >> 31 ? k ^ 1u << 31 : ~k); }

// A page's score in 64 bits by 16 lanes; `l` is the lane's place among them.
__device__ __forceinline__ u64 score_of(const Args& a, const double* wgt, const int* table, int h, int p, int l) {
  const int id = table ? table[p] : -1;
  if (id < 0 || id >= a.num_blocks) return key_of(-__builtin_inf());
  const uint16_t* b = a.bounds + ((size_t)id * a.nkv + h) * 2 * a.hd;
  double sum[2] = {};
  for (int c = l; c < a.hd / 4; c += 16) {
    float x[8];
    unpack8(*reinterpret_cast<const u32x4*>(b + c * 8), x);
#pragma unroll
    for (int j = 0; j < 8; ++j) sum[j & 1] = fma(wgt[c * 8 + j], (double)x[j], sum[j & 1]);
  }
  double s = sum[0] + sum[1];
#pragma unroll
  for (int o = 1; o < 16; o <<= 1) s += __shfl_xor(s, o, 64);
  return key_of(s);
}

// From scores that are off by an error E at most.  With the threshold of these scores in [lo, hi], that of the true ones is in
// [lo - E, hi + E]: pages above hi + 2 E are kept, those below lo - 2 E are not, and those between (1 to 8 of 1000 where
// bounds are normal) are scored again in 64 bits and take the places that are left.  Where there are too many of them, or
// scores without a bound, all are.
// W waves a row: one for up to 1024 pages (1018 rows over 730 to 1000 pages of 4 heads: 21 us, by all four of a workgroup 45), four for
// more.  A wave has turns * 64 pages in a row, R > 0: R of them at most a lane, in registers; 0: they are read anew each time.
template <int R, int W>
struct Screened {
  static constexpr int kBand = 64 * W;      // pages scored again at most: a thread each
  Long any;
  unsigned lo[W], hi[W];
  float error[W];
  int sure[W], band, page[kBand];
  u64 key[kBand];
  u64 kept[R ? R * W : 1];      // of the pages scored again: a bit a page
};

template <int R, int W>
__global__ __launch_bounds__(kThreads) void pick_screened_kernel(Args a) {
  constexpr int N = 64 * W;
  typedef Screened<R, W> S;
  extern __shared__ __attribute__((aligned(16))) double wgt_s[];      // 2 hd a row: of lo, of hi
  __shared__ S teams[kWaves / W];
  static_assert(alignof(S) >= 16 && offsetof(S, any.hist) % 16 == 0, "each team's counts are read 16 bytes at a time");
  const int team = __builtin_amdgcn_readfirstlane(threadIdx.x / N), tid = threadIdx.x % N;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int item = blockIdx.x * (kWaves / W) + team, t = item / a.nkv, h = item - t * a.nkv, G = a.nh / a.nkv;
  if (t >= a.T) return;
  S& s = teams[team];
  double* wgt = wgt_s + team * 2 * a.hd;
  u64* row = a.keys + ((size_t)t * a.nkv + h) * a.key_stride;
  float* scores = reinterpret_cast<float*>(row);
  // all that is read is under way together; a wave by itself reads scores before it knows how many there are
  int seqs;
  const bool tiles = together(begins_of(a, t, lane, seqs));
  const int ctx = a.ctx[t], begin = a.first;
  float raw[R ? R : 1], E_first = tid < a.table_cols ? scores[a.key_stride + tid] : 0.f;
  if constexpr (W == 1) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int i = begin + r * 64 + lane;
      raw[r] = i < a.table_cols ? scores[i] : 0.f;
    }
  }
  weigh<N>(wgt, a.q + t * a.q_stride + h * G * a.hd, a.hd, G);
  const int n = ctx <= 0 ? 0 : min((ctx - 1) / a.page + 1, a.table_cols), seq = __builtin_amdgcn_readlane(seqs, t % kRows);
  int* out = a.out + ((size_t)t * a.nkv + h) * a.count;
  if (n <= a.count) {
    for (int i = tid; i < a.count; i += N) out[i] = i < n ? i : -1;
    return;
  }
  const int end = n - a.recent, need = a.count - a.first - a.recent;
  for (int i = tid; i < a.first; i += N) out[i] = i;
  for (int i = tid; i < a.recent; i += N) out[a.count - a.recent + i] = end + i;
  if (need == 0) return;
  out += a.first;
  const int turns = (end - begin + N - 1) / N, begin_w = begin + w * turns * 64;
  unsigned k[R ? R : 1];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int i = begin_w + r * 64 + lane;
    const bool there = r < turns && i < end;
    if constexpr (W > 1) raw[r] = there ? scores[i] : 0.f;
    k[r] = there ? key_of(raw[r]) : 0;      // below any score's
  }
  // `f` of the turns' keys
  auto each = [&](auto f) {
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < turns) f(r, k[r]);
    } else {
      for (int r = 0; r < turns; ++r) {
        const int i = begin_w + r * 64 + lane;
        f(r, i < end ? key_of(scores[i]) : 0u);
      }
    }
  };
  // errors are those of chunks of pages, 16 of them a wave at a time, or of a rounding
  float E = 0.f;
  if (tiles)
    for (int i = tid; (i / kWaves) * a.chunk + 16 * (i % kWaves) < end - begin; i += N) E = fmaxf(E, i == tid ? E_first : scores[a.key_stride + i]);
  unsigned lo = ~0u, hi = 0;
  each([&](int, unsigned x) {
    lo = min(lo, x ? x : ~0u);
    hi = max(hi, x);
  });
  if (!tiles)
    each([&](int, unsigned x) {
      const float size = fabsf(float_of(x));
      if (x && size <= 0x1p126f) E = fmaxf(E, size * 0x1p-23f + kLeast);
    });
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    lo = min(lo, (unsigned)__shfl_xor((int)lo, o, 64));
    hi = max(hi, (unsigned)__shfl_xor((int)hi, o, 64));
    E = fmaxf(E, __shfl_xor(E, o, 64));
  }
  if constexpr (R > 0) {
    for (int i = tid; i < R * W; i += N) s.kept[i] = 0;
  }
  if (tid == 0) s.band = 0;
  if constexpr (W > 1) {
    if (lane == 0) {
      s.lo[w] = lo;
      s.hi[w] = hi;
      s.error[w] = E;
    }
    sync<W>();
#pragma unroll
    for (int v = 0; v < W; ++v) {
      lo = min(lo, s.lo[v]);
      hi = max(hi, s.hi[v]);
      E = fmaxf(E, s.error[v]);
    }
  }
  const int* table = seq >= 0 && seq < a.n_seqs ? a.tables + (size_t)seq * a.table_stride : nullptr;
  const int l16 = lane & 15, p16 = tid >> 4;
  if (hi != ~0u) {
    int left = need;      // places for the pages of the window [lo, hi]
    while (lo < hi && !(float_of(hi) - float_of(lo) <= E)) {
      const int shift = max(32 - __clz(hi - lo) - 8, 0);
      for (int i = tid; i < 256; i += N) s.any.hist[i] = 0;
      sync<W>();
      each([&](int, unsigned x) {
        if (x >= lo && x <= hi) atomicAdd(&s.any.hist[(x - lo) >> shift], 1);
      });
      sync<W>();
      int in;
      const int digit = digit_of(s.any.hist, lane, left, in);
      lo += (unsigned)digit << shift;
      hi = lo + min(hi - lo, (1u << shift) - 1);
      sync<W>();
    }
    const float from = float_of(lo) - 2.01f * E, above = float_of(hi) + 2.01f * E;
    const unsigned from_k = key_of(from), above_k = key_of(above);
    int sure = 0;
    sync<W>();
    each([&](int r, unsigned x) {
      const u64 over = __ballot(x > above_k), between = __ballot(x >= from_k && x <= above_k);
      sure += __popcll(over);
      if (!between) return;
      int at = 0;
      if (lane == 0) at = atomicAdd(&s.band, __popcll(between));
      at = __shfl(at, 0, 64) + __popcll(between & ((1ull << lane) - 1));
      if ((between >> lane & 1) && at < S::kBand) s.page[at] = begin_w + r * 64 + lane;
    });
    if constexpr (W > 1) {
      if (lane == 0) s.sure[w] = sure;
    }
    sync<W>();
    if constexpr (W > 1) {
      sure = 0;
#pragma unroll
      for (int v = 0; v < W; ++v) sure += s.sure[v];
    }
    const int m = __builtin_amdgcn_readfirstlane(s.band);
    left = need - sure;
    if (m <= S::kBand) {
      if (m > left)
        for (int i = p16; i < m; i += N / 16) {
          const u64 x = score_of(a, wgt, table, h, s.page[i], l16);
          if (l16 == 0) s.key[i] = x;
        }
      sync<W>();
      if (tid < m) {
        const int p = s.page[tid];
        const u64 x = s.key[tid];
        int before = 0;
        if (m > left)
          for (int i = 0; i < m; ++i) before += s.key[i] > x || (s.key[i] == x && s.page[i] < p);
        if constexpr (R > 0) {
          if (before < left) atomicOr(reinterpret_cast<unsigned*>(s.kept) + (p - begin) / 32, 1u << (p - begin) % 32);
        } else {
          scores[p] = before < left ? __builtin_inff() : -__builtin_inff();
        }
      }
      sync<W>();
      // the kept ones in order: after those of the waves before
      auto kept_of = [&](int r, unsigned x) {
        u64 b = __ballot(x > above_k);
        if constexpr (R > 0) b |= s.kept[w * turns + r];
        return b;
      };
      int at = 0;
      if constexpr (W > 1) {
        int mine = 0;
        each([&](int r, unsigned x) { mine += __popcll(kept_of(r, x)); });
        if (lane == 0) s.sure[w] = mine;
        sync<W>();
        for (int v = 0; v < w; ++v) at += s.sure[v];
      }
      each([&](int r, unsigned x) {
        const u64 b = kept_of(r, x);
        if (b >> lane & 1) out[at + __popcll(b & ((1ull << lane) - 1))] = begin_w + r * 64 + lane;
        at += __popcll(b);
      });
      return;
    }
  }
  sync<W>();
  for (int p = begin + p16; p < end; p += N / 16) {
    const u64 x = score_of(a, wgt, table, h, p, l16);
    if (l16 == 0) row[p] = x;
  }
  sync<W>();
  pick_long<W>(row, begin, end, need, out, s.any);
}

// MOST: keys of a thread in registers at most (their number is the kernel's registers, and so how many workgroups share a compute unit).
template <int MOST>
__global__ __launch_bounds__(kThreads) void pick_pages_kernel(Args a) {
  const int t = blockIdx.x / a.nkv, h = blockIdx.x - t * a.nkv, tid = threadIdx.x, begin = a.first;
  const u64* keys = a.keys + ((size_t)t * a.nkv + h) * a.key_stride;
  u64 ahead[2];      // read beside the context; there are keys only if a table may have more pages than are kept
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    const int i = begin + r * kThreads + tid;
    ahead[r] = a.table_cols > a.count && i < a.table_cols ? keys[i] : 0;
  }
  const int n = pages_of(a, t), end = n - a.recent;
  int* out = a.out + ((size_t)t * a.nkv + h) * a.count;
  if (n <= a.count) {
    for (int i = tid; i < a.count; i += kThreads) out[i] = i < n ? i : -1;
    return;
  }
  const int need = a.count - a.first - a.recent;
  for (int i = tid; i < a.first; i += kThreads) out[i] = i;
  for (int i = tid; i < a.recent; i += kThreads) out[a.count - a.recent + i] = end + i;
  if (need == 0) return;
  out += a.first;
  __shared__ Shared sh;
  if (end - begin <= 2 * kThreads) return pick<2>(keys, ahead, begin, end, need, out, sh);
  if (end - begin <= 4 * kThreads) return pick<4>(keys, ahead, begin, end, need, out, sh);
  if constexpr (MOST > 4) {
    if (end - begin <= 8 * kThreads) return pick<8>(keys, ahead, begin, end, need, out, sh);
    if (end - begin <= 16 * kThreads) return pick<16>(keys, ahead, begin, end, need, out, sh);
    if (end - begin <= 32 * kThreads) return pick<32>(keys, ahead, begin, end, need, out, sh);
  }
  pick_long<kWaves>(keys, begin, end, need, out, sh.any);
}

template <int HD>
int scores(Args& a, bool groups, hipStream_t s) {
  const int span = a.table_cols - a.first - a.recent, tiles = (a.T + kRows - 1) / kRows * a.nkv;
  // pages of a workgroup, a multiple of `unit`, so that there are about `want` workgroups
  auto chunk = [&](long long items, int unit, int want, int most) {
    return (int)min(max((items * span / want + unit - 1) / unit * unit, (long long)unit), (long long)most);
  };
  if (!groups) {
    a.row_chunk = chunk((long long)a.nkv * a.T, 32, 2048, 1024);
    const dim3 grid(a.nkv * a.T, (span + a.row_chunk - 1) / a.row_chunk);
    page_scores_kernel<HD><<<grid, kThreads, 0, s>>>(a);
    DGI_CHECK_LAUNCH();
    return 0;
  }
  a.chunk = chunk(tiles, 64, 1024, 1 << 20);
  page_screen_kernel<HD><<<dim3(tiles, (span + a.chunk - 1) / a.chunk), kThreads, 0, s>>>(a);
  DGI_CHECK_LAUNCH();
  page_scores_alone_kernel<HD><<<512, kThreads, 0, s>>>(a);
  DGI_CHECK_LAUNCH();
  return 0;
}

template <int R, int W>
void pick_screened(const Args& a, hipStream_t s) {
  constexpr int rows = kWaves / W;
  pick_screened_kernel<R, W><<<(a.nkv * a.T + rows - 1) / rows, kThreads, rows * 2 * a.hd * sizeof(double), s>>>(a);
}

}  // namespace

extern "C" int dgi_select_pages(const void* q, long long q_stride, const void* bounds, const int* tables, int table_stride, int table_cols,
                                int n_seqs, int num_blocks, const int* ctx, const int* row_seq, int T, int nh, int nkv, int hd, int page,
                                int count, int first, int recent, void* keys, int key_stride, int key_rows, int* out, hipStream_t s) {
  // Rows in groups only if there are more than sequences (else hardly two of one), and where that saves more than the third launch and the
  // second look at some pages take, about 9 us.  Row by row / in groups, us: 32 rows of 8 heads of 128 over 500 pages 16.8, 18.3, over
  // 1000 22.9, 21.2; 64 over 100 13.6, 15.5, over 500 22.9, 19.3; 128 over 100 17.2, 15.7, over 1000 53, 30; 64 rows of 4 heads over 500
  // 17.3, 19.2; 512 rows of one head of 64 over 500 15.8, 18.4, over 1000 21.1, 21.2; 128 rows of 2 heads of 256 over 500 23.9, 24.4.  The tables
  // were as wide as the contexts: how long these are the host does not know, and a wider table counts as its width, here and in the keys of a
  // lane below (1018 rows of 28 heads on 4 over 730 to 1000 pages 53, of a table of 8192 columns 87).
  const int span = table_cols - first - recent;
  const bool groups = row_seq && T > n_seqs && (double)T * nkv * (span + 40) * min(hd, 128) >= 18e6;
  for (int t0 = 0; t0 < T; t0 += key_rows) {
    Args a{(const uint16_t*)q + t0 * q_stride, q_stride, (const uint16_t*)bounds,
           row_seq ? tables : tables + (size_t)t0 * table_stride, table_stride, table_cols, row_seq ? n_seqs : n_seqs - t0, num_blocks,
           ctx + t0, row_seq ? row_seq + t0 : nullptr, min(key_rows, T - t0), nh, nkv, hd, page, count, first, recent, (u64*)keys,
           key_stride, out + (size_t)t0 * nkv * count, 0, 0};
    if (table_cols > count) {
      int rc = -5;
      if (hd == 64) rc = scores<64>(a, groups, s);
      else if (hd == 128) rc = scores<128>(a, groups, s);
      else if (hd == 256) rc = scores<256>(a, groups, s);
      if (rc) return rc;
    }
    if (!groups || table_cols <= count) {
      if (span <= 4 * kThreads) pick_pages_kernel<4><<<nkv * a.T, kThreads, 0, s>>>(a);
      else pick_pages_kernel<32><<<nkv * a.T, kThreads, 0, s>>>(a);
    } else if (span <= 4 * 64) {
      pick_screened<4, 1>(a, s);
    } else if (span <= 16 * 64) {
      pick_screened<16, 1>(a, s);
    } else if (span <= 32 * kThreads) {
      pick_screened<32, kWaves>(a, s);
    } else {
      pick_screened<0, kWaves>(a, s);
    }
    DGI_CHECK_LAUNCH();
  }
  return 0;
}
