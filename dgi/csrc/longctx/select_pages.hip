// dgi/csrc/longctx/select_pages.hip — which pages of its context a row's group of heads is to read.
//
// With P_d = sum over the group of max(q_d, 0) and N_d = sum of min(q_d, 0), a page scores P . hi + N . lo: the sum over the group of
// the largest q . k that a key within the page's bounds can have.  Kept are the first and last pages (as many as the caller says) and the
// best of the others, ties to the lowest.
//
// Scores are summed in 64 bits: which page is kept is a whole number, and may not depend on the order in which a sum was taken.  Two
// launches: scores, as integers of the same order, into a workspace [T, n_kv, pages]; then the choice, by digits of these integers
// taken from the top.
#include "../common.h"

using namespace dgi;

namespace {

typedef unsigned long long u64;

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
};

__device__ __forceinline__ int pages_of(const Args& a, int t) {
  const int c = a.ctx[t];
  return c <= 0 ? 0 : min((c - 1) / a.page + 1, a.table_cols);
}

constexpr int kThreads = 256, kWaves = kThreads / 64;

// Four 16-byte chunks of a page's [lo | hi] a lane, HD / 16 lanes a page.
template <int HD>
__global__ __launch_bounds__(kThreads) void page_scores_kernel(Args a, int chunk) {
  constexpr int LP = HD / 16, PW = 64 / LP;      // lanes a page, pages a wave at a time
  const int t = blockIdx.x / a.nkv, h = blockIdx.x - t * a.nkv;
  const int n = pages_of(a, t);
  if (n <= a.count) return;
  const int begin = a.first + blockIdx.y * chunk, end = min(begin + chunk, n - a.recent);
  if (begin >= end) return;
  const int w = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane % LP, p0 = lane / LP;
  const int G = a.nh / a.nkv;
  // chunk l + LP i: the lo half for i < 2, the hi half behind it
  double wgt[4][8];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) wgt[i][j] = 0.0;
  for (int g = 0; g < G; ++g) {
    const uint16_t* qp = a.q + t * a.q_stride + (h * G + g) * HD;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x[8];
      unpack8(*reinterpret_cast<const u32x4*>(qp + (l + LP * i) * 8), x);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        wgt[i][j] += x[j] > 0.f ? 0.f : x[j];
        wgt[i + 2][j] += x[j] < 0.f ? 0.f : x[j];
      }
    }
  }
  const int seq = a.row_seq ? a.row_seq[t] : t;
  const bool known = seq >= 0 && seq < a.n_seqs;
  const int* table = a.tables + (size_t)(known ? seq : 0) * a.table_stride;
  u64* keys = a.keys + ((size_t)t * a.nkv + h) * a.key_stride;
  for (int base = begin + w * PW; base < end; base += kWaves * PW) {
    const int p = base + p0;
    const int id = known && p < end ? table[p] : -1;
    const bool there = id >= 0 && id < a.num_blocks;
    double sum = 0.0;
    if (there) {
      const uint16_t* bp = a.bounds + ((size_t)id * a.nkv + h) * 2 * HD + l * 8;
      u32x4 v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = *reinterpret_cast<const u32x4*>(bp + LP * i * 8);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float x[8];
        unpack8(v[i], x);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum = fma(wgt[i][j], (double)x[j], sum);
      }
    }
#pragma unroll
    for (int o = 1; o < LP; o <<= 1) sum += __shfl_xor(sum, o, 64);
    if (l == 0 && p < end) keys[p] = key_of(there ? sum : -__builtin_inf());
  }
}

// A workgroup per (row, kv head).  The threshold is found by digits of 8 bits within the window that still holds it, the first one
// cut from the range of the keys; then the kept pages are written in order.
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

  __shared__ u64 s_lo[kWaves], s_hi[kWaves];
  __shared__ int hist[256], s_digit, s_above, s_in;
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
    s_lo[w] = lo;
    s_hi[w] = hi;
  }
  __syncthreads();
  for (int v = 0; v < kWaves; ++v) {
    lo = min(lo, s_lo[v]);
    hi = max(hi, s_hi[v]);
  }
  // the window [lo, hi] holds the threshold; `above` it all are kept, `need` of it
  bool whole = false;      // the window's keys are all kept
  while (lo < hi) {
    const int bits = 64 - __clzll(hi - lo);
    const int shift = max(bits - 8, 0);
    hist[tid] = 0;
    __syncthreads();
    for (int i = begin + tid; i < end; i += kThreads) {
      const u64 k = keys[i];
      if (k >= lo && k <= hi) atomicAdd(&hist[(int)((k - lo) >> shift)], 1);
    }
    __syncthreads();
    if (w == 0) {      // lane: digits 4 lane .. 4 lane + 3; how many keys lie above each
      const int c0 = hist[4 * lane], c1 = hist[4 * lane + 1], c2 = hist[4 * lane + 2], c3 = hist[4 * lane + 3];
      int above = c0 + c1 + c2 + c3;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_down(above, o, 64);
        if (lane + o < 64) above += x;
      }
      above -= c0 + c1 + c2 + c3;
      const int c[4] = {c0, c1, c2, c3};
#pragma unroll
      for (int j = 3; j >= 0; --j) {
        if (above < need && above + c[j] >= need) {
          s_digit = 4 * lane + j;
          s_above = above;
          s_in = c[j];
        }
        above += c[j];
      }
    }
    __syncthreads();
    need -= s_above;
    lo += (u64)s_digit << shift;
    hi = lo + min(hi - lo, (u64)((1ull << shift) - 1));      // lo + 2^shift may not fit
    if (s_in == need) {
      whole = true;
      break;
    }
    __syncthreads();
  }
  // kept: keys > hi, and of those in [lo, hi] all, or (then lo == hi) the first `need`
  __shared__ int s_gt[kWaves], s_eq[kWaves];
  int done = a.first, ties = 0;
  for (int base = begin; base < end; base += kThreads) {
    const int i = base + tid;
    const u64 k = i < end ? keys[i] : 0;
    const bool in = i < end && k >= lo && k <= hi;
    const u64 eq = __ballot(in);
    __syncthreads();
    if (lane == 0) s_eq[w] = __popcll(eq);
    __syncthreads();
    int before = ties;
    for (int v = 0; v < kWaves; ++v) {
      if (v < w) before += s_eq[v];
      ties += s_eq[v];
    }
    const bool kept = i < end && (k > hi || (in && (whole || before + __popcll(eq & ((1ull << lane) - 1)) < need)));
    const u64 gt = __ballot(kept);
    if (lane == 0) s_gt[w] = __popcll(gt);
    __syncthreads();
    int at = done;
    for (int v = 0; v < kWaves; ++v) {
      if (v < w) at += s_gt[v];
      done += s_gt[v];
    }
    if (kept) out[at + __popcll(gt & ((1ull << lane) - 1))] = i;
  }
}

}  // namespace

extern "C" int dgi_select_pages(const void* q, long long q_stride, const void* bounds, const int* tables, int table_stride, int table_cols,
                                int n_seqs, int num_blocks, const int* ctx, const int* row_seq, int T, int nh, int nkv, int hd, int page,
                                int count, int first, int recent, void* keys, int key_stride, int* out, hipStream_t s) {
  if (T == 0) return 0;
  const Args a{(const uint16_t*)q, q_stride, (const uint16_t*)bounds, tables, table_stride, table_cols, n_seqs, num_blocks, ctx, row_seq,
               T, nh, nkv, page, count, first, recent, (u64*)keys, key_stride, out};
  if (table_cols > count) {
    const int chunk = 256;
    const dim3 grid(nkv * T, (table_cols - first - recent + chunk - 1) / chunk);
    if (hd == 64) page_scores_kernel<64><<<grid, kThreads, 0, s>>>(a, chunk);
    else if (hd == 128) page_scores_kernel<128><<<grid, kThreads, 0, s>>>(a, chunk);
    else if (hd == 256) page_scores_kernel<256><<<grid, kThreads, 0, s>>>(a, chunk);
    else return -5;
    DGI_CHECK_LAUNCH();
  }
  pick_pages_kernel<<<nkv * T, kThreads, 0, s>>>(a);
  DGI_CHECK_LAUNCH();
  return 0;
}
