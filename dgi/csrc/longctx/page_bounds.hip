// dgi/csrc/longctx/page_bounds.hip — the least and largest key of every channel of a page ("bounds"), kept by the append that rotates
// and writes a step's keys, and rebuilt from the keys of pages that came by another way.
//
// bounds [num_blocks, n_kv, 2, head_dim] bf16: row 0 the least, row 1 the largest cached value of a channel.  A minimum rounds
// nothing, so they are exact whatever the order, and a page's bounds can go on from step to step.  A value that is no number makes its
// channel's bounds no number (minimum / maximum of IEEE 754-2019).
//
// Bound by bytes: the append reads a row's q | k | v once and writes it once (4115 rows of 64 heads on 8 of 128, 172 MB: 45 us, 3.8 TB/s;
// one row: 4.0 us, a launch), the rebuilding reads the keys once (16384 pages of 16 keys, 8 heads of 128, 604 MB: 132 us, 4.6 TB/s, where a
// kernel that only reads reaches 6.4).
#include "../common.h"
#include "page_runs.h"

using namespace dgi;

namespace {

// the halves of eight bf16 that go into a running minimum / maximum, in fp32 (exact)
__device__ __forceinline__ void widen8(float* lo, float* hi, const float* x) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo[j] = __builtin_elementwise_minimum(lo[j], x[j]);
    hi[j] = __builtin_elementwise_maximum(hi[j], x[j]);
  }
}

constexpr int kThreads = 256, kWaves = kThreads / 64;

// A head's dims as tasks of one lane: a pair of 16-byte chunks that rotate with each other (mode 0: dims i and i + rd / 2), a chunk
// that rotates in itself (mode 1: dims 2 i and 2 i + 1), or one behind the rotated dims that stays.
struct Task {
  int at, other;      // dims of the chunk and of the one that it rotates with (-1: none)
  bool turns;
  float c[8], s[8];   // cos and sin; mode 1: four of them
};
__device__ __forceinline__ int tasks_of(int hd, int rd, int mode) { return (mode == 0 ? rd >> 4 : rd >> 3) + ((hd - rd) >> 3); }
__device__ __forceinline__ Task task_of(int i, int rd, int mode) {
  const int turning = mode == 0 ? rd >> 4 : rd >> 3;
  Task x;
  x.turns = i < turning;
  x.at = x.turns ? i * 8 : rd + (i - turning) * 8;
  x.other = x.turns && mode == 0 ? x.at + (rd >> 1) : -1;
  return x;
}
__device__ __forceinline__ void angles(Task& x, const float* __restrict__ cs, int rd, int mode) {
  if (!x.turns) return;
  const float *c = cs + (mode == 0 ? x.at : x.at >> 1), *s = c + (rd >> 1);
#pragma unroll
  for (int j = 0; j < 8; j += 4) {
    if (mode == 1 && j) break;
    *reinterpret_cast<float4*>(x.c + j) = *reinterpret_cast<const float4*>(c + j);
    *reinterpret_cast<float4*>(x.s + j) = *reinterpret_cast<const float4*>(s + j);
  }
}
// a (and b, the chunk it rotates with) turned
__device__ __forceinline__ void turn(const Task& x, u32x4& a, u32x4& b) {
  if (!x.turns) return;
  float p[8], q[8], u[8], v[8];
  unpack8(a, p);
  if (x.other >= 0) {
    unpack8(b, q);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = p[j] * x.c[j] - q[j] * x.s[j];
      v[j] = q[j] * x.c[j] + p[j] * x.s[j];
    }
    b = pack8(v);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[2 * j] = p[2 * j] * x.c[j] - p[2 * j + 1] * x.s[j];
      u[2 * j + 1] = p[2 * j + 1] * x.c[j] + p[2 * j] * x.s[j];
    }
  }
  a = pack8(u);
}

// The first T workgroups are for the keys, the others for queries and values of a row.
//
// A row that is the first of the step in its page takes the keys of all rows of the page (page_runs.h) and its bounds, so that
// every page has one writer; its waves take a row each in turn, the same task of a row each lane, and are joined in LDS.  The workgroups of
// the rows behind it end at once.
//
// A lane has the same task of every head that it takes, and so one read of the angles.
__global__ __launch_bounds__(kThreads) void rope_cache_bounds_kernel(
    const uint16_t* __restrict__ qkv, long long ld, int T, const int* __restrict__ positions, int max_pos,
    const float* __restrict__ cos_sin, int nh, int nkv, int hd, int rd, int mode, const int* __restrict__ slots, long long n_slots,
    uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_cache, uint16_t* __restrict__ v_cache, uint16_t* __restrict__ bounds,
    int block_size) {
  const bool keys = blockIdx.x < T;
  const int t = keys ? blockIdx.x : blockIdx.x - T, tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  const int tasks = tasks_of(hd, rd, mode), slot = slots[t];
  const bool cached = has_slot(slot, n_slots);
  const int blk = cached ? slot / block_size : 0, off = cached ? slot - blk * block_size : 0;
  auto angles_at = [&](int row) { return cos_sin + (size_t)min(max(positions[row], 0), max_pos - 1) * rd; };

  if (!keys) {
    const uint16_t* row = qkv + t * ld;
    const int side = kThreads / tasks;      // heads at a time
    Task x = task_of(tid % tasks, rd, mode);
    if (tid < side * tasks) {
      angles(x, angles_at(t), rd, mode);
#pragma unroll 4
      for (int head = tid / tasks; head < nh; head += side) {
        const uint16_t* qp = row + head * hd;
        uint16_t* op = q_out + ((size_t)t * nh + head) * hd;
        u32x4 a = *reinterpret_cast<const u32x4*>(qp + x.at), b = *reinterpret_cast<const u32x4*>(qp + max(x.other, 0));
        turn(x, a, b);
        *reinterpret_cast<u32x4*>(op + x.at) = a;
        if (x.other >= 0) *reinterpret_cast<u32x4*>(op + x.other) = b;
      }
    }
    if (cached)
      for (int it = tid; it < nkv * (hd >> 3); it += kThreads) {
        const int h = it / (hd >> 3), c = it - h * (hd >> 3);
        *reinterpret_cast<u32x4*>(v_cache + (((size_t)blk * nkv + h) * block_size + off) * hd + c * 8) =
            *reinterpret_cast<const u32x4*>(row + (size_t)(nh + nkv + h) * hd + c * 8);
      }
    return;
  }

  if (!cached) return;
  auto ballot = [&](auto f) { return (unsigned long long)__ballot(f(lane)); };
  if (!begins_page(ballot, slots, n_slots, block_size, t, slot - off)) return;
  const PageRows run = page_rows(ballot, slots, n_slots, block_size, T, t, slot - off);
  __shared__ __attribute__((aligned(16))) u32x4 part[4][kWaves][64];
  for (int base = 0; base < nkv * tasks; base += 64) {
    const int it = base + lane;
    const bool live = it < nkv * tasks;
    const int h = live ? it / tasks : 0;
    Task x = task_of(live ? it - h * tasks : 0, rd, mode);
    float lo[2][8], hi[2][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[0][j] = lo[1][j] = __builtin_inff();
      hi[0][j] = hi[1][j] = -__builtin_inff();
    }
    if (live)
#pragma unroll 2
      for (int r = w; r < run.rows; r += kWaves) {
        const uint16_t* kp = qkv + (t + r) * ld + (nh + h) * hd;
        const int at = run.plain ? slot + r : slots[t + r];
        u32x4 a = *reinterpret_cast<const u32x4*>(kp + x.at), b = *reinterpret_cast<const u32x4*>(kp + max(x.other, 0));
        angles(x, angles_at(t + r), rd, mode);
        if (!run.plain && !has_slot(at, n_slots)) continue;
        uint16_t* op = k_cache + (((size_t)blk * nkv + h) * block_size + (at - (slot - off))) * hd;
        turn(x, a, b);
        float v[8];      // what attention will read
        *reinterpret_cast<u32x4*>(op + x.at) = a;
        unpack8(a, v);
        widen8(lo[0], hi[0], v);
        if (x.other >= 0) {
          *reinterpret_cast<u32x4*>(op + x.other) = b;
          unpack8(b, v);
          widen8(lo[1], hi[1], v);
        }
      }
    part[0][w][lane] = pack8(lo[0]);      // exact: the values are bf16
    part[1][w][lane] = pack8(hi[0]);
    part[2][w][lane] = pack8(lo[1]);
    part[3][w][lane] = pack8(hi[1]);
    __syncthreads();
    // wave w: the least (w even) or largest of the task's first or second chunk
    const int at = w < 2 ? x.at : x.other;
    if (live && at >= 0) {
      uint16_t* bp = bounds + (((size_t)blk * nkv + h) * 2 + (w & 1)) * hd + at;
      float m[8], v[8];
      unpack8(part[w][0][lane], m);
      auto join = [&](const u32x4& from) {
        unpack8(from, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m[j] = w & 1 ? __builtin_elementwise_maximum(m[j], v[j]) : __builtin_elementwise_minimum(m[j], v[j]);
      };
#pragma unroll
      for (int i = 1; i < kWaves; ++i) join(part[w][i][lane]);
      if (off > 0) join(*reinterpret_cast<const u32x4*>(bp));
      *reinterpret_cast<u32x4*>(bp) = pack8(m);
    }
    __syncthreads();
  }
}

// A wave per (page, kv head): CH lanes take a key, 64 / CH keys at a time.
template <int HD>
__global__ __launch_bounds__(kThreads) void page_bounds_kernel(const uint16_t* __restrict__ k_cache, uint16_t* __restrict__ bounds,
                                                               const int* __restrict__ pages, const int* __restrict__ lens, long long items,
                                                               int num_blocks, int nkv, int block_size) {
  constexpr int CH = HD / 8, R = 64 / CH;
  const long long item = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6);
  if (item >= items) return;
  const int i = (int)(item / nkv), h = (int)(item - (long long)i * nkv);
  const int page = pages[i];
  if (page < 0 || page >= num_blocks) return;
  const int n = min(max(lens[i], 0), block_size);
  const int lane = threadIdx.x & 63, c = lane % CH, r0 = lane / CH;
  const uint16_t* kp = k_cache + ((size_t)page * nkv + h) * block_size * HD + c * 8;
  float lo[8], hi[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    lo[j] = __builtin_inff();
    hi[j] = -__builtin_inff();
  }
  for (int r = r0; r < n; r += R) {
    float x[8];
    unpack8(*reinterpret_cast<const u32x4*>(kp + (size_t)r * HD), x);
    widen8(lo, hi, x);
  }
#pragma unroll
  for (int o = CH; o < 64; o <<= 1)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = __builtin_elementwise_minimum(lo[j], __shfl_xor(lo[j], o, 64));
      hi[j] = __builtin_elementwise_maximum(hi[j], __shfl_xor(hi[j], o, 64));
    }
  uint16_t* bp = bounds + ((size_t)page * nkv + h) * 2 * HD + c * 8;
  if (r0 == 0) *reinterpret_cast<u32x4*>(bp) = pack8(lo);
  if (r0 == 1) *reinterpret_cast<u32x4*>(bp + HD) = pack8(hi);
}

}  // namespace

extern "C" int dgi_rope_cache_bounds(const void* qkv, long long ld, int T, const int* positions, int max_pos, const float* cos_sin, int nh,
                                     int nkv, int hd, int rd, int mode, const int* slots, long long n_slots, void* q_out, void* k_cache,
                                     void* v_cache, void* bounds, int block_size, hipStream_t s) {
  if (T == 0) return 0;
  rope_cache_bounds_kernel<<<2 * T, kThreads, 0, s>>>((const uint16_t*)qkv, ld, T, positions, max_pos, cos_sin, nh, nkv, hd, rd, mode, slots,
                                                  n_slots, (uint16_t*)q_out, (uint16_t*)k_cache, (uint16_t*)v_cache, (uint16_t*)bounds,
                                                  block_size);
  DGI_CHECK_LAUNCH();
  return 0;
}

extern "C" int dgi_page_bounds(const void* k_cache, void* bounds, const int* pages, const int* lens, int n, int num_blocks, int nkv, int hd,
                               int block_size, hipStream_t s) {
  const long long items = (long long)n * nkv;
  if (items == 0) return 0;
  const dim3 grid((unsigned)((items + kWaves - 1) / kWaves));
  auto launch = [&](auto kernel) {
    kernel<<<grid, kThreads, 0, s>>>((const uint16_t*)k_cache, (uint16_t*)bounds, pages, lens, items, num_blocks, nkv, block_size);
  };
  if (hd == 64) launch(page_bounds_kernel<64>);
  else if (hd == 128) launch(page_bounds_kernel<128>);
  else if (hd == 256) launch(page_bounds_kernel<256>);
  else return -5;
  DGI_CHECK_LAUNCH();
  return 0;
}
