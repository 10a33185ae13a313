// dgi/csrc/longctx/page_bounds.hip — the least and largest key of every channel of a page ("bounds"), kept by the append that rotates
// and writes a step's keys, and rebuilt from the keys of pages that came by another way.
//
// bounds [num_blocks, n_kv, 2, head_dim] bf16: row 0 the least, row 1 the largest cached value of a channel.  A minimum rounds
// nothing, so they are exact whatever the order, and a page's bounds can go on from step to step.  A value that is no number makes its
// channel's bounds no number (minimum / maximum of IEEE 754-2019).
//
// Bound by bytes: the append reads a row's q | k | v once and writes it once, the rebuilding reads the keys once.
#include "../common.h"

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

// Chunk c (8 dims) of a head at `hp`, rotated by the row's [cos | sin] at cs: the pairs of mode 0 are (i, i + rd / 2), of mode 1
// (2 i, 2 i + 1); chunks beyond the rotated dims pass through.
__device__ __forceinline__ void rotated_chunk(const uint16_t* __restrict__ hp, int c, const float* __restrict__ cs, int rd, int mode, float* o) {
  float a[8];
  unpack8(*reinterpret_cast<const u32x4*>(hp + c * 8), a);
  if (c * 8 >= rd) {
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = a[j];
    return;
  }
  const int half = rd >> 1;
  if (mode == 0) {
    const bool second = c * 8 >= half;
    const int p = second ? c * 8 - half : c * 8;
    float b[8], cv[8], sv[8];
    unpack8(*reinterpret_cast<const u32x4*>(hp + (second ? p : p + half)), b);
    *reinterpret_cast<float4*>(cv) = *reinterpret_cast<const float4*>(cs + p);
    *reinterpret_cast<float4*>(cv + 4) = *reinterpret_cast<const float4*>(cs + p + 4);
    *reinterpret_cast<float4*>(sv) = *reinterpret_cast<const float4*>(cs + half + p);
    *reinterpret_cast<float4*>(sv + 4) = *reinterpret_cast<const float4*>(cs + half + p + 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = second ? a[j] * cv[j] + b[j] * sv[j] : a[j] * cv[j] - b[j] * sv[j];
  } else {
    const float4 cv = *reinterpret_cast<const float4*>(cs + c * 4);
    const float4 sv = *reinterpret_cast<const float4*>(cs + half + c * 4);
    const float cc[4] = {cv.x, cv.y, cv.z, cv.w}, ss[4] = {sv.x, sv.y, sv.z, sv.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      o[2 * j] = a[2 * j] * cc[j] - a[2 * j + 1] * ss[j];
      o[2 * j + 1] = a[2 * j + 1] * cc[j] + a[2 * j] * ss[j];
    }
  }
}

// A workgroup per row: its queries and values, and, where the row is the first of the step in its page, the keys and bounds of all
// rows that follow it there (rows of rising slots, one page's side by side: at most a page of them).  So every page has one writer.
__global__ __launch_bounds__(kThreads) void rope_cache_bounds_kernel(
    const uint16_t* __restrict__ qkv, long long ld, int T, const int* __restrict__ positions, int max_pos,
    const float* __restrict__ cos_sin, int nh, int nkv, int hd, int rd, int mode, const int* __restrict__ slots, long long n_slots,
    uint16_t* __restrict__ q_out, uint16_t* __restrict__ k_cache, uint16_t* __restrict__ v_cache, uint16_t* __restrict__ bounds,
    int block_size) {
  const int t = blockIdx.x, tid = threadIdx.x;
  const int chunks = hd >> 3;
  const uint16_t* row = qkv + t * ld;
  const float* cs = cos_sin + (size_t)min(max(positions[t], 0), max_pos - 1) * rd;
  const int slot = slots[t];
  const bool cached = slot >= 0 && slot < n_slots;
  const int blk = cached ? slot / block_size : 0, off = cached ? slot - blk * block_size : 0;

  for (int it = tid; it < (nh + nkv) * chunks; it += kThreads) {
    const int head = it / chunks, c = it - head * chunks;
    if (head < nh) {
      float o[8];
      rotated_chunk(row + head * hd, c, cs, rd, mode, o);
      *reinterpret_cast<u32x4*>(q_out + ((size_t)t * nh + head) * hd + c * 8) = pack8(o);
    } else if (cached) {
      const int h = head - nh;
      *reinterpret_cast<u32x4*>(v_cache + (((size_t)blk * nkv + h) * block_size + off) * hd + c * 8) =
          *reinterpret_cast<const u32x4*>(row + (size_t)(nh + nkv + h) * hd + c * 8);
    }
  }

  if (!cached || (off > 0 && t > 0 && slots[t - 1] == slot - 1)) return;      // the whole workgroup: no keys of its own
  int run = 1;
  while (off + run < block_size && t + run < T && slots[t + run] == slot + run) ++run;

  __shared__ __attribute__((aligned(16))) u32x4 part[2][kWaves][64];
  const int w = tid >> 6, lane = tid & 63;
  for (int base = 0; base < nkv * chunks; base += 64) {
    const int it = base + lane;
    const bool live = it < nkv * chunks;
    const int h = live ? it / chunks : 0, c = live ? it - h * chunks : 0;
    float lo[8], hi[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      lo[j] = __builtin_inff();
      hi[j] = -__builtin_inff();
    }
    if (live)
      for (int r = w; r < run; r += kWaves) {
        const float* csr = cos_sin + (size_t)min(max(positions[t + r], 0), max_pos - 1) * rd;
        float o[8], x[8];
        rotated_chunk(qkv + (t + r) * ld + (nh + h) * hd, c, csr, rd, mode, o);
        const u32x4 k = pack8(o);
        *reinterpret_cast<u32x4*>(k_cache + (((size_t)blk * nkv + h) * block_size + off + r) * hd + c * 8) = k;
        unpack8(k, x);      // what attention will read
        widen8(lo, hi, x);
      }
    part[0][w][lane] = pack8(lo);      // exact: the values are bf16
    part[1][w][lane] = pack8(hi);
    __syncthreads();
    if (w == 0 && live) {
      uint16_t* bp = bounds + ((size_t)blk * nkv + h) * 2 * hd + c * 8;
#pragma unroll
      for (int v = 1; v < kWaves; ++v) {
        float x[8], y[8];
        unpack8(part[0][v][lane], x);
        unpack8(part[1][v][lane], y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          lo[j] = __builtin_elementwise_minimum(lo[j], x[j]);
          hi[j] = __builtin_elementwise_maximum(hi[j], y[j]);
        }
      }
      if (off > 0) {
        float x[8], y[8];
        unpack8(*reinterpret_cast<const u32x4*>(bp), x);
        unpack8(*reinterpret_cast<const u32x4*>(bp + hd), y);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          lo[j] = __builtin_elementwise_minimum(lo[j], x[j]);
          hi[j] = __builtin_elementwise_maximum(hi[j], y[j]);
        }
      }
      *reinterpret_cast<u32x4*>(bp) = pack8(lo);
      *reinterpret_cast<u32x4*>(bp + hd) = pack8(hi);
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
  rope_cache_bounds_kernel<<<T, kThreads, 0, s>>>((const uint16_t*)qkv, ld, T, positions, max_pos, cos_sin, nh, nkv, hd, rd, mode, slots,
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
