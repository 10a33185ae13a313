// dgi/csrc/longctx/tree_rows.hip — attention of drafted trees of few (node, head) pairs over a paged cache.
//
// 16 pairs of a sequence's nodes and a kv head's group are the columns of one product (tree_tiles.hip has 128 of them).  A
// workgroup owns them and a run of keys; its waves take tiles of 32 keys in turn and are merged through LDS, runs of one sequence by a
// second launch.  Scores are formed transposed, S^T = K Q^T, so that a lane owns a query column and the weights stay in the registers
// that the product O^T += V^T P^T takes them from; keys and values go through LDS, whole rows a load, a tile under way while the one
// before is multiplied.  Weights are rounded to bf16 for that product (as the cached values are; their sum is taken before),
// everything else is fp32.
//
// Bound by the cache's bytes where contexts are long: 32 sequences of 4000 keys, 8 nodes, 32 heads on 8, 100 us, 5.3 TB/s.  A short one is
// a chain of round trips (lengths, then page ids beside the queries, then keys and values) and two launches: one sequence of 600 keys 10 us.
// 32 columns a workgroup, which read the keys once for two groups of columns, take 108 and 13: twice the sums leave one wave a SIMD.
#include "../common.h"

#include <type_traits>

using namespace dgi;

namespace {

constexpr int kList = 512;      // pages of a list in LDS at a time
constexpr int NW = 4, NT = 64 * NW;

struct Args {
  const uint16_t* q;
  long long q_stride;
  const uint16_t* k;
  const uint16_t* v;
  const int* tables;
  int table_stride, table_cols, n_seqs, num_blocks, rows;
  const int* ctx;
  uint16_t* out;
  long long out_stride;
  float* part_o;      // [item][kv head][run][16][HD] of normalised sums, [item][kv head][run][16] of their log2 sums
  float* part_l;
  int splits, nh, nkv, bs_log2;
  float scale_log2;
  const int* cu;
  const unsigned long long* mask;
  int mask_stride, max_nodes, min_part;
};

// Where 16-byte chunk ch of a row lies in LDS: keys are read 16 rows at one chunk, values transposed.
template <int HD>
__device__ __forceinline__ int k_lds_off(int row, int ch) { return row * HD + ((ch ^ (HD == 64 ? row >> 1 & 7 : row & 15)) << 3); }
template <int HD>
__device__ __forceinline__ int v_lds_chunk(int row, int ch) { return row * HD + ((ch ^ (((row & 7) << 1) & (HD / 8 - 1))) << 3); }
template <int HD>
__device__ __forceinline__ int v_lds_off(int row, int col) { return v_lds_chunk<HD>(row, col >> 3) + (col & 7); }

template <int HD>
constexpr int wave_lds() { return 64 * HD; }      // a tile of rows (32 x HD bf16), then 16 rows of sums (fp32)

// A sequence's runs of keys: as many as there are places for, of min_part keys at least, each a multiple of 32 keys and of a page.
struct Runs {
  int row0, nodes, ctx, part, runs;
};
__device__ __forceinline__ Runs runs_of(const Args& a, int seq) {
  const int q0 = a.cu[seq], q1 = a.cu[seq + 1], c = a.ctx[seq];
  Runs r;
  r.row0 = q0;
  r.nodes = q0 < 0 ? 0 : min(min(q1, a.rows) - q0, a.max_nodes);
  r.ctx = min(max(c, 0), a.table_cols << a.bs_log2);
  const int n = max(1, min(a.splits, (r.ctx + a.min_part - 1) / a.min_part)), unit = max(32, 1 << a.bs_log2);
  r.part = max(unit, (((r.ctx + n - 1) / n) + unit - 1) / unit * unit);
  r.runs = max(1, (r.ctx + r.part - 1) / r.part);
  return r;
}

// WIDE: pages of 16 keys and more, so that 16 keys of a tile lie side by side.
template <int HD, bool WIDE>
__global__ __launch_bounds__(NT) void tree_rows_kernel(Args a) {
  constexpr int KS = HD / 32, NC = HD / 16, VCH = HD / 8;
  __shared__ __attribute__((aligned(16))) char smem[NW * wave_lds<HD>()];
  __shared__ int list[kList];      // pages; -1: not in the cache
  __shared__ float ml[NW][2][16];

  // the column tiles of a (run, sequence, kv head) eight workgroups apart: on one XCD, whose L2 has the keys after the first
  const int G = a.nh / a.nkv, tiles = (a.max_nodes * G + 15) / 16;
  const int eight = blockIdx.x / (8 * tiles), tile_at = blockIdx.x - eight * 8 * tiles, unit = eight * 8 + tile_at % 8;
  if (unit >= a.nkv * a.n_seqs * a.splits) return;
  const int h = unit % a.nkv, seq = unit / a.nkv % a.n_seqs, split = unit / a.nkv / a.n_seqs, item = seq * tiles + tile_at / 8;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int bs = 1 << a.bs_log2;
  const Runs run = runs_of(a, seq);
  const int pair0 = (item - seq * tiles) * 16;      // (node, head) pairs from here on
  if (pair0 >= run.nodes * G || split >= run.runs) return;
  const int ctx = run.ctx, lo = split * run.part, hi = min(lo + run.part, ctx), tree_key = ctx - run.nodes;      // the key of node 0
  const int* table = a.tables + (size_t)seq * a.table_stride;
  uint16_t* vt = reinterpret_cast<uint16_t*>(smem + w * wave_lds<HD>());

  // queries: column qi; fragments of the second operand, dims 32 s + 8 g ..
  u32x4 qf[KS];
  const int pair = pair0 + qi, node_q = pair / G, head_q = h * G + pair - node_q * G;
  const bool live = node_q < run.nodes;
  const uint16_t* qp = a.q + (size_t)(run.row0 + (live ? node_q : 0)) * a.q_stride + (live ? head_q : 0) * HD + 8 * g;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = live ? *reinterpret_cast<const u32x4*>(qp + 32 * s) : u32x4{0, 0, 0, 0};
  const unsigned long long bits = live ? a.mask[(size_t)seq * a.mask_stride + node_q] : 0;
  // where the lane's chunk of row i 64 / VCH + lane / VCH goes in LDS: the same for every P-th i, but for whole rows
  constexpr int P = VCH / 4;      // 16 rows
  int k_at[P], v_at[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    k_at[i] = k_lds_off<HD>(i * (64 / VCH) + lane / VCH, lane % VCH);
    v_at[i] = v_lds_chunk<HD>(i * (64 / VCH) + lane / VCH, lane % VCH);
  }

  float m_run = -__builtin_inff(), l_run = 0.f;
  f32x4 o[NC];
#pragma unroll
  for (int c = 0; c < NC; ++c) o[c] = f32x4{0, 0, 0, 0};

  const int per = kList << a.bs_log2;
  for (int at = lo; at < hi; at += per) {
    const int keys = min(per, hi - at), entries = (keys + bs - 1) >> a.bs_log2, ntiles = (keys + 31) >> 5;
    __syncthreads();
    for (int e = tid; e < entries; e += NT) {
      const int id = table[(at >> a.bs_log2) + e];
      list[e] = id >= 0 && id < a.num_blocks ? id : -1;
    }
    __syncthreads();
    u32x4 kr[VCH / 2], vr[VCH / 2];
    // a key's row in the cache, of page 0 if it has no page; whether it has one
    auto row_of = [&](int tok, bool& there) {
      const int id = list[min(tok >> a.bs_log2, entries - 1)];
      there = id >= 0 && tok < keys;
      return (((size_t)max(id, 0) * a.nkv + h) << a.bs_log2) + (tok & (bs - 1));
    };
    struct Half {
      size_t row;
      bool there;
    };
    auto half = [&](int t, int u) {      // WIDE: in scalar registers
      bool there;
      const size_t r = row_of(32 * t + 16 * u, there);
      return Half{((size_t)__builtin_amdgcn_readfirstlane((int)(r >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)r),
                  (bool)__builtin_amdgcn_readfirstlane((int)there)};
    };
    // a tile's rows, whole lines a load
    auto load = [&](int t, const Half* x, const uint16_t* cache, u32x4* to) {
      constexpr int R = 64 / VCH;      // rows a load
#pragma unroll
      for (int i = 0; i < VCH / 2; ++i) {
        bool there;
        to[i] = *reinterpret_cast<const u32x4*>(WIDE ? cache + x[i * R / 16].row * HD + (i * R % 16 * HD + lane * 8)
                                                     : cache + row_of(32 * t + i * R + lane / VCH, there) * HD + lane % VCH * 8);
      }
    };
    auto stage = [&](const u32x4* from, const int* to) {      // into LDS, behind the reads of what was there
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < VCH / 2; ++i) *reinterpret_cast<u32x4*>(vt + to[i % P] + i / P * (64 / VCH * P * HD)) = from[i];
    };
    auto tile = [&](int t, const Half* now, const Half* next, auto LAST) {
      constexpr int R = 64 / VCH;
      stage(kr, k_at);
      if constexpr (!LAST.value) {
        __builtin_amdgcn_sched_barrier(0);
        load(t + NW, next, a.k, kr);
        __builtin_amdgcn_sched_barrier(0);
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      f32x4 sc[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        sc[u] = f32x4{0, 0, 0, 0};
#pragma unroll
        for (int s = 0; s < KS; ++s)
          sc[u] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(*reinterpret_cast<const u32x4*>(vt + k_lds_off<HD>(16 * u + qi, 4 * s + g))),
                                                          as_bf16x8(qf[s]), sc[u], 0, 0, 0);
      }
      const int key0 = at + 32 * t;      // the tile's first key
      // every key is there and before the tree: seen by all
      const bool full = WIDE && now[0].there && now[1].there && key0 + 32 <= min(hi, tree_key);
      unsigned odd = 0;
      if (!full) {
        // Values of keys that are not there are zeros.  Values of the tree's keys that are infinite or no numbers reach the rows that see
        // them alone, but zero times such a value is no number: they are taken out here and added below for the rows that see them.
#pragma unroll
        for (int i = 0; i < VCH / 2; ++i) {
          const int tok = 32 * t + i * R + lane / VCH;
          bool there = WIDE && now[i * R / 16].there && tok < keys;
          if (!WIDE) row_of(tok, there);
          bool is = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (!there) vr[i][j] = 0;
            const bool lo_odd = (vr[i][j] & 0x7f80u) == 0x7f80u, hi_odd = (vr[i][j] & 0x7f800000u) == 0x7f800000u;
            is = is || lo_odd || hi_odd;
            vr[i][j] &= (lo_odd ? 0xffff0000u : ~0u) & (hi_odd ? 0xffffu : ~0u);
          }
          const unsigned long long b = __ballot(is);
#pragma unroll
          for (int j = 0; j < R; ++j) odd |= (b >> (j * VCH) & ((1ull << VCH) - 1)) ? 1u << (i * R + j) : 0u;
        }
      }
      stage(vr, v_at);
      if constexpr (!LAST.value) {
        __builtin_amdgcn_sched_barrier(0);
        load(t + NW, next, a.v, vr);
        __builtin_amdgcn_sched_barrier(0);
      }
      // ---- online softmax; the lane's keys are 16 u + 4 g + i
      float x[2][4], mx = -__builtin_inff();
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          x[u][i] = sc[u][i] * a.scale_log2;
          if (!full) {
            const int tok = 32 * t + 16 * u + 4 * g + i, node = at + tok - tree_key;
            bool there = WIDE && now[u].there && tok < keys;
            if (!WIDE) row_of(tok, there);
            if (!there || !(node < 0 || (bits >> (node & 63) & 1))) x[u][i] = -__builtin_inff();
          }
          mx = fmaxf(mx, x[u][i]);
        }
      // the sums are scaled anew only where a maximum grows by more than 8 (weights stay below 2^8), and there the four lanes of a
      // column agree on it
      if (__any(mx > m_run + 8.f)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run, mx);
        const float alpha = m_new == -__builtin_inff() ? 0.f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[c] *= alpha;
        m_run = m_new;
      }
      const float m_use = m_run == -__builtin_inff() ? 0.f : m_run;
      float p[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) p[u][i] = __builtin_amdgcn_exp2f(x[u][i] - m_use);
      l_run += ((p[0][0] + p[0][1]) + (p[0][2] + p[0][3])) + ((p[1][0] + p[1][1]) + (p[1][2] + p[1][3]));
      const u32x4 pf = {pack_bf16x2(p[0][0], p[0][1]), pack_bf16x2(p[0][2], p[0][3]), pack_bf16x2(p[1][0], p[1][1]),
                        pack_bf16x2(p[1][2], p[1][3])};
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_wave_barrier();
      const int tq = qi >> 2, tp = qi & 3;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const short4v a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vt + v_lds_off<HD>(4 * g + tq, 16 * c + 4 * tp)));
        const short4v a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(vt + v_lds_off<HD>(16 + 4 * g + tq, 16 * c + 4 * tp)));
        u32x4 vf;
        vf[0] = (uint32_t)(uint16_t)a0[0] | ((uint32_t)(uint16_t)a0[1] << 16);
        vf[1] = (uint32_t)(uint16_t)a0[2] | ((uint32_t)(uint16_t)a0[3] << 16);
        vf[2] = (uint32_t)(uint16_t)a1[0] | ((uint32_t)(uint16_t)a1[1] << 16);
        vf[3] = (uint32_t)(uint16_t)a1[2] | ((uint32_t)(uint16_t)a1[3] << 16);
        o[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(vf), as_bf16x8(pf), o[c], 0, 0, 0);
      }
      for (; odd; odd &= odd - 1) {      // what was taken out: key kk of the tile
        const int kk = __ffs(odd) - 1, j = (kk >> 4) * 4 + (kk & 3);
        bool there;
        const uint16_t* vp = a.v + row_of(32 * t + kk, there) * HD + 4 * g;
        const uint32_t two = __shfl(j & 4 ? (j & 2 ? pf[3] : pf[2]) : (j & 2 ? pf[1] : pf[0]), 16 * (kk >> 2 & 3) + qi, 64);
        const float p = __uint_as_float(j & 1 ? two & 0xffff0000u : two << 16);
        const int node = at + 32 * t + kk - tree_key;
        const bool sees = node < 0 || (bits >> node & 1);
#pragma unroll
        for (int c = 0; c < NC; ++c)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint16_t x = vp[16 * c + i];
            if (sees && (x & 0x7f80) == 0x7f80) o[c][i] += p * bf16_to_f32(x);
          }
      }
    };
    if (w < ntiles) {
      Half now[2], next[2];
      auto find = [&](Half* x, int t) {
        if constexpr (WIDE) {
          x[0] = half(t, 0);
          x[1] = half(t, 1);
        }
      };
      find(now, w);
      load(w, now, a.k, kr);
      load(w, now, a.v, vr);
      int t = w;
      for (; t + NW < ntiles; t += NW) {
        find(next, t + NW);
        tile(t, now, next, std::false_type{});
        now[0] = next[0];
        now[1] = next[1];
      }
      tile(t, now, next, std::true_type{});
    }
  }

  // ---- the waves' results: HD / 4 threads a column
  l_run += __shfl_xor(l_run, 16, 64);
  l_run += __shfl_xor(l_run, 32, 64);
  __syncthreads();
  f32x4* ow = reinterpret_cast<f32x4*>(smem + w * wave_lds<HD>());
#pragma unroll
  for (int c = 0; c < NC; ++c) ow[qi * (HD / 4) + ((4 * c + g) ^ (qi & 7))] = o[c];
  if (g == 0) {
    ml[w][0][qi] = m_run;
    ml[w][1][qi] = l_run;
  }
  __syncthreads();
  for (int idx = tid; idx < 16 * (HD / 4); idx += NT) {
    const int col = idx / (HD / 4), d = idx - col * (HD / 4), r = pair0 + col, node = r / G;
    if (node >= run.nodes) continue;
    float M = -__builtin_inff();
#pragma unroll
    for (int v = 0; v < NW; ++v) M = fmaxf(M, ml[v][0][col]);
    const float use = M == -__builtin_inff() ? 0.f : M;
    float L = 0.f;
    f32x4 acc = {0, 0, 0, 0};
#pragma unroll
    for (int v = 0; v < NW; ++v) {
      const float sc = __builtin_amdgcn_exp2f(ml[v][0][col] - use);
      L += ml[v][1][col] * sc;
      acc += reinterpret_cast<f32x4*>(smem + v * wave_lds<HD>())[col * (HD / 4) + (d ^ (col & 7))] * sc;
    }
    if (L != 0.f) acc /= L;
    else acc = f32x4{0, 0, 0, 0};
    if (run.runs == 1) {
      uint2 x;
      x.x = pack_bf16x2(acc[0], acc[1]);
      x.y = pack_bf16x2(acc[2], acc[3]);
      *reinterpret_cast<uint2*>(a.out + (size_t)(run.row0 + node) * a.out_stride + (h * G + r - node * G) * HD + 4 * d) = x;
    } else {
      const size_t slab = (((size_t)item * a.nkv + h) * a.splits + split) * 16 + col;
      *reinterpret_cast<f32x4*>(a.part_o + slab * HD + 4 * d) = acc;
      if (d == 0) a.part_l[slab] = L == 0.f ? -__builtin_inff() : M + __builtin_amdgcn_logf(L);
    }
  }
}

// Runs of the same columns, weighed by their sums: HD / 4 threads a column.
template <int HD>
__global__ __launch_bounds__(256) void tree_rows_runs_kernel(Args a) {
  constexpr int L = HD / 4, U = 8;
  const int item = blockIdx.x / a.nkv, h = blockIdx.x - item * a.nkv, col = blockIdx.y * (256 / L) + threadIdx.x / L, d = threadIdx.x % L * 4;
  const int G = a.nh / a.nkv, tiles = (a.max_nodes * G + 15) / 16, seq = item / tiles;
  const int r = (item - seq * tiles) * 16 + col, node = r / G;
  const Runs run = runs_of(a, seq);
  if (node >= run.nodes || run.runs == 1) return;
  const size_t base = ((size_t)item * a.nkv + h) * a.splits * 16 + col;
  float M = -__builtin_inff(), W = 0.f;
  f32x4 acc = {0, 0, 0, 0};
  for (int s = 0; s < run.runs; s += U) {
    float l[U], top = M;
    bool any = false;
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t at = base + (size_t)min(s + u, run.runs - 1) * 16;
      l[u] = a.part_l[at];
      x[u] = *reinterpret_cast<const f32x4*>(a.part_o + at * HD + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= run.runs) l[u] = -__builtin_inff();
      top = fmaxf(top, l[u]);
      any = any || l[u] != -__builtin_inff();      // a sum that is no number is not of the maximum, and stays
    }
    if (!any) continue;
    const float old = __builtin_amdgcn_exp2f(M - top);
    M = top;
    W *= old;
    acc *= old;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const float wgt = __builtin_amdgcn_exp2f(l[u] - M);
      W += wgt;
      if (l[u] != -__builtin_inff()) acc += wgt * x[u];
    }
  }
  if (W != 0.f) acc /= W;
  uint2 x;
  x.x = pack_bf16x2(acc[0], acc[1]);
  x.y = pack_bf16x2(acc[2], acc[3]);
  *reinterpret_cast<uint2*>(a.out + (size_t)(run.row0 + node) * a.out_stride + (h * G + r - node * G) * HD + d) = x;
}

template <int HD>
int launch(const Args& a, int items, hipStream_t s) {
  const long long units = (long long)a.nkv * a.n_seqs * a.splits;
  const unsigned grid = (unsigned)((units + 7) / 8 * 8 * (items / a.n_seqs));
  if (a.bs_log2 >= 4) tree_rows_kernel<HD, true><<<grid, NT, 0, s>>>(a);
  else tree_rows_kernel<HD, false><<<grid, NT, 0, s>>>(a);
  DGI_CHECK_LAUNCH();
  if (a.splits > 1) {
    tree_rows_runs_kernel<HD><<<dim3(a.nkv * items, 16 * (HD / 4) / 256), 256, 0, s>>>(a);
    DGI_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

extern "C" int dgi_tree_rows(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride,
                             int table_cols, int n_seqs, int num_blocks, int rows, const int* cu, const int* ctx, const void* mask,
                             int mask_stride, int max_nodes, void* out, long long out_stride, float* part_o, float* part_l, int splits,
                             int min_part, int nh, int nkv, int hd, int block_size, float scale, hipStream_t s) {
  if (n_seqs == 0 || rows == 0) return 0;
  Args a{(const uint16_t*)q, q_stride, (const uint16_t*)k, (const uint16_t*)v, tables, table_stride, table_cols, n_seqs, num_blocks, rows, ctx,
         (uint16_t*)out, out_stride, part_o, part_l, splits, nh, nkv, 0, scale * 1.4426950408889634f, cu, (const unsigned long long*)mask,
         mask_stride, max_nodes, min_part};
  while ((1 << a.bs_log2) < block_size) ++a.bs_log2;
  const int items = n_seqs * ((max_nodes * (nh / nkv) + 15) / 16);
  if (hd == 64) return launch<64>(a, items, s);
  if (hd == 128) return launch<128>(a, items, s);
  if (hd == 256) return launch<256>(a, items, s);
  return -5;
}
