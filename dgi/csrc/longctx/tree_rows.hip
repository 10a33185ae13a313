// dgi/csrc/longctx/tree_rows.hip — attention of drafted trees of few (node, head) pairs over a paged cache.
//
// Up to 32 pairs of a sequence's nodes and a kv head's group are the columns of one product (tree_tiles.hip has more of them).  A
// workgroup owns them and a run of keys; its waves take tiles of 32 keys in turn and are merged through LDS, runs of one sequence by a
// second launch.  Scores are formed transposed, S^T = K Q^T, so that a lane owns a query column and the weights stay in the registers
// that the product O^T += V^T P^T takes them from; V is transposed on its way out of LDS.  Weights are rounded to bf16 for that product
// (as the cached values are; their sum is taken before), everything else is fp32.  Bound by the cache's bytes where contexts are
// long, else by the chain of loads that a run is.
#include "../common.h"

using namespace dgi;

namespace {

constexpr int kList = 512;      // pages of a list in LDS at a time

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
  float* part_o;      // [item][split][16 NQ][HD] of normalised sums, [item][split][16 NQ] of their log2 sums
  float* part_l;
  int splits, nh, nkv, bs_log2;
  float scale_log2;
  const int* cu;
  const unsigned long long* mask;
  int mask_stride, max_nodes, min_part;
};

__device__ __forceinline__ int o_swz(int q) { return ((q & 3) << 3) | (q >> 2); }

template <int HD>
__device__ __forceinline__ int v_lds_off(int row, int col) {
  constexpr int NCH = HD / 8;
  const int ch = (col >> 3) ^ (((row & 7) << 1) & (NCH - 1));
  return row * HD + (ch << 3) + (col & 7);
}

template <int HD>
constexpr int wave_lds() { return 32 * HD * 2 > 16 * HD * 4 ? 32 * HD * 2 : 16 * HD * 4; }

// Runs of a tree's keys: as many as there are places for, of min_part keys at least, each a multiple of 32 keys and of a page.
__device__ __forceinline__ int tree_part(const Args& a, int ctx) {
  const int n = max(1, min(a.splits, (ctx + a.min_part - 1) / a.min_part));
  const int unit = max(32, 1 << a.bs_log2);
  return (((ctx + n - 1) / n) + unit - 1) / unit * unit;
}

template <int HD, int NQ, int NW>
__global__ __launch_bounds__(64 * NW) void tree_rows_kernel(Args a) {
  constexpr int KS = HD / 32, NC = HD / 16, VCH = HD / 8, NT = 64 * NW;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  int2* list = reinterpret_cast<int2*>(smem + NW * wave_lds<HD>());      // [kList] (page, keys seen)
  float* ml = reinterpret_cast<float*>(list + kList);                    // [NW][2][16 NQ]
  int* s_n = reinterpret_cast<int*>(ml + NW * 32 * NQ);                  // [NW + 1]

  const int item = blockIdx.x / a.nkv, h = blockIdx.x - item * a.nkv, split = blockIdx.y;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qi = lane & 15, g = lane >> 4;
  const int G = a.nh / a.nkv, bs = 1 << a.bs_log2;
  uint16_t* vt = reinterpret_cast<uint16_t*>(smem + w * wave_lds<HD>());

  // ---- whose rows, which keys
  const int tiles = (a.max_nodes * G + 16 * NQ - 1) / (16 * NQ), seq = item / tiles;
  const int row0 = a.cu[seq], nodes = row0 < 0 ? 0 : min(min(a.cu[seq + 1], a.rows) - row0, a.max_nodes);
  const int first_node = (item - seq * tiles) * 16 * NQ;                 // (node, head) pairs from here on
  if (first_node >= nodes * G) return;
  const int ctx = min(max(a.ctx[seq], 0), a.table_cols << a.bs_log2);
  const int part = tree_part(a, ctx), lo = split * part, hi = min(lo + part, ctx);
  if (lo >= hi && split > 0) return;
  const int* table = a.tables + (size_t)seq * a.table_stride;

  // ---- queries: column qi of group n; fragments of the second operand, dims 32 s + 8 g ..
  u32x4 qf[NQ][KS];
  unsigned long long bits[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const int r = first_node + 16 * n + qi;
    const int node = r / G, head = h * G + r - node * G;
    const bool live = node < nodes;
    const uint16_t* qp = a.q + (size_t)(row0 + (live ? node : 0)) * a.q_stride + (live ? head : 0) * HD + 8 * g;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[n][s] = live ? *reinterpret_cast<const u32x4*>(qp + 32 * s) : u32x4{0, 0, 0, 0};
    bits[n] = live ? a.mask[(size_t)seq * a.mask_stride + node] : 0;
  }
  const int tree_key = ctx - nodes;      // the key of node 0

  float m_run[NQ], l_run[NQ];
  f32x4 o[NQ][NC];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m_run[n] = -__builtin_inff();
    l_run[n] = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[n][c] = f32x4{0, 0, 0, 0};
  }

  const int per = kList << a.bs_log2;
  for (int at = lo; at < hi; at += per) {
    // ---- the list: the pages of keys at .., also those that are not in the cache, so that a place says which key it is
    __syncthreads();
    const int n = min(per, hi - at), entries = (n + bs - 1) >> a.bs_log2;
    for (int e = tid; e < entries; e += NT) {
      const int id = table[(at >> a.bs_log2) + e];
      const bool there = id >= 0 && id < a.num_blocks;
      list[e] = int2{there ? id : 0, there ? min(bs, hi - at - (e << a.bs_log2)) : 0};
    }
    __syncthreads();
    const int keys = entries << a.bs_log2, ntiles = (keys + 31) >> 5;

    for (int t = w; t < ntiles; t += NW) {
      // ---- K fragments (rows = keys, two groups of 16) and V rows
      u32x4 kf[2][KS], vr[VCH / 2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int tok = 32 * t + 16 * u + qi, e = min(tok >> a.bs_log2, entries - 1);
        const int2 pg = list[e];
        const int off = min(tok & (bs - 1), max(pg.y - 1, 0));
        const uint16_t* p = a.k + ((((size_t)pg.x * a.nkv + h) << a.bs_log2) + off) * HD + 8 * g;
#pragma unroll
        for (int s = 0; s < KS; ++s) kf[u][s] = *reinterpret_cast<const u32x4*>(p + 32 * s);
      }
#pragma unroll
      for (int i = 0; i < VCH / 2; ++i) {
        const int tok = 32 * t + i * (64 / VCH) + lane / VCH, e = min(tok >> a.bs_log2, entries - 1);
        const int2 pg = list[e];
        // zeros past the keys that are seen: their weight is zero, but what lies there may be no number
        const int off = tok & (bs - 1);
        const uint16_t* p = a.v + ((((size_t)pg.x * a.nkv + h) << a.bs_log2) + off) * HD + (lane % VCH) * 8;
        vr[i] = tok < keys && off < pg.y ? *reinterpret_cast<const u32x4*>(p) : u32x4{0, 0, 0, 0};
      }
      // Values of the tree's keys that are infinite or no numbers reach the rows that see them alone, but zero times such a value is no
      // number: they are taken out here and added below where the weight is not zero.
      unsigned odd = 0;
      if (at + 32 * t + 32 > tree_key) {
#pragma unroll
        for (int i = 0; i < VCH / 2; ++i) {
          bool is = false;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const bool lo_odd = (vr[i][j] & 0x7f80u) == 0x7f80u, hi_odd = (vr[i][j] & 0x7f800000u) == 0x7f800000u;
            is = is || lo_odd || hi_odd;
            vr[i][j] &= (lo_odd ? 0xffff0000u : ~0u) & (hi_odd ? 0xffffu : ~0u);
          }
          const unsigned long long b = __ballot(is);
#pragma unroll
          for (int j = 0; j < 64 / VCH; ++j) odd |= (b >> (j * VCH) & ((1ull << VCH) - 1)) ? 1u << (i * (64 / VCH) + j) : 0u;
        }
      }
      // ---- which of the lane's keys (16 u + 4 g + i) are there
      bool there[2][4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int tok = 32 * t + 16 * u + 4 * g + i;
          there[u][i] = tok < keys && (tok & (bs - 1)) < list[min(tok >> a.bs_log2, entries - 1)].y;
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < VCH / 2; ++i) *reinterpret_cast<u32x4*>(vt + v_lds_off<HD>(i * (64 / VCH) + lane / VCH, lane % VCH * 8)) = vr[i];
      u32x4 pf[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        float x[2][4], mx = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          f32x4 acc = {0, 0, 0, 0};
#pragma unroll
          for (int s = 0; s < KS; ++s)
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(kf[u][s]), as_bf16x8(qf[n][s]), acc, 0, 0, 0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            bool see = there[u][i];
            const int node = at + 32 * t + 16 * u + 4 * g + i - tree_key;
            see = see && (node < 0 || (bits[n] >> (node & 63) & 1));
            x[u][i] = see ? acc[i] * a.scale_log2 : -__builtin_inff();
            mx = fmaxf(mx, x[u][i]);
          }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
        const float m_new = fmaxf(m_run[n], mx), m_use = m_new == -__builtin_inff() ? 0.f : m_new;
        const float alpha = __builtin_amdgcn_exp2f(m_run[n] - m_use);
        float psum = 0.f, p[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            p[u][i] = __builtin_amdgcn_exp2f(x[u][i] - m_use);
            psum += p[u][i];
          }
        psum += __shfl_xor(psum, 16, 64);
        psum += __shfl_xor(psum, 32, 64);
        l_run[n] = l_run[n] * alpha + psum;
        m_run[n] = m_new;
#pragma unroll
        for (int c = 0; c < NC; ++c) o[n][c] *= alpha;
        pf[n] = u32x4{pack_bf16x2(p[0][0], p[0][1]), pack_bf16x2(p[0][2], p[0][3]), pack_bf16x2(p[1][0], p[1][1]),
                      pack_bf16x2(p[1][2], p[1][3])};
      }
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
#pragma unroll
        for (int n = 0; n < NQ; ++n) o[n][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(vf), as_bf16x8(pf[n]), o[n][c], 0, 0, 0);
      }
      for (; odd; odd &= odd - 1) {      // what was taken out: key kk of the tile
        const int kk = __ffs(odd) - 1, tok = 32 * t + kk, j = (kk >> 4) * 4 + (kk & 3);
        const uint16_t* vp = a.v + ((((size_t)list[tok >> a.bs_log2].x * a.nkv + h) << a.bs_log2) + (tok & (bs - 1))) * HD + 4 * g;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const uint32_t two = __shfl(j & 4 ? (j & 2 ? pf[n][3] : pf[n][2]) : (j & 2 ? pf[n][1] : pf[n][0]), 16 * (kk >> 2 & 3) + qi, 64);
          const float p = __uint_as_float(j & 1 ? two & 0xffff0000u : two << 16);
#pragma unroll
          for (int c = 0; c < NC; ++c)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const uint16_t x = vp[16 * c + i];
              if ((x & 0x7f80) == 0x7f80 && p != 0.f) o[n][c][i] += p * bf16_to_f32(x);
            }
        }
      }
    }
  }

  // ---- the waves' results, 16 columns at a time
  if (g == 0)
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      ml[w * 32 * NQ + 16 * n + qi] = m_run[n];
      ml[w * 32 * NQ + 16 * NQ + 16 * n + qi] = l_run[n];
    }
  const bool split_up = part < ctx;
  const size_t slab = (((size_t)item * a.nkv + h) * a.splits + split) * 16 * NQ;
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    __syncthreads();
    float* ow = reinterpret_cast<float*>(smem + w * wave_lds<HD>());
#pragma unroll
    for (int c = 0; c < NC; ++c)
#pragma unroll
      for (int i = 0; i < 4; ++i) ow[qi * HD + ((16 * c + 4 * g + i) ^ o_swz(qi))] = o[n][c][i];
    __syncthreads();
    for (int idx = tid; idx < 16 * HD; idx += NT) {
      const int qq = idx / HD, d = idx - qq * HD;
      const int r = first_node + 16 * n + qq;
      const int node = r / G, head = h * G + r - node * G;
      if (node >= nodes) continue;
      float M = -__builtin_inff();
#pragma unroll
      for (int v = 0; v < NW; ++v) M = fmaxf(M, ml[v * 32 * NQ + 16 * n + qq]);
      const float use = M == -__builtin_inff() ? 0.f : M;
      float L = 0.f, acc = 0.f;
#pragma unroll
      for (int v = 0; v < NW; ++v) {
        const float sc = exp2f(ml[v * 32 * NQ + 16 * n + qq] - use);
        L += ml[v * 32 * NQ + 16 * NQ + 16 * n + qq] * sc;
        acc += reinterpret_cast<float*>(smem + v * wave_lds<HD>())[qq * HD + (d ^ o_swz(qq))] * sc;
      }
      const float res = L == 0.f ? 0.f : acc / L;
      if (!split_up) {
        a.out[(size_t)(row0 + node) * a.out_stride + head * HD + d] = f32_to_bf16(res);
      } else {
        a.part_o[(slab + 16 * n + qq) * HD + d] = res;
        if (d == 0) a.part_l[slab + 16 * n + qq] = L == 0.f ? -__builtin_inff() : M + log2f(L);
      }
    }
  }
}

// Runs of the same columns: weighed by their sums.
template <int HD, int NQ>
__global__ __launch_bounds__(HD) void tree_rows_reduce_kernel(Args a) {
  const int item = blockIdx.x / a.nkv, h = blockIdx.x - item * a.nkv, col = blockIdx.y, d = threadIdx.x, G = a.nh / a.nkv;
  const int tiles = (a.max_nodes * G + 16 * NQ - 1) / (16 * NQ), seq = item / tiles;
  const int r = (item - seq * tiles) * 16 * NQ + col, node = r / G;
  if (a.cu[seq] < 0 || node >= min(min(a.cu[seq + 1], a.rows) - a.cu[seq], a.max_nodes)) return;
  const int ctx = min(max(a.ctx[seq], 0), a.table_cols << a.bs_log2), part = tree_part(a, ctx);
  if (part >= ctx) return;
  const int runs = (ctx + part - 1) / part, row = a.cu[seq] + node, head = h * G + r - node * G;
  const size_t base = ((size_t)item * a.nkv + h) * a.splits * 16 * NQ + col;
  float M = -__builtin_inff();
  for (int i = 0; i < runs; ++i) M = fmaxf(M, a.part_l[base + (size_t)i * 16 * NQ]);
  float W = 0.f, acc = 0.f;
  for (int i = 0; i < runs; ++i) {
    const float l = a.part_l[base + (size_t)i * 16 * NQ];
    if (l == -__builtin_inff()) continue;
    const float wgt = exp2f(l - M);
    W += wgt;
    acc += wgt * a.part_o[(base + (size_t)i * 16 * NQ) * HD + d];
  }
  a.out[(size_t)row * a.out_stride + head * HD + d] = f32_to_bf16(W == 0.f ? 0.f : acc / W);
}

template <int HD, int NQ, int NW>
int launch(const Args& a, int items, hipStream_t s) {
  const int lds = NW * wave_lds<HD>() + kList * 8 + NW * 32 * NQ * 4 + (NW + 1) * 4;
  tree_rows_kernel<HD, NQ, NW><<<dim3(a.nkv * items, a.splits), 64 * NW, lds, s>>>(a);
  DGI_CHECK_LAUNCH();
  if (a.splits > 1) {
    tree_rows_reduce_kernel<HD, NQ><<<dim3(a.nkv * items, 16 * NQ), HD, 0, s>>>(a);
    DGI_CHECK_LAUNCH();
  }
  return 0;
}

template <int NQ, int NW>
int launch_dims(const Args& a, int items, int hd, hipStream_t s) {
  if (hd == 64) return launch<64, NQ, NW>(a, items, s);
  if (hd == 128) return launch<128, NQ, NW>(a, items, s);
  if (hd == 256) return launch<256, NQ, NW>(a, items, s);
  return -5;
}

}  // namespace

// Query columns of a workgroup of a tree: 16 or 32 of its (node, head) pairs.
extern "C" int dgi_tree_columns(int max_nodes, int G) { return max_nodes * G <= 16 ? 16 : 32; }

extern "C" int dgi_tree_rows(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride,
                              int table_cols, int n_seqs, int num_blocks, int rows, const int* cu, const int* ctx, const void* mask,
                              int mask_stride, int max_nodes, void* out, long long out_stride, float* part_o, float* part_l, int splits,
                              int min_part, int nh, int nkv, int hd, int block_size, float scale, hipStream_t s) {
  if (n_seqs == 0 || rows == 0) return 0;
  Args a{};
  a.q = (const uint16_t*)q;
  a.q_stride = q_stride;
  a.k = (const uint16_t*)k;
  a.v = (const uint16_t*)v;
  a.tables = tables;
  a.table_stride = table_stride;
  a.table_cols = table_cols;
  a.n_seqs = n_seqs;
  a.num_blocks = num_blocks;
  a.rows = rows;
  a.ctx = ctx;
  a.out = (uint16_t*)out;
  a.out_stride = out_stride;
  a.part_o = part_o;
  a.part_l = part_l;
  a.splits = splits;
  a.nh = nh;
  a.nkv = nkv;
  while ((1 << a.bs_log2) < block_size) ++a.bs_log2;
  a.scale_log2 = scale * 1.4426950408889634f;
  a.cu = cu;
  a.mask = (const unsigned long long*)mask;
  a.mask_stride = mask_stride;
  a.max_nodes = max_nodes;
  a.min_part = min_part;
  const int cols = dgi_tree_columns(max_nodes, nh / nkv), items = n_seqs * ((max_nodes * (nh / nkv) + cols - 1) / cols);
  if (cols == 16) return launch_dims<1, 4>(a, items, hd, s);
  return launch_dims<2, 4>(a, items, hd, s);
}
