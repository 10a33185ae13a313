// dgi/csrc/longctx/selected_attention.hip — attention of every row over the pages selected for it, one list per (row, kv head).
//
//   o = sum_j p_j v_j / sum_j p_j,  p_j = 2^(x_j - max x),  x_j = scale log2(e) q . k_j     over the keys j of the row's pages,
// in one pass over the keys with the running maximum and sum in fp32; a row that sees nothing is zero.
//
// A workgroup owns the G heads of a kv head for one row or, where rows of one sequence follow each other, for as many of them as
// make 16 query columns: neighbours of a prompt mostly select the same pages, which are then read once, and the columns of the matrix
// instruction are used.  It reads the union of their lists (made by a launch of its own, a bit per page and row in LDS), each column
// masked to its own row's.  Its waves take tiles of 32 keys in turn and are merged through LDS; where rows are few, each is by itself, and its
// list is cut between workgroups, whose sums a second launch adds up.
//
// Scores are formed transposed, S^T = K Q^T, so that a lane owns a query column and the weights stay in the registers that the product
// O^T += V^T P^T takes them from.  Weights are rounded to bf16 for that product (as the cached values are; their sum is taken before),
// everything else is fp32.  A tile's keys and values are asked for while the one before is multiplied, whole rows a load, and go
// through LDS: operands of the key product loaded as they are needed touch every line twice, 64 bytes at a time.
//
// Decode rows are bound by the bytes of their pages: 64 rows of 64 heads on 8, 128 pages of 16 keys each, 97 us, 5.5 TB/s.  Rows of
// prompts by the path from the L2 to a compute unit's registers: 2 x 509 rows of 28 heads on 4, 64 pages each, 97 us, 1.5 GB of keys
// and values where row by row it is 2.1 GB (205 us; together with key operands straight from memory 133; without the loads 70).
// Three workgroups a compute unit spill registers (104).
#include "../common.h"

#include <type_traits>

using namespace dgi;

namespace {

constexpr int kList = 256;       // pages of a list in LDS at a time
constexpr int kBits = 2048;      // words for the union's bits
constexpr int NW = 4, NT = 64 * NW;

struct Args {
  const uint16_t* q;
  long long q_stride;
  const uint16_t* k;
  const uint16_t* v;
  const int* tables;
  int table_stride, table_cols, n_seqs, num_blocks, rows;
  const int* ctx;
  const int* row_seq;
  const int* pages;
  int count;
  uint16_t* out;
  long long out_stride;
  float* part_o;      // [row][kv head][run][G][HD] of normalised sums, [row][kv head][run][G] of their log2 sums
  float* part_l;
  int splits, nh, nkv, bs_log2;
  float scale_log2;
  int4* plan;         // [rows][kv head][count] what the rows that begin with a row read: page, place, rows that selected it
  int* plan_total;    // [rows][kv head] how many entries
  int* plan_rows;     // [rows] how many rows go together, 0: the row goes with one before it
};

// Where 16-byte chunk ch of a row lies in LDS: keys are read 16 rows at one chunk (16 banks' worth apart), values transposed.
template <int HD>
__device__ __forceinline__ int k_lds_off(int row, int ch) { return row * HD + ((ch ^ (HD == 64 ? row >> 1 & 7 : row & 15)) << 3); }
template <int HD>
__device__ __forceinline__ int v_lds_chunk(int row, int ch) { return row * HD + ((ch ^ (((row & 7) << 1) & (HD / 8 - 1))) << 3); }
template <int HD>
__device__ __forceinline__ int v_lds_off(int row, int col) { return v_lds_chunk<HD>(row, col >> 3) + (col & 7); }

template <int HD>
constexpr int wave_lds() { return 64 * HD; }      // a tile of values (32 x HD bf16), then 16 rows of sums (fp32)

// Rows that go together: of one aligned group of 16 / G, as long as the sequence is the same.  0: the row goes with one before it.
// Lane i of each wave looks at row i of the group.
__device__ __forceinline__ int rows_from(const Args& a, int t, int most, int lane) {
  if (most == 1 || !a.row_seq) return 1;
  const int at = t % most, row = t - at + lane;
  const int seq = lane < most && row < a.rows ? a.row_seq[row] : -1;
  const int prev = __shfl_up(seq, 1, 64);
  // rows of the group that do not go on with the one before, and those behind it
  const unsigned begins = (unsigned)__ballot(lane < most && (lane == 0 || row >= a.rows || seq != prev)) | 1u << most;
  if (!(begins >> at & 1)) return 0;
  return __ffs(begins >> (at + 1));
}

// What the workgroups of rows that go together read: the union of their lists, ascending, or, where a row names a page twice (it counts
// twice) or the bits do not fit, one list after another.  A workgroup per (first row, kv head).
template <int THREADS>
__global__ __launch_bounds__(THREADS) void selected_plan_kernel(Args a, int n_bits) {
  extern __shared__ unsigned bits[];                     // [rows][words] the pages that a row selected
  int* before = reinterpret_cast<int*>(bits + n_bits);   // [words] pages of any row in the words before
  __shared__ int s_n[THREADS / 64];
  const int G = a.nh / a.nkv, side = 16 / G, groups = (a.rows + side - 1) / side;
  // the first rows of all groups, the second ones, ..: most of the others have nothing to do, and would leave every other XCD without work
  const int unit = blockIdx.x / a.nkv, h = blockIdx.x - unit * a.nkv, place = unit / groups, t0 = (unit - place * groups) * side + place;
  const int tid = threadIdx.x, w = tid >> 6, lane = tid & 63;
  if (t0 >= a.rows) return;
  const int m = rows_from(a, t0, side, lane);
  if (h == 0 && tid == 0) a.plan_rows[t0] = m;
  if (m == 0) return;
  const int seq = a.row_seq[t0];
  const bool known = seq >= 0 && seq < a.n_seqs;
  const int* table = a.tables + (size_t)(known ? seq : 0) * a.table_stride;
  int most = known && lane < m ? a.ctx[t0 + lane] : 0;
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) most = max(most, __shfl_xor(most, o, 64));
  most = __shfl(most, 0, 64);
  int4* list = a.plan + (size_t)t0 * a.nkv * a.count + (size_t)h * m * a.count;
  auto entry = [&](int i) {      // entry e of row r; i = r count + e
    const int r = i / a.count;
    return a.pages[((size_t)(t0 + r) * a.nkv + h) * a.count + (i - r * a.count)];
  };
  auto fits = [&](int p) { return p >= 0 && p < a.table_cols && ((long long)p << a.bs_log2) < most; };
  const int words = min((int)(((long long)most + (32ll << a.bs_log2) - 1) >> (a.bs_log2 + 5)), (a.table_cols + 31) >> 5), all = m * a.count;
  bool together = m > 1 && m * words <= n_bits;
  if (together) {
    for (int i = tid; i < m * words; i += THREADS) bits[i] = 0;
    __syncthreads();
    bool twice = false;
    for (int i = tid; i < all; i += THREADS) {
      const int p = entry(i);
      if (fits(p)) twice = twice || (atomicOr(&bits[i / a.count * words + (p >> 5)], 1u << (p & 31)) >> (p & 31) & 1);
    }
    together = !__syncthreads_or(twice);
  }
  if (!together) {
    for (int i = tid; i < all; i += THREADS) {
      const int p = entry(i), id = fits(p) ? table[p] : -1;
      const bool there = id >= 0 && id < a.num_blocks;
      list[i] = int4{there ? id : 0, there ? p << a.bs_log2 : 0, there ? 1 << (i / a.count) : 0, 0};
    }
    if (tid == 0) a.plan_total[t0 * a.nkv + h] = all;
    return;
  }
  const int per = (words + THREADS - 1) / THREADS, first = min(tid * per, words), last = min(first + per, words);
  int n = 0;
  for (int i = first; i < last; ++i) {
    unsigned u = 0;
    for (int r = 0; r < m; ++r) u |= bits[r * words + i];
    before[i] = n;
    n += __popc(u);
  }
  int sum = n;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(sum, o, 64);
    if (lane >= o) sum += x;
  }
  if (lane == 63) s_n[w] = sum;
  __syncthreads();
  int from = sum - n;
  for (int v = 0; v < w; ++v) from += s_n[v];
  if (tid == THREADS - 1) a.plan_total[t0 * a.nkv + h] = from + n;
  for (int i = first; i < last; ++i) before[i] += from;
  __syncthreads();
  for (int i = tid; i < all; i += THREADS) {      // the first row that has a page writes it
    const int p = entry(i), r = i / a.count, word = p >> 5;
    if (!fits(p)) continue;
    unsigned who = 0, u = 0;
    for (int s = 0; s < m; ++s) {
      const unsigned x = bits[s * words + word];
      who |= (x >> (p & 31) & 1) << s;
      u |= x;
    }
    if (who & ((1u << r) - 1)) continue;
    const int id = table[p];
    const bool there = id >= 0 && id < a.num_blocks;
    list[before[word] + __popc(u & ((1u << (p & 31)) - 1))] = int4{there ? id : 0, there ? p << a.bs_log2 : 0, there ? (int)who : 0, 0};
  }
}

// PLAN: rows that go together and their list, which is not cut, come from the launch before; otherwise each row is by itself.
template <int HD, bool WIDE, bool PLAN>
__global__ __launch_bounds__(NT, HD == 256 ? 1 : 2) void selected_kernel(Args a) {
  constexpr int KS = HD / 32, NC = HD / 16, VCH = HD / 8;
  __shared__ __attribute__((aligned(16))) char smem[NW * wave_lds<HD>()];
  __shared__ int4 list[kList];            // page, its first key's place in the sequence, rows that selected it
  __shared__ float ml[NW][2][16];
  __shared__ int s_n[NW];

  const int G = a.nh / a.nkv, bs = 1 << a.bs_log2;
  const int unit = blockIdx.x / a.nkv, h = blockIdx.x - unit * a.nkv;
  int t0 = unit, m = 1;
  if constexpr (PLAN) {      // in the plan's order of rows
    const int side = 16 / G, groups = (a.rows + side - 1) / side, place = unit / groups;
    t0 = (unit - place * groups) * side + place;
    if (t0 >= a.rows) return;
    m = a.plan_rows[t0];
    if (m == 0) return;
  }
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63, qi = lane & 15, g = lane >> 4;
  uint16_t* vt = reinterpret_cast<uint16_t*>(smem + w * wave_lds<HD>());

  const int seq = a.row_seq ? a.row_seq[t0] : t0;
  const bool known = seq >= 0 && seq < a.n_seqs;
  // column qi: head qi % G of row qi / G
  const int rr = qi / G, head = h * G + qi - rr * G;
  const bool live = rr < m;
  const int ctx = known && live ? a.ctx[t0 + rr] : 0;
  u32x4 qf[KS];
  const uint16_t* qp = a.q + (size_t)(t0 + (live ? rr : 0)) * a.q_stride + (live ? head : 0) * HD + 8 * g;
#pragma unroll
  for (int s = 0; s < KS; ++s) qf[s] = live ? *reinterpret_cast<const u32x4*>(qp + 32 * s) : u32x4{0, 0, 0, 0};
  int most = ctx, least = live ? ctx : 0x7fffffff;      // the longest and the shortest context of the rows
  if constexpr (PLAN) {
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      most = max(most, __shfl_xor(most, o, 64));
      least = min(least, __shfl_xor(least, o, 64));
    }
    least = __builtin_amdgcn_readfirstlane(least);
  }
  most = __builtin_amdgcn_readfirstlane(most);      // lane 0's column is live
  if constexpr (!PLAN) least = most;
  const int total = PLAN ? a.plan_total[t0 * a.nkv + h] : a.count;
  const int splits = PLAN ? 1 : a.splits, split = PLAN ? 0 : blockIdx.y;
  const int part = (total + splits - 1) / splits, lo = split * part, hi = most > 0 ? min(lo + part, total) : lo;
  const int4* planned = PLAN ? a.plan + (size_t)t0 * a.nkv * a.count + (size_t)h * m * a.count : nullptr;

  // where the lane's chunk of row i 64 / VCH + lane / VCH goes in LDS: the same for every P-th i, but for whole rows
  constexpr int P = VCH / 4;      // 16 rows
  int k_at[P], v_at[P];
#pragma unroll
  for (int i = 0; i < P; ++i) {
    k_at[i] = k_lds_off<HD>(i * (64 / VCH) + lane / VCH, lane % VCH);
    v_at[i] = v_lds_chunk<HD>(i * (64 / VCH) + lane / VCH, lane % VCH);
  }
  const int ctx_g = ctx - 4 * g;      // the lane's keys begin at 4 g

  float m_run, l_run;
  f32x4 o[NC];
  // A pass over the keys for all rows.  Values that are infinite or no numbers reach the rows that see them alone, but zero times such a
  // value is no number: where rows go together and a result is not finite, each is done again by itself, the values that it does not
  // see as zeros.
  for (int turn = -1, turns = 0; turn < turns; ++turn) {
    const bool alone = PLAN && turn >= 0;
    const unsigned who = alone ? 1u << turn : (1u << m) - 1;
    const int limit = alone ? a.ctx[t0 + turn] : most;
    m_run = -__builtin_inff();
    l_run = 0.f;
#pragma unroll
    for (int c = 0; c < NC; ++c) o[c] = f32x4{0, 0, 0, 0};
    for (int at = lo; at < hi; at += kList) {
      int entries = min(kList, hi - at);
      __syncthreads();
      if constexpr (PLAN) {
        if (tid < entries) list[tid] = planned[at + tid];
      } else {      // entries without a page are left out
        int id = -1, p = -1;
        if (tid < entries) {
          p = a.pages[((size_t)t0 * a.nkv + h) * a.count + at + tid];
          if (p >= 0 && p < a.table_cols && ((long long)p << a.bs_log2) < most) id = a.tables[(size_t)seq * a.table_stride + p];
        }
        const bool there = id >= 0 && id < a.num_blocks;
        const unsigned long long b = __ballot(there);
        if (lane == 0) s_n[w] = __popcll(b);
        __syncthreads();
        int from = 0;
        entries = 0;
        for (int v = 0; v < NW; ++v) {
          if (v < w) from += s_n[v];
          entries += s_n[v];
        }
        if (there) list[from + __popcll(b & ((1ull << lane) - 1))] = int4{id, p << a.bs_log2, 1, 0};
      }
      __syncthreads();
      const int keys = entries << a.bs_log2, ntiles = (keys + 31) >> 5;
      u32x4 kr[VCH / 2], vr[VCH / 2];
      // Sixteen keys of a tile lie side by side in one page (WIDE), or each lane finds its own: where they lie in the cache, in the
      // sequence, and who selected them.  Past the list: its last page, selected by nobody.
      struct Keys {
        size_t row;
        int base;
        unsigned who;
      };
      auto keys_at = [&](int tok) {
        const int e = min(tok >> a.bs_log2, entries - 1), off = tok & (bs - 1);
        const int4 page = list[e];
        return Keys{(((size_t)page.x * a.nkv + h) << a.bs_log2) + off, page.y + off, tok < keys ? (unsigned)page.z : 0u};
      };
      auto half = [&](int t, int u) {      // WIDE: in scalar registers
        const Keys x = keys_at(32 * t + 16 * u);
        return Keys{((size_t)__builtin_amdgcn_readfirstlane((int)(x.row >> 32)) << 32) | (unsigned)__builtin_amdgcn_readfirstlane((int)x.row),
                    __builtin_amdgcn_readfirstlane(x.base), (unsigned)__builtin_amdgcn_readfirstlane(x.who)};
      };
      // a tile's rows, whole lines a load
      auto load = [&](int t, const Keys* x, const uint16_t* cache, u32x4* to) {
#pragma unroll
        for (int i = 0; i < VCH / 2; ++i) {
          constexpr int R = 64 / VCH;      // rows a load
          const int u = i * R / 16;
          to[i] = *reinterpret_cast<const u32x4*>(WIDE ? cache + x[u].row * HD + ((i * R - 16 * u) * HD + lane * 8)
                                                       : cache + keys_at(32 * t + i * R + lane / VCH).row * HD + lane % VCH * 8);
        }
      };
      // and into LDS, behind the reads of what was there
      auto stage = [&](const u32x4* from, const int* at) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < VCH / 2; ++i) *reinterpret_cast<u32x4*>(vt + at[i % P] + i / P * (64 / VCH * P * HD)) = from[i];
      };
      auto tile = [&](int t, Keys* now, Keys* next, auto LAST) {
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
        const int end = max(now[0].base, now[1].base) + 16;
        // values that no row (alone: not this one) sees are zeros: their weight is zero, but what lies there may be no number
        if (!WIDE || alone || !now[0].who || !now[1].who || end > most) {
#pragma unroll
          for (int i = 0; i < VCH / 2; ++i) {
            constexpr int R = 64 / VCH;
            const int u = i * R / 16;
            const Keys x = WIDE ? Keys{0, now[u].base + i * R - 16 * u, now[u].who} : keys_at(32 * t + i * R + lane / VCH);
            if (x.base >= limit - (WIDE ? lane / VCH : 0) || !(x.who & who)) vr[i] = u32x4{0, 0, 0, 0};
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
          for (int i = 0; i < 4; ++i) x[u][i] = sc[u][i] * a.scale_log2;
        if (!WIDE || (now[0].who & now[1].who & who) != who || end > least) {      // not all columns see all keys
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const Keys k = WIDE ? Keys{0, now[u].base + i, now[u].who} : keys_at(32 * t + 16 * u + 4 * g + i);
              if (!((k.who & who) >> rr & 1) || k.base >= (WIDE ? ctx_g : ctx)) x[u][i] = -__builtin_inff();
            }
        }
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) mx = fmaxf(mx, x[u][i]);
        // the sums are scaled anew only where a maximum grows by more than 8 (weights stay below 2^8), and there the four lanes of
        // a column agree on it
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
      };
      if (w < ntiles) {
        Keys now[2], next[2];
        auto find = [&](Keys* x, int t) {
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
    bool odd = false;
    for (int idx = tid; idx < m * G * (HD / 4); idx += NT) {
      const int col = idx / (HD / 4), d = idx - col * (HD / 4), row = col / G;
      if (!(who >> row & 1)) continue;
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
#pragma unroll
      for (int i = 0; i < 4; ++i) odd = odd || !(fabsf(acc[i]) < __builtin_inff());
      const int head_at = h * G + col - row * G;
      if (splits == 1) {
        uint2 r;
        r.x = pack_bf16x2(acc[0], acc[1]);
        r.y = pack_bf16x2(acc[2], acc[3]);
        *reinterpret_cast<uint2*>(a.out + (size_t)(t0 + row) * a.out_stride + head_at * HD + 4 * d) = r;
      } else {
        const size_t slab = (((size_t)(t0 + row) * a.nkv + h) * splits + split) * G + col - row * G;
        *reinterpret_cast<f32x4*>(a.part_o + slab * HD + 4 * d) = acc;
        if (d == 0) a.part_l[slab] = L == 0.f ? -__builtin_inff() : M + __builtin_amdgcn_logf(L);
      }
    }
    if (PLAN && m > 1 && !alone && __syncthreads_or(odd)) turns = m;
  }
}

// The runs of a row's list, weighed by their sums: HD / 4 lanes a head.
template <int HD>
__global__ __launch_bounds__(256) void selected_runs_kernel(Args a) {
  const int G = a.nh / a.nkv, idx = blockIdx.x * 256 + threadIdx.x, col = idx / (HD / 4), d = idx % (HD / 4) * 4;      // col: row, head
  if (col >= a.rows * a.nh) return;
  const int row = col / a.nh, head = col - row * a.nh, h = head / G;
  const size_t base = ((size_t)row * a.nkv + h) * a.splits * G + head - h * G;
  constexpr int U = 8;
  float M = -__builtin_inff(), W = 0.f;
  f32x4 acc = {0, 0, 0, 0};
  for (int s = 0; s < a.splits; s += U) {
    float l[U], top = M;
    bool any = false;
    f32x4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const size_t at = base + (size_t)min(s + u, a.splits - 1) * G;
      l[u] = a.part_l[at];
      x[u] = *reinterpret_cast<const f32x4*>(a.part_o + at * HD + d);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s + u >= a.splits) l[u] = -__builtin_inff();
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
  uint2 r;
  r.x = pack_bf16x2(acc[0], acc[1]);
  r.y = pack_bf16x2(acc[2], acc[3]);
  *reinterpret_cast<uint2*>(a.out + (size_t)row * a.out_stride + head * HD + d) = r;
}

template <int HD>
int launch(const Args& a, hipStream_t s) {
  if (a.plan) {
    const int side = 16 / (a.nh / a.nkv), rows = (a.rows + side - 1) / side * side;
    const int words = (a.table_cols + 31) / 32, n_bits = (int)min((long long)side * words, (long long)kBits), lds = (n_bits + min(words, kBits / 2)) * 4;
    // a wave for lists that it has in a few turns: all of them at once (2 x 509 rows of 64 pages, 4 heads: 7.3 us, four waves 9.5)
    if ((long long)side * a.count <= 1024) selected_plan_kernel<64><<<a.nkv * rows, 64, lds, s>>>(a, n_bits);
    else selected_plan_kernel<NT><<<a.nkv * rows, NT, lds, s>>>(a, n_bits);
    DGI_CHECK_LAUNCH();
    if (a.bs_log2 >= 4) selected_kernel<HD, true, true><<<a.nkv * rows, NT, 0, s>>>(a);
    else selected_kernel<HD, false, true><<<a.nkv * rows, NT, 0, s>>>(a);
  } else {
    const dim3 grid(a.nkv * a.rows, a.splits);
    if (a.bs_log2 >= 4) selected_kernel<HD, true, false><<<grid, NT, 0, s>>>(a);
    else selected_kernel<HD, false, false><<<grid, NT, 0, s>>>(a);
  }
  DGI_CHECK_LAUNCH();
  if (a.splits > 1) {
    selected_runs_kernel<HD><<<(unsigned)(((long long)a.rows * a.nh * (HD / 4) + 255) / 256), 256, 0, s>>>(a);
    DGI_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

extern "C" int dgi_paged_selected(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride,
                                  int table_cols, int n_seqs, int num_blocks, const int* ctx, const int* row_seq, const int* pages, int count,
                                  void* out, long long out_stride, float* part_o, float* part_l, int splits, void* plan, int* plan_total,
                                  int* plan_rows, int T, int nh, int nkv, int hd, int block_size, float scale, hipStream_t s) {
  if (T == 0) return 0;
  if (splits < 1 || (plan && splits > 1)) return -5;      // lists of rows that go together are not cut
  Args a{(const uint16_t*)q, q_stride, (const uint16_t*)k, (const uint16_t*)v, tables, table_stride, table_cols, n_seqs, num_blocks, T, ctx,
         row_seq, pages, count, (uint16_t*)out, out_stride, part_o, part_l, splits, nh, nkv, 0, scale * 1.4426950408889634f,
         (int4*)plan, plan_total, plan_rows};
  while ((1 << a.bs_log2) < block_size) ++a.bs_log2;
  if (hd == 64) return launch<64>(a, s);
  if (hd == 128) return launch<128>(a, s);
  if (hd == 256) return launch<256>(a, s);
  return -5;
}
