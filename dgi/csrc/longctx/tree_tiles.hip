// dgi/csrc/longctx/tree_tiles.hip — attention of drafted trees of many (node, head) pairs over a paged cache.
//
// All heads of a kv head's group and all nodes of a sequence see the same keys but for the tree's own: their (node, head) pairs are the
// rows of one product, r = node G + head.  A workgroup owns 128 of them (32 a wave) and a run of keys.  Tiles of 64 keys and values go
// straight to LDS, two stages, one barrier a tile; scores are formed transposed, S^T = K Q^T, so that a lane owns a row and the weights are
// the operand of O^T += V^T P^T where they lie.  Only the tiles that hold the tree's keys are masked.
//
// Bound by the matrix cores where there are many pairs (4 nodes n heads hd products a key), by the cache's bytes where there are few; with
// few sequences also by how many workgroups share the keys.  The tiles of 64 keys of all (128 rows, sequence) of a kv head, one after
// another, are dealt out in equal shares, so that a long context beside short ones does not hold up the launch; what a share's ends
// cut is added up by a second launch.
//
// 16 trees of 60 nodes, 64 heads on 8, 1000 to 8000 keys: 174 us, 636 TF/s of 111 Gflop (with workgroups by sequence and run of
// its keys instead of equal shares, 260).  A tile takes 2.0 us for the two workgroups of a compute unit, 1070 TF/s; the rest is the
// beginning and end of the two parts that a share has (20 us) and the second launch (10 us).
#include "../prefill_attention_kernel.h"

using namespace dgi;
using namespace dgi::prefill;

namespace {

constexpr int kRows = 128, kWaves = 4;      // rows of a workgroup
constexpr float kLowest = -__FLT_MAX__;     // maximum of no key

struct Args {
  const uint16_t* q;
  long long q_stride;
  const uint16_t* k;
  const uint16_t* v;
  const int* tables;
  int table_stride, table_cols, n_seqs, num_blocks, rows;
  const int* cu;
  const int* ctx;
  const unsigned long long* mask;
  int mask_stride, max_nodes;
  uint16_t* out;
  long long out_stride;
  float* part_o;      // [share][kv head][2][128][HD] of normalised sums, [share][kv head][2][128] of their log2 sums
  float* part_l;
  int shares, least, nh, nkv, bs_log2;      // shares of a kv head at most, steps of a share at least
  float scale_log2;
};

// A sequence: its first row, its nodes, its row tiles, its context, and the steps (tiles of 64 keys, one for an empty context) that each row
// tile counts as: those that it takes, or `pad`.
struct Seq {
  int q0, nodes, tiles, ctx, steps;
};
// kLead more steps go into the deal for each: what it costs to begin and end one (10 us where a step takes 2)
constexpr int kLead = 4;
__device__ __forceinline__ Seq sequence(const Args& a, int s, int pad) {
  if (s >= a.n_seqs) return {0, 0, 0, 0, 0};
  const int q0 = a.cu[s], q1 = a.cu[s + 1], ctx = min(max(a.ctx[s], 0), a.table_cols << a.bs_log2);
  const int nodes = q0 < 0 ? 0 : max(0, min(min(q1, a.rows) - q0, a.max_nodes));
  return {q0, nodes, (nodes * (a.nh / a.nkv) + kRows - 1) / kRows, ctx, pad ? pad : kLead + max(1, (ctx + KT - 1) / KT)};
}

// The order of a kv head's steps: row tile 0 of every sequence, row tile 1, ..  One wave counts; `first` is its lane's sequence, of the first
// 64; results are in all lanes.
// (sequences before `seq` in row tile mt, all tiles before it)
__device__ int steps_before(const Args& a, const Seq& first, int lane, int mt, int seq, int pad) {
  long long sum = 0;
  Seq q = first;
  for (int s0 = 0;;) {
    sum += (long long)q.steps * (min(q.tiles, mt) + (s0 + lane < seq && q.tiles > mt ? 1 : 0));
    if ((s0 += 64) >= a.n_seqs) break;
    q = sequence(a, s0 + lane, pad);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  return (int)min(sum, 0x7fffffffll);
}
// Steps of a share.  Where whole row tiles, as many for each share, are few steps more than equal shares, each counts as the longest: nothing
// is cut.  kSlack is what a cut costs, the second beginning and the second launch (12 trees of 43 nodes, 64 heads on 8, 371 keys: 29 us, with cuts
// 36; 16 of 60 nodes over 300 to 900 keys 46, 58; 64 of 64 over 300 109, 115).
constexpr int kSlack = 20;
__device__ int share_of(const Args& a, Seq& first, int lane, int& pad) {
  pad = 0;
  long long sum = 0;
  int tiles = 0, longest = 0;
  Seq q = first;
  for (int s0 = 0;;) {
    sum += (long long)q.steps * q.tiles;
    tiles += q.tiles;
    if (q.tiles > 0) longest = max(longest, q.steps);
    if ((s0 += 64) >= a.n_seqs) break;
    q = sequence(a, s0 + lane, 0);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    sum += __shfl_xor(sum, o, 64);
    tiles += __shfl_xor(tiles, o, 64);
    longest = max(longest, __shfl_xor(longest, o, 64));
  }
  const int len = max(a.least, ((int)min(sum, 0x7fffffffll) + a.shares - 1) / a.shares);
  const long long whole = (long long)((tiles + a.shares - 1) / a.shares) * longest;
  if (tiles == 0 || whole > len + kSlack) return len;
  pad = first.steps = longest;
  return (int)whole;
}
// whose step `at` is; row tile -1: behind the last one
struct Place {
  int mt, seq, step;
};
__device__ Place place_of(const Args& a, const Seq& first, int lane, int at, int pad) {
  for (int mt = 0, before = 0;; ++mt) {
    int any = 0;
    Seq q = first;
    for (int s0 = 0;;) {
      const int mine = q.tiles > mt ? q.steps : 0;
      int sum = mine;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int x = __shfl_up(sum, o, 64);
        if (lane >= o) sum += x;
      }
      const int from = before + sum - mine;
      const unsigned long long here = __ballot(at >= from && at < from + mine);
      if (here) {
        const int l = __ffsll(here) - 1;
        return {mt, s0 + l, at - __shfl(from, l, 64)};
      }
      const int all = __shfl(sum, 63, 64);
      before += all;
      any += all;
      if ((s0 += 64) >= a.n_seqs) break;
      q = sequence(a, s0 + lane, pad);
    }
    if (!any) return {-1, 0, 0};
  }
}

template <int HD>
__global__ __launch_bounds__(kWaves * 64, 2) void tree_tiles_kernel(Args a) {
  __shared__ __attribute__((aligned(16))) uint16_t lds[2 * KT * 2 * HD];
  __shared__ int s_place[5];
  __shared__ unsigned s_odd[kWaves];
  const int G = a.nh / a.nkv, nkv = a.nkv, bs = 1 << a.bs_log2;
  // kv heads side by side: with eight of them each has an XCD's L2 to itself
  const int share = blockIdx.x / nkv, kvh = blockIdx.x - share * nkv;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (w == 0) {
    Seq first = sequence(a, lane, 0);
    int pad;
    const int len = share_of(a, first, lane, pad);
    const Place p = (long long)share * len > 0x7fffffff ? Place{-1, 0, 0} : place_of(a, first, lane, share * len, pad);
    if (lane == 0) {
      s_place[0] = p.mt;
      s_place[1] = p.seq;
      s_place[2] = p.step;
      s_place[3] = len;
      s_place[4] = pad;
    }
  }
  __syncthreads();
  int mt = __builtin_amdgcn_readfirstlane(s_place[0]), seq = __builtin_amdgcn_readfirstlane(s_place[1]);
  int step0 = __builtin_amdgcn_readfirstlane(s_place[2]), left = __builtin_amdgcn_readfirstlane(s_place[3]);
  const int pad = __builtin_amdgcn_readfirstlane(s_place[4]);
  if (mt < 0) return;
  const int most = (a.max_nodes * G + kRows - 1) / kRows;
  for (; left > 0; step0 = 0) {      // a sequence's row tile, or the part of it that is the share's
  Seq sq = sequence(a, seq, pad);
  while (sq.tiles <= mt) {
    if (++seq >= a.n_seqs) {
      seq = 0;
      if (++mt >= most) return;
    }
    sq = sequence(a, seq, pad);
  }
  const int q0 = sq.q0, nodes = sq.nodes, ctx = sq.ctx, dealt = min(sq.steps - step0, left);
  left -= dealt;
  // without the lead: steps [begin, end) of the sequence
  const int begin = max(step0 - kLead, 0), end = step0 + dealt - kLead;
  if (end <= begin) return;      // a lead alone: whoever has the next share begins
  const int kv_begin = min(begin * KT, ctx), kv_end = min(end * KT, ctx);
  const bool begins = begin == 0, whole = begins && end == sq.steps - kLead;
  const int* bt = a.tables + (size_t)seq * a.table_stride;

  const int lr = lane & 31, hh = lane >> 5;
  const int r = mt * kRows + 32 * w + lr, node = r / G, head = kvh * G + r - node * G;
  const bool row_valid = node < nodes, wave_rows = mt * kRows + 32 * w < nodes * G;
  const int tree_key = ctx - nodes;      // the key of node 0
  const unsigned long long tmask = row_valid ? a.mask[(size_t)seq * a.mask_stride + node] : 0;

  constexpr int NS = HD / 16, ND = HD / 32, CH = HD / 8;
  const float scale = a.scale_log2 == 0.f ? 1.f : fabsf(a.scale_log2);
  float m_run = kLowest, l_run = 0.f;
  bool huge = false;      // the wave's maxima
  f32x16 o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[d][i] = 0.f;

  // A wave stages RW rows of a tile, 1 KB a load; in pages of at least RW tokens they lie side by side, so that its loads share an
  // id and an address.  The swizzle is in which chunk of its row a lane loads.
  const size_t head_stride = (size_t)bs * HD;
  constexpr int RW = KT / kWaves, NP = RW * CH / 64;
  const int row0 = w * RW;
  const bool whole_rows = bs >= RW;
  int k_at[NP], v_at;
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const int row = p * (64 / CH) + lane / CH;
    k_at[p] = 2 * (row * HD + 8 * k_slot<HD>(row0 + row, lane % CH)) - 1024 * p;
  }
  v_at = 2 * (lane / CH * HD + 8 * v_slot<HD>(row0 + lane / CH, lane % CH));
  int none = 0;
  asm("" : "+v"(none));                   // a vector load: a scalar one's wait would be one for all reads of LDS
  auto known = [&](int id) __attribute__((always_inline)) { return (unsigned)id < (unsigned)a.num_blocks ? id : 0; };
  auto read_id = [&](int kb0) __attribute__((always_inline)) {
    return whole_rows ? bt[(min(kb0 + row0, kv_end - 1) >> a.bs_log2) + none] : bt[min(kb0 + row0 + lane % RW, kv_end - 1) >> a.bs_log2];
  };
  auto full = [&](int kb0) __attribute__((always_inline)) { return whole_rows && kb0 + KT <= kv_end; };
  __amdgpu_buffer_rsrc_t k_rows, v_rows;
  auto at_page = [&](int id, int key) __attribute__((always_inline)) {
    const size_t from = ((size_t)known(__builtin_amdgcn_readfirstlane(id)) * nkv + kvh) * head_stride + (size_t)(key & (bs - 1)) * HD;
    k_rows = __builtin_amdgcn_make_buffer_rsrc((void*)(a.k + from), 0, RW * HD * 2, 0x00027000);
    v_rows = __builtin_amdgcn_make_buffer_rsrc((void*)(a.v + from), 0, RW * HD * 2, 0x00027000);
  };
  auto load = [&](auto l_, int stage) __attribute__((always_inline)) {
    constexpr int l = decltype(l_)::value, p = l < NP ? l : l - NP;
    const lds_ptr at = (lds_ptr)(lds + stage * KT * 2 * HD + (l < NP ? 0 : KT * HD) + row0 * HD);
    load_chunk<1024 * p>(l < NP ? k_rows : v_rows, l < NP ? k_at[p] : v_at, at);
  };
  // a tile that ends early, or whose rows have several pages: each lane finds its own, no row is after the last key
  auto load_part = [&](int kb0, int stage, int id) __attribute__((always_inline)) {
    const lds_ptr kl = (lds_ptr)(lds + stage * KT * 2 * HD + row0 * HD), vl = (lds_ptr)(lds + stage * KT * 2 * HD + KT * HD + row0 * HD);
    int part_lane = lane;
    asm volatile("" : "+v"(part_lane));      // computed here: kept from before the loop its addresses would cost registers
    const int first = min(kb0 + row0, kv_end - 1), last = kv_end - 1 - first;
    if (whole_rows) {
      at_page(id, first);
#pragma unroll 1
      for (int p = 0; p < NP; ++p) {
        const int row = p * (64 / CH) + part_lane / CH;
        load_chunk<0>(k_rows, 2 * (min(row, last) * HD + 8 * k_slot<HD>(row0 + row, part_lane % CH)), kl + p * 1024);
        load_chunk<0>(v_rows, 2 * (min(row, last) * HD + 8 * v_slot<HD>(row0 + row, part_lane % CH)), vl + p * 1024);
      }
      return;
    }
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const int row = p * (64 / CH) + part_lane / CH;
      const size_t from = ((size_t)known(__shfl(id, row, 64)) * nkv + kvh) * head_stride + (size_t)(min(kb0 + row0 + row, kv_end - 1) & (bs - 1)) * HD;
      load_chunk((const char*)(a.k + from + 8 * k_slot<HD>(row0 + row, part_lane % CH)), kl + p * 1024);
      load_chunk((const char*)(a.v + from + 8 * v_slot<HD>(row0 + row, part_lane % CH)), vl + p * 1024);
    }
  };
  // The first tile's page id, the queries, a look at the run's pages, then the first tile: three round trips, not one behind the other.
  int id = kv_end > kv_begin ? read_id(kv_begin) : 0;
  u32x4 qf[NS];
  const uint16_t* qp = a.q + (size_t)(q0 + (row_valid ? node : 0)) * a.q_stride + (row_valid ? head : 0) * HD;
#pragma unroll
  for (int s = 0; s < NS; ++s) qf[s] = row_valid ? *reinterpret_cast<const u32x4*>(qp + 16 * s + 8 * hh) : u32x4{0, 0, 0, 0};
  // a page that is not in the cache: its keys are not there, page 0 is read in its place
  bool bad = false;
  for (int e = (kv_begin >> a.bs_log2) + tid; e < (kv_end + bs - 1) >> a.bs_log2; e += kWaves * 64) bad = bad || (unsigned)bt[e] >= (unsigned)a.num_blocks;
  bad = __syncthreads_or(bad);      // and all have read the LDS of the part before
  if (kv_end > kv_begin) {
    if (full(kv_begin)) {
      at_page(id, kv_begin + row0);
      each<0, 2 * NP>([&](auto l) __attribute__((always_inline)) { load(l, 0); });
    } else load_part(kv_begin, 0, id);
    id = read_id(kv_begin + KT);
  }
  // the softmax takes maxima of raw scores, and unseen keys are -inf: a negative scale is the query's sign, zero a query of zeros (no number
  // where it is infinite or none)
  if (a.scale_log2 <= 0.f) {
#pragma unroll
    for (int s = 0; s < NS; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = qf[s][j], none = ((x & 0x7f80u) == 0x7f80u ? 0x7fc0u : 0u) | ((x & 0x7f800000u) == 0x7f800000u ? 0x7fc00000u : 0u);
        qf[s][j] = a.scale_log2 == 0.f ? none : x ^ 0x80008000u;
      }
  }
  // LDS addresses of this lane's operands in stage 0: keys lr, dims 16 s + 8 hh ..; values of dims 32 d .., keys 4 hh + tq
  typedef __attribute__((address_space(3))) const char* lds_at;
  lds_at ka[NS], va[ND];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    ka[s] = (lds_at)(lds + k_off<HD>(lr, 2 * s + hh));
    asm("" : "+v"(ka[s]));
  }
#pragma unroll
  for (int d = 0; d < ND; ++d) {
    const int col = 32 * d + 16 * ((lane >> 4) & 1) + 4 * (lane & 3);
    va[d] = (lds_at)(lds + KT * HD + v_off<HD>(4 * hh + ((lane & 15) >> 2), col >> 3) + (col & 7));
    asm("" : "+v"(va[d]));
  }

  auto step = [&](int kb0, auto stage_) __attribute__((always_inline)) {
    constexpr int stage = decltype(stage_)::value, at = stage * KT * 2 * HD * 2;
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): this wave's loads of the tile
    __syncthreads();                      // everybody's; and the other stage has been read
    const bool next = full(kb0 + KT);
    if (next) {
      at_page(id, kb0 + KT + row0);
      each<0, 2 * NP>([&](auto l) __attribute__((always_inline)) { load(l, 1 - stage); });
    } else if (kb0 + KT < kv_end) load_part(kb0 + KT, 1 - stage, id);
    id = read_id(kb0 + 2 * KT);
    // Values of the tree's keys that are infinite or no numbers reach the rows that see them alone, and those that stand for keys that are
    // not there reach none, but zero times such a value is no number: they are taken out of the tile here and added below for the rows that
    // see them.
    unsigned long long odd = 0;
    if (kb0 + KT > tree_key || bad) {
      // a wave looks at the rows that it staged; row r of the tile is bit r
      uint16_t* vt = lds + stage * KT * 2 * HD + KT * HD + row0 * HD;
      unsigned mine = 0;
      u32x4 x[NP];
#pragma unroll
      for (int p = 0; p < NP; ++p) x[p] = *reinterpret_cast<const u32x4*>(vt + p * 512 + lane * 8);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        bool is = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool lo_odd = (x[p][j] & 0x7f80u) == 0x7f80u, hi_odd = (x[p][j] & 0x7f800000u) == 0x7f800000u;
          is = is || lo_odd || hi_odd;
          x[p][j] &= (lo_odd ? 0xffff0000u : ~0u) & (hi_odd ? 0xffffu : ~0u);
        }
        const unsigned long long b = __ballot(is);
        if (b) {
          *reinterpret_cast<u32x4*>(vt + p * 512 + lane * 8) = x[p];
#pragma unroll
          for (int i = 0; i < 64 / CH; ++i) mine |= (b >> (i * CH) & ((1ull << CH) - 1)) ? 1u << (p * (64 / CH) + i) : 0u;
        }
      }
      if (lane == 0) s_odd[w] = mine;
      __syncthreads();
#pragma unroll
      for (int i = 0; i < kWaves; ++i) odd |= (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane(s_odd[i]) << (RW * i);
    }
    if (!wave_rows) return;
    // ---- S^T = K Q^T for two 32-key blocks: the first block's operands all under way before its products, the second's between them,
    // the first values between the second's
    f32x16 sc[2];
    auto read_v = [&](int j, int d) __attribute__((always_inline)) {
      const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(va[d] + (at + 32 * HD * j)));
      const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_short4*)(va[d] + (at + 32 * HD * j + 16 * HD)));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    auto read_k = [&](int kb, int s) __attribute__((always_inline)) {
      return *(const __attribute__((address_space(3))) bf16x8*)(ka[s] + (at + 64 * HD * kb));
    };
    typedef short short8v __attribute__((ext_vector_type(8)));
    short8v vf[2][ND];
    {
      bf16x8 kf[NS];
#pragma unroll
      for (int s = 0; s < NS; ++s) kf[s] = read_k(0, s);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kb][i] = 0.f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
          sc[kb] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf[s], as_bf16x8(qf[s]), sc[kb], 0, 0, 0);
          if (kb == 0) kf[s] = read_k(1, s);
          else {
#pragma unroll
            for (int f = s * 2 * ND / NS; f < (s + 1) * 2 * ND / NS; ++f) vf[f / ND][f % ND] = read_v(f / ND, f % ND);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    }
    // ---- online softmax; lane owns row lr, keys kb0 + 32 kb + (i & 3) + 8 (i >> 2) + 4 hh
    if (kb0 + KT > tree_key || kb0 + KT > kv_end || bad) {
      const int key0 = kb0 + 4 * hh;
      const int lim = kv_end - 1 - key0, t = tree_key - key0;      // last key; keys before t are seen, after it as the mask says
      unsigned long long see = lim < 0 ? 0 : lim >= 63 ? ~0ull : (2ull << lim) - 1;
      see &= t >= 64 ? ~0ull : t >= 0 ? (tmask << t) | ((1ull << t) - 1) : t > -64 ? tmask >> -t : 0ull;
      if (bad) see &= __ballot((unsigned)bt[min(kb0 + lane, kv_end - 1) >> a.bs_log2] < (unsigned)a.num_blocks) >> (4 * hh);
      const unsigned see_lo = (unsigned)see, see_hi = (unsigned)(see >> 32);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[kb][i] = (kb ? see_hi : see_lo) >> ((i & 3) + 8 * (i >> 2)) & 1 ? sc[kb][i] : -__builtin_inff();
    }
    float mx = -__builtin_inff();
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[kb][i]);
    mx *= scale;
    // the sums are scaled anew only where the maximum grows by more than 8 (weights stay below 2^8)
    if (__any(mx > m_run + 8.f)) {
      mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
      const float m_new = fmaxf(m_run, mx);
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_new);
      l_run *= alpha;
#pragma unroll
      for (int d = 0; d < ND; ++d) o[d] *= alpha;
      m_run = m_new;
      huge = __any(fabsf(m_run) > 0x1p24f && m_run != kLowest);
    }
    // A score's product with the scale is not rounded before the maximum, which is, is taken off: where half a last place of that is much, the
    // difference is made ahead.
    const float scale_now = huge ? 1.f : scale, m_now = huge ? 0.f : m_run;
    if (huge) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float x = sc[kb][i] * scale;
          asm("" : "+v"(x));
          sc[kb][i] = x - m_run;
        }
    }
    float ps[4];
    u32x4 pf;
    auto weight = [&](int kb, int i) __attribute__((always_inline)) {
      sc[kb][i] = __builtin_amdgcn_exp2f(sc[kb][i] * scale_now - m_now);
      ps[i & 3] = kb == 0 && i < 4 ? sc[kb][i] : ps[i & 3] + sc[kb][i];
    };
#pragma unroll
    for (int i = 0; i < 16; ++i) weight(0, i);
    __builtin_amdgcn_sched_barrier(0);
    each<0, 4 * ND>([&](auto i_) __attribute__((always_inline)) {
      constexpr int i = decltype(i_)::value, j = i / ND, d = i % ND;
      if constexpr (d == 0) {
#pragma unroll
        for (int jj = 0; jj < 4; ++jj) pf[jj] = pack_bf16x2(sc[j >> 1][8 * (j & 1) + 2 * jj], sc[j >> 1][8 * (j & 1) + 2 * jj + 1]);
      }
      o[d] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, vf[j & 1][d]), as_bf16x8(pf), o[d], 0, 0, 0);
      if constexpr (j < 2) {
        vf[j][d] = read_v(j + 2, d);
#pragma unroll
        for (int k = i * 8 / ND; k < (i + 1) * 8 / ND; ++k) weight(1, k);
      }
      __builtin_amdgcn_sched_barrier(0);
    });
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    // ---- what was taken out of the tile
    while (odd) {
      const int kk = __ffsll(odd) - 1, key = kb0 + kk;
      odd &= odd - 1;
      if (key >= kv_end) break;
      float p = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i)
        if (i == ((kk >> 5) << 4 | (kk >> 3 & 3) << 2 | (kk & 3))) p = sc[i >> 4][i & 15];
      p = __shfl(p, lr + 32 * (kk >> 2 & 1), 64);
      const int id = bt[key >> a.bs_log2], node = key - tree_key;
      const bool sees = known(id) == id && (node < 0 || (tmask >> node & 1));
      const uint16_t* vp = a.v + ((size_t)known(id) * nkv + kvh) * head_stride + (size_t)(key & (bs - 1)) * HD;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint16_t x = vp[32 * d + 8 * (i >> 2) + 4 * hh + (i & 3)];
          if (sees && (x & 0x7f80) == 0x7f80) o[d][i] += p * bf16_to_f32(x);
        }
    }
  };
  for (int kb0 = kv_begin; kb0 < kv_end; kb0 += 2 * KT) {
    step(kb0, ic<0>{});
    if (kb0 + KT < kv_end) step(kb0 + KT, ic<1>{});
  }
  l_run += __shfl_xor(l_run, 32, 64);
  const float inv = l_run == 0.f ? 0.f : 1.f / l_run;
  if (row_valid && whole) {
    uint16_t* op = a.out + (size_t)(q0 + node) * a.out_stride + head * HD;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint2 x;
        x.x = pack_bf16x2(o[d][4 * i] * inv, o[d][4 * i + 1] * inv);
        x.y = pack_bf16x2(o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv);
        *reinterpret_cast<uint2*>(op + 32 * d + 8 * i + 4 * hh) = x;
      }
  } else if (row_valid) {
    // a share has one part at most that a share before has begun, and one that it begins and does not end
    const size_t at = ((size_t)blockIdx.x * 2 + begins) * kRows + 32 * w + lr;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        *reinterpret_cast<f32x4*>(a.part_o + at * HD + 32 * d + 8 * i + 4 * hh) =
            f32x4{o[d][4 * i] * inv, o[d][4 * i + 1] * inv, o[d][4 * i + 2] * inv, o[d][4 * i + 3] * inv};
    if (hh == 0) a.part_l[at] = l_run == 0.f ? -__builtin_inff() : m_run + __builtin_amdgcn_logf(l_run);
  }
  ++seq;
  }
}

// The parts of a sequence's row tile that several shares have, weighed by their sums: HD / 8 lanes a row, several parts under way.  Two rows
// one after another (16 trees of 60 nodes, 64 heads on 8, 1000 to 8000 keys, all launches: 174 us; one row and eight parts at a time: 182), or,
// where a row has eight parts and more, four groups of lanes a row, a quarter of its parts each (one tree of 64 nodes, 32 heads on 8, 8000 keys: 33 us,
// not 43; but 6 of 49 over 290, with five parts, 34, not 25).
template <int HD, int WAYS>
__global__ __launch_bounds__(256) void tree_parts_kernel(Args a) {
  constexpr int L = HD / 8, R = 256 / L / WAYS, TURNS = WAYS == 1 ? 2 : 1;
  const int G = a.nh / a.nkv, most = (a.max_nodes * G + kRows - 1) / kRows;
  const int unit = blockIdx.x / a.nkv, kvh = blockIdx.x - unit * a.nkv, seq = unit / most, mt = unit - seq * most;
  const int lane = threadIdx.x & 63, way = threadIdx.x / L % WAYS;
  Seq first = sequence(a, lane, 0);
  int pad;
  const int len = share_of(a, first, lane, pad);
  const Seq sq = sequence(a, seq, pad);
  if (sq.tiles <= mt) return;
  const int from = steps_before(a, first, lane, mt, seq, pad), to = from + sq.steps - 1, s0 = (from + kLead) / len, s1 = to / len;
  if (s0 == s1) return;
  for (int turn = 0; turn < TURNS; ++turn) {
    const int in_tile = (TURNS * blockIdx.y + turn) * R + threadIdx.x / (L * WAYS), r = mt * kRows + in_tile, node = r / G, d = threadIdx.x % L * 8;
    if (node >= sq.nodes) break;
    // the first part is one that its share begins, the others are not
    auto at = [&](int s) { return ((size_t)(s * a.nkv + kvh) * 2 + (s == s0)) * kRows + in_tile; };
    constexpr int U = 4;
    float M = -__builtin_inff(), W = 0.f, acc[8] = {};
    for (int s = s0 + way * U; s <= s1; s += U * WAYS) {
      float l[U], m = M;
      bool any = false;
      f32x4 x[U], y[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const size_t p = at(min(s + u, s1));
        l[u] = a.part_l[p];
        x[u] = *reinterpret_cast<const f32x4*>(a.part_o + p * HD + d);
        y[u] = *reinterpret_cast<const f32x4*>(a.part_o + p * HD + d + 4);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (s + u > s1) l[u] = -__builtin_inff();
        m = fmaxf(m, l[u]);
        any = any || l[u] != -__builtin_inff();      // a sum that is no number is not of the maximum, and stays
      }
      if (!any) continue;
      const float old = exp2f(M - m);
      M = m;
      W *= old;
#pragma unroll
      for (int j = 0; j < 8; ++j) acc[j] *= old;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float wgt = exp2f(l[u] - M);
        W += wgt;
        if (l[u] == -__builtin_inff()) continue;      // a part without keys
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          acc[j] += wgt * x[u][j];
          acc[4 + j] += wgt * y[u][j];
        }
      }
    }
    if constexpr (WAYS > 1) {
#pragma unroll
      for (int o = L; o < L * WAYS; o <<= 1) {
        const float other = __shfl_xor(M, o, 64), m = fmaxf(M, other), w = __shfl_xor(W, o, 64);
        const float mine = W == 0.f ? 0.f : exp2f(M - m), theirs = w == 0.f ? 0.f : exp2f(other - m);      // zero: no keys
        W = W * mine + w * theirs;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float x = __shfl_xor(acc[j], o, 64);
          acc[j] = acc[j] * mine + x * theirs;
        }
        M = m;
      }
      if (way > 0) continue;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = W == 0.f ? 0.f : acc[j] / W;
    *reinterpret_cast<u32x4*>(a.out + (size_t)(sq.q0 + node) * a.out_stride + (kvh * G + r - node * G) * HD + d) = pack8(acc);
  }
}

template <int HD>
int launch(const Args& a, hipStream_t s) {
  tree_tiles_kernel<HD><<<a.shares * a.nkv, kWaves * 64, 0, s>>>(a);
  DGI_CHECK_LAUNCH();
  if (a.shares > 1) {
    const int most = (a.max_nodes * (a.nh / a.nkv) + kRows - 1) / kRows;
    const int units = a.n_seqs * most * a.nkv, groups = kRows * HD / 8 / 256;
    if (a.shares < 8 * a.n_seqs * most) tree_parts_kernel<HD, 1><<<dim3(units, groups / 2), 256, 0, s>>>(a);
    else tree_parts_kernel<HD, 4><<<dim3(units, groups * 4), 256, 0, s>>>(a);
    DGI_CHECK_LAUNCH();
  }
  return 0;
}

}  // namespace

extern "C" int dgi_tree_tiles(const void* q, long long q_stride, const void* k, const void* v, const int* tables, int table_stride,
                              int table_cols, int n_seqs, int num_blocks, int rows, const int* cu, const int* ctx, const void* mask,
                              int mask_stride, int max_nodes, void* out, long long out_stride, float* part_o, float* part_l, int shares,
                              int least, int nh, int nkv, int hd, int block_size, float scale, hipStream_t s) {
  if (n_seqs == 0 || rows == 0) return 0;
  Args a{(const uint16_t*)q, q_stride, (const uint16_t*)k, (const uint16_t*)v, tables, table_stride, table_cols, n_seqs, num_blocks, rows, cu, ctx,
         (const unsigned long long*)mask, mask_stride, max_nodes, (uint16_t*)out, out_stride, part_o, part_l, shares, least, nh, nkv, 0,
         scale * 1.4426950408889634f};
  while ((1 << a.bs_log2) < block_size) ++a.bs_log2;
  if (hd == 64) return launch<64>(a, s);
  if (hd == 128) return launch<128>(a, s);
  return -5;
}
