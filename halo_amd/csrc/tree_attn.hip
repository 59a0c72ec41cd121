// Attention of drafted token trees over a paged cache (gfx950, wave64).
//
// Node i of request b (row cu[b] + i of q) sees the request's committed rows
// 0 .. length_b - 1 and, of the tree's own rows length_b + j, those whose bit
// j is set in the node's mask (its ancestors and itself; without masks the
// nodes j <= i):
//   s_ij = scale q_i . k_j,   out_i = sum_j e^(s_ij) v_j / sum_j e^(s_ij),
//   lse_i = log sum_j e^(s_ij),
// one pass over the rows with a running maximum and sum.  A row that a node
// does not see has no part in it whatever it holds, NaN and infinities
// included; a node that sees nothing gives out 0 and lse -inf.  The reference
// verifies no drafted tokens; the nearest path is its chunk walk
// (halo/kv_cache_chunked.py:864-964).
//
// Work.  The query heads of a KV head and the nodes are flattened, row
// r = (node r / rep, head r % rep); a unit is (request, KV head, block of
// rows), so each K/V row is read once for all the heads and nodes of a block.
// A request's key tiles are its committed rows in steps of KT from row 0 and
// its tree rows in steps of KT from row length_b, so a tree tile meets whole
// words of the masks.  The lengths are on the device only: every workgroup
// sums the units' tiles, takes the share L = total / workgroups that fit the
// GPU, and finds its item, one of ceil(tiles / L) even cuts of a unit; a
// second launch merges the partials of the units that were cut.  The host
// needs no lengths and a captured call follows them.
#include <type_traits>

#include "block_pool.hpp"
#include "mfma.hpp"

namespace halo {

struct TreeParams {
  const void* q;
  int64_t q_stride_n, q_stride_h;  // elements
  const char* k;
  const char* v;
  uint32_t sb, sh, sr;  // pool strides in 16-byte pieces
  int blocks;
  Div bs;
  const int32_t* table;
  int64_t table_stride;
  int W;
  const int32_t* lengths;
  const int32_t* cu;
  const uint32_t* mask;  // 32-bit words, or null
  int64_t mask_stride;
  int B, H, H_kv, rep, N, max_nodes;
  int slots, min_tiles;  // workgroups that the GPU holds; shortest item worth its merge
  float scale2;
  void* out;
  int64_t o_stride_n, o_stride_h;
  int out_dtype, out_vec4;
  float* lse;
  float4* part_o;
  float2* part_ml;
};

// Slack (log2 units) by which a tile's max may exceed the running max before
// the running max moves (probabilities stay below 2^8).
constexpr float kTreeLazyMax = 8.0f;

struct TreeReq {
  int lo, ctx, n, rbs, tiles;
};
template <int KT, int R>
__device__ __forceinline__ TreeReq tree_req(const TreeParams& P, int b) {
  TreeReq r = {0, 0, 0, 0, 0};
  if (b < P.B) {
    r.lo = max(P.cu[b], 0);
    r.n = max(min(min(P.cu[b + 1], P.N) - r.lo, P.max_nodes), 0);
    r.ctx = min(max(P.lengths[b], 0), P.W * P.bs.d);
    r.rbs = (r.n * P.rep + R - 1) / R;
    if (r.n > 0) r.tiles = (r.ctx + KT - 1) / KT + (r.n + KT - 1) / KT;
  }
  return r;
}

// One item (or, for the merge, one unit) of the launch.
struct TreeItem {
  int b, lo, ctx, n, rbs, tiles;
  int h, rb, cut, cuts;  // the cut-th of `cuts` cuts of the unit (h, rb)
  int64_t part;          // partial of the unit's first cut
};

// Every lane returns the same; false past the last item.  ITEMS: x counts
// items (head, cut, row block; the row blocks that read the same rows side by
// side), else units (row block, head).
template <int KT, int R, bool ITEMS>
__device__ __forceinline__ bool tree_find(const TreeParams& P, int x, TreeItem& it) {
  const int lane = threadIdx.x & 63;
  const TreeReq r0 = tree_req<KT, R>(P, lane);
  int64_t total = 0;
  int units = 0;
  for (int b0 = 0; b0 < P.B; b0 += 64) {
    const TreeReq r = b0 == 0 ? r0 : tree_req<KT, R>(P, b0 + lane);
    int u = P.H_kv * r.rbs;
    int64_t t = (int64_t)u * r.tiles;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
      u += __shfl_xor(u, off, 64);
      t += __shfl_xor(t, off, 64);
    }
    units += u;
    total += t;
  }
  // sum of ceil(tiles / L) <= total / L + units: a share that fills the GPU once if the units leave room
  const int room = P.slots > 2 * units ? P.slots - units : P.slots / 2;
  const int L = max(P.min_tiles, (int)min((total + room - 1) / room, (int64_t)0x7fffffff));
  int base = 0;
  int64_t part = 0;
  for (int b0 = 0; b0 < P.B; b0 += 64) {
    const TreeReq r = b0 == 0 ? r0 : tree_req<KT, R>(P, b0 + lane);
    const int cuts = (int)(((int64_t)r.tiles + L - 1) / L);
    const int u = P.H_kv * r.rbs;
    const int mine = ITEMS ? u * cuts : u;
    int at = mine;
    int64_t parts = cuts > 1 ? (int64_t)u * cuts : 0;
    const int64_t own = parts;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int y = __shfl_up(at, off, 64);
      const int64_t z = __shfl_up(parts, off, 64);
      if (lane >= off) {
        at += y;
        parts += z;
      }
    }
    const uint64_t past = __ballot(base + at > x);
    if (past != 0) {
      const int w = __builtin_ctzll(past);
      const int first = uni(base + __shfl(at - mine, w, 64));
      it.b = b0 + w;
      it.lo = uni(__shfl(r.lo, w, 64));
      it.ctx = uni(__shfl(r.ctx, w, 64));
      it.n = uni(__shfl(r.n, w, 64));
      it.rbs = uni(__shfl(r.rbs, w, 64));
      it.tiles = uni(__shfl(r.tiles, w, 64));
      it.cuts = uni(__shfl(cuts, w, 64));
      part = uni64(part + __shfl(parts - own, w, 64));
      const int y = x - first;
      it.cut = 0;
      if constexpr (ITEMS) {
        it.rb = y % it.rbs;
        it.cut = (y / it.rbs) % it.cuts;
        it.h = y / it.rbs / it.cuts;
      } else {
        it.h = y % P.H_kv;
        it.rb = y / P.H_kv;
      }
      it.part = part + (int64_t)(it.rb * P.H_kv + it.h) * it.cuts;
      return true;
    }
    base += uni(__shfl(at, 63, 64));
    part += uni64(__shfl(parts, 63, 64));
  }
  return false;
}

// Where row `key` of key tile `t` lies in the pool, in 16-byte pieces from the
// start of head 0, or kNoRow: behind the committed rows, behind the tree, past
// the table, or in a block that is not in the pool (a table entry outside
// [0, blocks): its rows are not attended).  In two steps, so that the table
// read can be in flight while other tiles are computed.
constexpr uint32_t kNoRow = 0xffffffffu;
template <int KT>
struct TreeRow {
  int blk, in_blk;
  __device__ __forceinline__ void load(const TreeParams& P, const TreeItem& it, int t, int key) {
    const int nc = (it.ctx + KT - 1) / KT;
    const int i = t < nc ? t * KT + key : (t - nc) * KT + key;  // committed or tree row
    const int pos = t < nc ? i : it.ctx + i;
    const int c = div_by(pos, P.bs);
    const bool ok = (t < nc ? i < it.ctx : i < it.n) && t < it.tiles && c < P.W;
    blk = -1;
    if (ok) blk = P.table[it.b * P.table_stride + c];
    in_blk = pos - c * P.bs.d;
  }
  __device__ __forceinline__ uint32_t place(const TreeParams& P) const {
    return blk >= 0 && blk < P.blocks ? (uint32_t)blk * P.sb + (uint32_t)in_blk * P.sr : kNoRow;
  }
};

// What rows that are not there read as.
__device__ uint4 tree_zeros[1];

// 16 bytes a lane from memory into the 1 KiB of LDS at `st` (lane l's piece at 16 l).
__device__ __forceinline__ void tree_dma(const char* from, char* st) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from),
                                   (__attribute__((address_space(3))) void*)(st), 16, 0, 0);
}

// Bits of the 32 tree rows from 32 w on that node i of the item's tree sees.
__device__ __forceinline__ uint32_t tree_bits(const TreeParams& P, const TreeItem& it, int i, int w) {
  if (P.mask != nullptr) return P.mask[(int64_t)(it.lo + i) * P.mask_stride + w];
  const int d = i - 32 * w;
  return d < 0 ? 0u : d >= 31 ? 0xffffffffu : (2u << d) - 1;
}

// A 16-bit operand's values that are not finite: which of a word's halves, as
// 0xffff; and operands with 1 where the value is `inf` or NaN.
template <int DT>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t E = DT == HALO_BF16 ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}
template <int DT>
__device__ __forceinline__ uint32_t is_halves(uint32_t w, bool minus) {
  constexpr uint32_t E = DT == HALO_BF16 ? 0x7f80u : 0x7c00u;
  constexpr uint32_t one = DT == HALO_BF16 ? 0x3f80u : 0x3c00u;
  const uint32_t other = minus ? E : (E | 0x8000u);  // the infinity that does not count
  const uint32_t odd = odd_halves<DT>(w);
  const uint32_t lo = (odd & 0xffffu) && (w & 0xffffu) != other ? one : 0u;
  const uint32_t hi = (odd >> 16) && (w >> 16) != other ? one << 16 : 0u;
  return lo | hi;
}

__device__ __forceinline__ void tree_store4(const TreeParams& P, int64_t at, const float* v4) {
  if (P.out_vec4) {
    store_elem4(P.out, at, P.out_dtype, v4);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) store_elem(P.out, at + j, P.out_dtype, v4[j]);
  }
}

// First channel of the four that piece x of lane half hh holds.  16-bit kernel,
// x = 4 db + i: MFMA row m of d-block db is channel (m / 16) D/2 + 16 db + m % 16,
// which spreads a transposed LDS read over all banks.  fp32 kernel, x = i D/32 + g:
// row m of block db is channel m D/32 + db, so a piece is four channels in a row.
template <int D, bool F32>
__device__ __forceinline__ int tree_channel(int x, int hh) {
  constexpr int DB = D / 32;
  if (F32) return (8 * (x / DB) + 4 * hh) * DB + 4 * (x % DB);
  const int m = 8 * (x & 3) + 4 * hh;
  return (m >> 4) * (D / 2) + 16 * (x >> 2) + (m & 15);
}

// A row's lse from its running maximum (log2 units) and sum; NaN stays NaN.
__device__ __forceinline__ float tree_lse(float m, float l) { return l == 0.f ? -INFINITY : (m + log2f(l)) * kLn2; }
__device__ __forceinline__ float tree_inv(float l) { return l == 0.f ? 0.f : 1.f / l; }

// Weight of a partial with maximum m where the largest is M: 0 where it saw nothing.
__device__ __forceinline__ float tree_weight(float m, float M) {
  return __builtin_amdgcn_exp2f(m - (M == -INFINITY ? 0.f : M));
}

constexpr int kTreeRows = 32;  // rows of a unit: the columns of one 32x32 product
constexpr int kTreeKT = 32;    // rows of a key tile
constexpr int kTreeWaves = 4;

// The four waves of a workgroup hold (m, l, o) of the same 32 rows over
// different tiles.  Each leaves its o in `mine` (16 KiB / 8 KiB at D = 128 / 64,
// pieces in its own register order) and folds a quarter of the pieces.
template <int D, bool F32>
__device__ __forceinline__ void tree_fold_store(const TreeParams& P, const TreeItem& it, int wave, int lane,
                                                float2 (*s_ml)[32], const char* const* o_of_wave) {
  constexpr int PIECES = D / 8, PER = PIECES / kTreeWaves;
  const int qc = lane & 31, hh = lane >> 5;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kTreeWaves; ++w) M = fmaxf(M, s_ml[w][qc].x);
  float wt[kTreeWaves], l = 0.f;
#pragma unroll
  for (int w = 0; w < kTreeWaves; ++w) {
    wt[w] = tree_weight(s_ml[w][qc].x, M);
    l += s_ml[w][qc].y * wt[w];
  }
  const int r = it.rb * kTreeRows + qc;
  if (r >= it.n * P.rep) return;
  const int node = r / P.rep, head = it.h * P.rep + (r - node * P.rep);
  const int64_t row = it.lo + node;
  const int64_t pu = it.part + it.cut;
  const float inv = tree_inv(l);
#pragma unroll
  for (int y = 0; y < PER; ++y) {
    const int x = wave * PER + y;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kTreeWaves; ++w) {
      const float4 a = *reinterpret_cast<const float4*>(o_of_wave[w] + (x * 64 + lane) * 16);
      v[0] += a.x * wt[w];
      v[1] += a.y * wt[w];
      v[2] += a.z * wt[w];
      v[3] += a.w * wt[w];
    }
    if (it.cuts > 1) {
      P.part_o[pu * (PIECES * 64) + x * 64 + lane] = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= inv;
      tree_store4(P, row * P.o_stride_n + head * P.o_stride_h + tree_channel<D, F32>(x, hh), v);
    }
  }
  if (wave == 0 && hh == 0) {
    if (it.cuts > 1) P.part_ml[pu * 32 + qc] = make_float2(M, l);
    else if (P.lse != nullptr) P.lse[row * P.H + head] = tree_lse(M, l);
  }
}

// 16-bit queries and pools, products on v_mfma_f32_32x32x16:
//   scores  S^T[key][row] = sum_d K[key][d] Q[row][d]          (A = K tile, B = Q^T)
//   output  O^T[d][row]  += sum_key V^T[d][key] P^T[key][row]  (A = V^T, B = P^T)
// S^T's accumulator gives lane (row, half h) the keys 8i + 4h + j, which are the
// keys of its P^T operands, so p goes to the second product (rounded to the
// pool's type, at most half a step of it) without a cross-lane move.  Each wave
// streams tiles of its own, every fourth of the item's, through two LDS stages
// of its own: no barrier in the loop.
template <int DT, int D>
__global__ void __launch_bounds__(256) tree_attn_kernel(TreeParams P) {
  constexpr int KS = D / 16, DB = D / 32, RB = D * 2, SL = RB / 16;
  constexpr int TB = kTreeKT * RB;  // bytes of a K or V tile
  constexpr int RPI = 1024 / RB;    // rows of one 1 KiB LDS-DMA instruction
  constexpr int NI = TB / 1024;
  __shared__ __attribute__((aligned(16))) char sA[kTreeWaves][2 * TB], sB[kTreeWaves][2 * TB];  // stage: K, then V
  __shared__ float2 s_ml[kTreeWaves][32];
  TreeItem it;
  if (!tree_find<kTreeKT, kTreeRows, true>(P, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int t_end = (int)((int64_t)it.tiles * (it.cut + 1) / it.cuts);
  const int t0 = (int)((int64_t)it.tiles * it.cut / it.cuts) + wave;
  const int nc = (it.ctx + kTreeKT - 1) / kTreeKT;

  const int r_eff = min(it.rb * kTreeRows + qc, it.n * P.rep - 1);
  const int node = r_eff / P.rep, head = it.h * P.rep + (r_eff - node * P.rep);
  uint4 qb[KS];  // lane (row, half): channels 16 s + 8 half .. + 8
  {
    const char* qrow =
        reinterpret_cast<const char*>(P.q) + ((it.lo + node) * P.q_stride_n + head * P.q_stride_h) * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const uint4*>(qrow + (s * 16 + hh * 8) * 2);
  }
  const char* kh = P.k + (int64_t)it.h * P.sh * 16;
  const char* vh = P.v + (int64_t)it.h * P.sh * 16;

  auto kswz = [](int r) { return RB == 256 ? (r & 15) : ((r >> 1) & 7); };
  auto vswz = [](int r) { return RB == 256 ? 2 * (r & 3) : 2 * ((r >> 1) & 1); };
  // Each instruction fills RPI rows, lane l the slot l % SL of row l / SL with the piece that belongs there.
  auto issue = [&](uint32_t place, char* st) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = j * RPI + lane / SL, slot = lane % SL;
      const uint32_t at = __shfl(place, row, 64);
      const char* k = at == kNoRow ? reinterpret_cast<const char*>(tree_zeros)
                                   : kh + (int64_t)at * 16 + ((slot ^ kswz(row)) << 4);
      const char* v = at == kNoRow ? reinterpret_cast<const char*>(tree_zeros)
                                   : vh + (int64_t)at * 16 + ((slot ^ vswz(row)) << 4);
      tree_dma(k, st + j * 1024);
      tree_dma(v, st + TB + j * 1024);
    }
  };
  auto kread = [&](const char* st, int s) {
    return *reinterpret_cast<const uint4*>(st + qc * RB + (((2 * s + hh) ^ kswz(qc)) << 4));
  };
  const int vG = lane >> 4, vei = (lane & 15) >> 2, vai = lane & 3;
  auto vread = [&](const char* st, int i) {
    const int t = i / DB, db = i % DB;
    const int rlo = 16 * t + 4 * (vG >> 1) + vei, rhi = rlo + 8;
    const int byte = ((vG & 1) * (D / 2) + 16 * db + 4 * vai) * 2;
    const int pc = byte >> 4, wi = byte & 15;
    const uint2 a0 = pf_tr16(st + TB + rlo * RB + ((pc ^ vswz(rlo)) << 4) + wi);
    const uint2 a1 = pf_tr16(st + TB + rhi * RB + ((pc ^ vswz(rhi)) << 4) + wi);
    return make_uint4(a0.x, a0.y, a1.x, a1.y);
  };

  pf32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pf32x16{};
  float m_run = -INFINITY, l_run = 0.f;

  // a tile's rows that are there, and of those the ones that this lane's row sees
  struct Tile {
    uint32_t there, bits;
  };
  auto open = [&](const TreeRow<kTreeKT>& row, int t, char* st) {
    Tile x;
    const uint32_t place = row.place(P);
    x.there = (uint32_t)__ballot(place != kNoRow);
    x.bits = x.there;
    if (t >= nc) x.bits &= tree_bits(P, it, node, t - nc);
    issue(place, st);
    return x;
  };
  auto compute = [&](const Tile& x, int t, const char* st) {
    pf32x16 S = pf32x16{};
#pragma unroll
    for (int s = 0; s < KS; ++s) S = PMfma<DT>::run(kread(st, s), qb[s], S);
    const uint32_t mine = x.bits >> (4 * hh);
    if (__ballot(x.bits != 0xffffffffu)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = (mine >> (8 * (e >> 2) + (e & 3))) & 1 ? S[e] : -INFINITY;
    }
    float bm = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) bm = fmaxf(bm, S[e]);
    bm = half_max(bm) * P.scale2;  // scale > 0
    const float m_old = m_run;
    m_run = bm > m_old + kTreeLazyMax ? bm : m_old;
    const float ms = m_run == -INFINITY ? 0.f : m_run;
    if (__ballot(m_run != m_old)) {
      const float alpha = m_run != m_old ? __builtin_amdgcn_exp2f(m_old - m_run) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    float p[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e], P.scale2, -ms));
      l_run += p[e];
    }
    uint4 pb[2];  // step t: keys 16 t + {4 h + j, 8 + 4 h + j}
#pragma unroll
    for (int u = 0; u < 2; ++u)
      pb[u] = make_uint4(PMfma<DT>::pack(p[8 * u], p[8 * u + 1]), PMfma<DT>::pack(p[8 * u + 2], p[8 * u + 3]),
                         PMfma<DT>::pack(p[8 * u + 4], p[8 * u + 5]), PMfma<DT>::pack(p[8 * u + 6], p[8 * u + 7]));
    // Tree rows that some nodes see and others do not: 0 x inf is not 0, so
    // values that are not finite are kept out of the product and reach the
    // rows that see them only.
    bool odd = false;
    if (t >= nc) {
      uint32_t any = 0;
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        const uint4 v = vread(st, i);
        any |= odd_halves<DT>(v.x) | odd_halves<DT>(v.y) | odd_halves<DT>(v.z) | odd_halves<DT>(v.w);
      }
      odd = __ballot(any != 0) != 0;
    }
    if (!odd) {
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) o[i % DB] = PMfma<DT>::run(vread(st, i), pb[i / DB], o[i % DB]);
      return;
    }
    uint4 sees[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = (mine >> (8 * ((8 * u + e) >> 2) + (e & 3))) & 1 ? 1.f : 0.f;
      sees[u] = make_uint4(PMfma<DT>::pack(f[0], f[1]), PMfma<DT>::pack(f[2], f[3]), PMfma<DT>::pack(f[4], f[5]),
                           PMfma<DT>::pack(f[6], f[7]));
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      pf32x16 plus = pf32x16{}, minus = pf32x16{};
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const uint4 v = vread(st, u * DB + db);
        const uint4 f = make_uint4(v.x & ~odd_halves<DT>(v.x), v.y & ~odd_halves<DT>(v.y),
                                   v.z & ~odd_halves<DT>(v.z), v.w & ~odd_halves<DT>(v.w));
        o[db] = PMfma<DT>::run(f, pb[u], o[db]);
        const uint4 a = make_uint4(is_halves<DT>(v.x, false), is_halves<DT>(v.y, false), is_halves<DT>(v.z, false),
                                   is_halves<DT>(v.w, false));
        const uint4 c = make_uint4(is_halves<DT>(v.x, true), is_halves<DT>(v.y, true), is_halves<DT>(v.z, true),
                                   is_halves<DT>(v.w, true));
        plus = PMfma<DT>::run(a, sees[u], plus);
        minus = PMfma<DT>::run(c, sees[u], minus);
      }
#pragma unroll
      for (int e = 0; e < 16; ++e) o[db][e] += (plus[e] > 0.f ? INFINITY : 0.f) + (minus[e] > 0.f ? -INFINITY : 0.f);
    }
  };

  TreeRow<kTreeKT> ra, rb;
  Tile ta = {0, 0}, tb = {0, 0};
  const int key = lane & 31;
  char* const stA = sA[wave];
  char* const stB = sB[wave];
  ra.load(P, it, t0, key);
  rb.load(P, it, t0 + kTreeWaves, key);
  if (t0 < t_end) ta = open(ra, t0, stA);
  if (t0 + kTreeWaves < t_end) tb = open(rb, t0 + kTreeWaves, stB);
  for (int t = t0; t < t_end; t += 2 * kTreeWaves) {
    const int t1 = t + kTreeWaves, t2 = t + 2 * kTreeWaves, t3 = t + 3 * kTreeWaves;
    ra.load(P, it, t2, key);
    rb.load(P, it, t3, key);
    __builtin_amdgcn_s_waitcnt(0);
    compute(ta, t, stA);
    if (t2 < t_end) ta = open(ra, t2, stA);
    if (t1 < t_end) {
      __builtin_amdgcn_s_waitcnt(0);
      compute(tb, t1, stB);
      if (t3 < t_end) tb = open(rb, t3, stB);
    }
  }
  // o to LDS: the pieces below NI over the stage A, the others over the stage B
  const float lt = half_sum(l_run);
  if (hh == 0) s_ml[wave][qc] = make_float2(m_run, lt);
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<float4*>(stA + ((db * 4 + i) * 64 + lane) * 16) =
          make_float4(o[db][4 * i], o[db][4 * i + 1], o[db][4 * i + 2], o[db][4 * i + 3]);
  __syncthreads();
  const char* ow[kTreeWaves] = {sA[0], sA[1], sA[2], sA[3]};
  tree_fold_store<D, false>(P, it, wave, lane, s_ml, ow);
}

// fp32 queries and pools: the same walk on v_mfma_f32_32x32x2 (fp32 products
// and sums).  Step s of the score product multiplies channel s (lane half 0)
// and D/2 + s (half 1).  One LDS stage a wave: K of the next tile is asked for
// once this tile's scores are there, V once its product is.
template <int D>
__global__ void __launch_bounds__(256) tree_attn_f32_kernel(TreeParams P) {
  constexpr int DB = D / 32, RB = D * 4, SL = RB / 16;
  constexpr int TB = kTreeKT * RB;
  constexpr int RPI = 1024 / RB;
  constexpr int NI = TB / 1024;
  __shared__ __attribute__((aligned(16))) char sK[kTreeWaves][TB], sV[kTreeWaves][TB];
  __shared__ float2 s_ml[kTreeWaves][32];
  TreeItem it;
  if (!tree_find<kTreeKT, kTreeRows, true>(P, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int t_end = (int)((int64_t)it.tiles * (it.cut + 1) / it.cuts);
  const int t0 = (int)((int64_t)it.tiles * it.cut / it.cuts) + wave;
  const int nc = (it.ctx + kTreeKT - 1) / kTreeKT;

  const int r_eff = min(it.rb * kTreeRows + qc, it.n * P.rep - 1);
  const int node = r_eff / P.rep, head = it.h * P.rep + (r_eff - node * P.rep);
  float qf[D / 2];  // channels hh D/2 + s
  {
    const float4* qrow = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(P.q) +
                                                         (it.lo + node) * P.q_stride_n + head * P.q_stride_h +
                                                         hh * (D / 2));
#pragma unroll
    for (int s = 0; s < D / 8; ++s) {
      const float4 x = qrow[s];
      qf[4 * s] = x.x;
      qf[4 * s + 1] = x.y;
      qf[4 * s + 2] = x.z;
      qf[4 * s + 3] = x.w;
    }
  }
  const char* kh = P.k + (int64_t)it.h * P.sh * 16;
  const char* vh = P.v + (int64_t)it.h * P.sh * 16;
  // K pieces are swizzled (piece ^ row % 16), V rows are read whole
  auto issue = [&](const char* base, uint32_t place, char* st, bool is_v) {
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = j * RPI + lane / SL, slot = lane % SL;
      const uint32_t at = __shfl(place, row, 64);
      const int piece = is_v ? slot : slot ^ (row & 15);
      tree_dma(at == kNoRow ? reinterpret_cast<const char*>(tree_zeros) : base + (int64_t)at * 16 + (piece << 4),
               st + j * 1024);
    }
  };
  pf32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pf32x16{};
  float m_run = -INFINITY, l_run = 0.f;
  const int key = lane & 31;
  char* const stK = sK[wave];
  char* const stV = sV[wave];
  TreeRow<kTreeKT> row;
  row.load(P, it, t0, key);
  uint32_t place = row.place(P);
  if (t0 < t_end) {
    issue(kh, place, stK, false);
    issue(vh, place, stV, true);
  }
  for (int t = t0; t < t_end; t += kTreeWaves) {
    const uint32_t there = (uint32_t)__ballot(place != kNoRow);
    uint32_t bits = there;
    if (t >= nc) bits &= tree_bits(P, it, node, t - nc);
    row.load(P, it, t + kTreeWaves, key);
    __builtin_amdgcn_s_waitcnt(0);
    pf32x16 S = pf32x16{};
#pragma unroll
    for (int s = 0; s < D / 8; ++s) {
      const float4 x =
          *reinterpret_cast<const float4*>(stK + qc * RB + (((hh * (D / 8) + s) ^ (qc & 15)) << 4));
      S = __builtin_amdgcn_mfma_f32_32x32x2f32(x.x, qf[4 * s], S, 0, 0, 0);
      S = __builtin_amdgcn_mfma_f32_32x32x2f32(x.y, qf[4 * s + 1], S, 0, 0, 0);
      S = __builtin_amdgcn_mfma_f32_32x32x2f32(x.z, qf[4 * s + 2], S, 0, 0, 0);
      S = __builtin_amdgcn_mfma_f32_32x32x2f32(x.w, qf[4 * s + 3], S, 0, 0, 0);
    }
    place = row.place(P);
    const bool more = t + kTreeWaves < t_end;
    if (more) issue(kh, place, stK, false);
    const uint32_t mine = bits >> (4 * hh);
    if (__ballot(bits != 0xffffffffu)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) S[e] = (mine >> (8 * (e >> 2) + (e & 3))) & 1 ? S[e] : -INFINITY;
    }
    float bm = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) bm = fmaxf(bm, S[e]);
    bm = half_max(bm) * P.scale2;
    const float m_old = m_run;
    m_run = bm > m_old + kTreeLazyMax ? bm : m_old;
    const float ms = m_run == -INFINITY ? 0.f : m_run;
    if (__ballot(m_run != m_old)) {
      const float alpha = m_run != m_old ? __builtin_amdgcn_exp2f(m_old - m_run) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
    float p[16];
    float ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e], P.scale2, -ms));
      ps[e & 3] += p[e];
    }
    l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
    typedef __attribute__((ext_vector_type(DB))) float vrow;
    auto vread = [&](int e) {
      return *reinterpret_cast<const vrow*>(stV + (8 * (e >> 2) + 4 * hh + (e & 3)) * RB + qc * DB * 4);
    };
    // tree rows: values that are not finite reach the rows that see them only
    bool odd = false;
    if (t >= nc) {
      bool bad = false;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const vrow v = vread(e);
#pragma unroll
        for (int db = 0; db < DB; ++db) bad |= !(fabsf(v[db]) < INFINITY);
      }
      odd = __ballot(bad) != 0;
    }
    // a tile's products are summed by themselves and then added to O: its rounding error stays below one
    // accumulator's over all keys
    pf32x16 tile[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) tile[db] = pf32x16{};
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const vrow v = vread(e);
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        const float x = odd && !(fabsf(v[db]) < INFINITY) ? 0.f : v[db];
        tile[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[e], tile[db], 0, 0, 0);
      }
    }
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] += tile[db];
    if (odd) {
#pragma unroll
      for (int x = 0; x < 2 * DB; ++x) {
        const float inf = x & 1 ? -INFINITY : INFINITY;
        pf32x16 n = pf32x16{};
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const float v = vread(e)[x >> 1];
          const float sees = (mine >> (8 * (e >> 2) + (e & 3))) & 1 ? 1.f : 0.f;
          n = __builtin_amdgcn_mfma_f32_32x32x2f32(v == inf || v != v ? 1.f : 0.f, sees, n, 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) o[x >> 1][e] += n[e] > 0.f ? inf : 0.f;
      }
    }
    if (more) issue(vh, place, stV, true);
  }
  const float lt = half_sum(l_run);
  if (hh == 0) s_ml[wave][qc] = make_float2(m_run, lt);
  // piece i DB + g: rows m = 8 i + 4 hh + {0..3} are 4 DB channels in a row
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int g = 0; g < DB; ++g) {
      float x[4];
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const int c = 4 * g + y;
        x[y] = o[c % DB][4 * i + c / DB];
      }
      *reinterpret_cast<float4*>(stK + ((i * DB + g) * 64 + lane) * 16) = make_float4(x[0], x[1], x[2], x[3]);
    }
  __syncthreads();
  const char* ow[kTreeWaves] = {sK[0], sK[1], sK[2], sK[3]};
  tree_fold_store<D, true>(P, it, wave, lane, s_ml, ow);
}

// Merge of a unit's partials: with M the largest of a row's maxima, out = sum_c
// 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c.  One workgroup folds four pieces of
// a unit, its waves every fourth partial each; the order is fixed.
template <int D, bool F32>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeParams P) {
  constexpr int PIECES = D / 8, PPW = 4;
  __shared__ float4 s_o[kTreeWaves][PPW][64];
  __shared__ float2 s_ml[kTreeWaves][32];
  TreeItem it;
  if (!tree_find<kTreeKT, kTreeRows, false>(P, blockIdx.x, it) || it.cuts <= 1) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int x0 = blockIdx.y * PPW;
  const int r = it.rb * kTreeRows + qc;
  const bool live = r < it.n * P.rep;
  float m = -INFINITY, l = 0.f;
  float4 acc[PPW];
#pragma unroll
  for (int x = 0; x < PPW; ++x) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (live) {
#pragma unroll 4
    for (int c = wave; c < it.cuts; c += kTreeWaves) {
      const int64_t pu = it.part + c;
      const float2 ml = P.part_ml[pu * 32 + qc];
      float4 v[PPW];
#pragma unroll
      for (int x = 0; x < PPW; ++x) v[x] = P.part_o[pu * (PIECES * 64) + (x0 + x) * 64 + lane];
      const float mn = fmaxf(m, ml.x);
      const float wo = tree_weight(m, mn), wn = tree_weight(ml.x, mn);
      m = mn;
      l = l * wo + ml.y * wn;
#pragma unroll
      for (int x = 0; x < PPW; ++x) {
        acc[x].x = __builtin_fmaf(v[x].x, wn, acc[x].x * wo);
        acc[x].y = __builtin_fmaf(v[x].y, wn, acc[x].y * wo);
        acc[x].z = __builtin_fmaf(v[x].z, wn, acc[x].z * wo);
        acc[x].w = __builtin_fmaf(v[x].w, wn, acc[x].w * wo);
      }
    }
  }
#pragma unroll
  for (int x = 0; x < PPW; ++x) s_o[wave][x][lane] = acc[x];
  if (hh == 0) s_ml[wave][qc] = make_float2(m, l);
  __syncthreads();
  if (!live) return;
  float M = -INFINITY;
#pragma unroll
  for (int w = 0; w < kTreeWaves; ++w) M = fmaxf(M, s_ml[w][qc].x);
  float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kTreeWaves; ++w) {
    const float wt = tree_weight(s_ml[w][qc].x, M);
    const float4 y = s_o[w][wave][lane];
    l += s_ml[w][qc].y * wt;
    a.x += y.x * wt;
    a.y += y.y * wt;
    a.z += y.z * wt;
    a.w += y.w * wt;
  }
  const float inv = tree_inv(l);
  const float v4[4] = {a.x * inv, a.y * inv, a.z * inv, a.w * inv};
  const int node = r / P.rep, head = it.h * P.rep + (r - node * P.rep);
  const int64_t row = it.lo + node;
  tree_store4(P, row * P.o_stride_n + head * P.o_stride_h + tree_channel<D, F32>(x0 + wave, hh), v4);
  if (P.lse != nullptr && blockIdx.y == 0 && wave == 0 && hh == 0) P.lse[row * P.H + head] = tree_lse(M, l);
}

}  // namespace halo

using namespace halo;

namespace {

// How a call is cut: units at most, workgroups that the GPU holds, launch size, partials at most.
struct TreeShape {
  int64_t units, grid, partials;
  int slots, min_tiles;
  bool merge;
};
TreeShape tree_shape(int dtype, int B, int H, int H_kv, int D, int64_t max_rows, int max_nodes) {
  TreeShape s;
  const int64_t rows = (int64_t)max_nodes * (H / H_kv);
  s.units = (int64_t)B * H_kv * ((rows + kTreeRows - 1) / kTreeRows);
  // LDS of a workgroup: 128 KiB at D = 128, 64 KiB at D = 64, fp32 the same with half the stages
  s.slots = 256 * (D == 64 ? 2 : 1);
  s.min_tiles = 2 * kTreeWaves;
  const int64_t longest = (max_rows + kTreeKT - 1) / kTreeKT + (max_nodes + kTreeKT - 1) / kTreeKT;
  s.merge = longest > s.min_tiles;
  // tree_find: at most `room` items besides one a unit
  s.grid = s.merge ? (s.slots / 2 + s.units > s.slots ? s.slots / 2 + s.units : s.slots) : s.units;
  s.partials = s.merge ? s.slots : 0;
  return s;
}

int64_t tree_part_bytes(int D) { return (int64_t)kTreeRows * D * 4 + kTreeRows * 8; }

bool tree_sizes_ok(int B, int H, int H_kv, int D, int64_t max_rows, int max_nodes) {
  return B > 0 && H > 0 && H_kv > 0 && H % H_kv == 0 && (D == 64 || D == 128) && max_rows > 0 &&
         max_rows < (1ll << 31) - 1024 && max_nodes > 0 && max_nodes <= 512 && (int64_t)max_nodes * (H / H_kv) < (1 << 24) &&
         (int64_t)B * H_kv * ((int64_t)max_nodes * (H / H_kv) / kTreeRows + 1) < (1ll << 30);
}

}  // namespace

extern "C" size_t halo_tree_workspace_size(int dtype, int B, int H, int H_kv, int D, int64_t max_rows, int max_nodes) {
  if (!tree_sizes_ok(B, H, H_kv, D, max_rows, max_nodes)) return 0;
  return (size_t)tree_shape(dtype, B, H, H_kv, D, max_rows, max_nodes).partials * (size_t)tree_part_bytes(D);
}

extern "C" int halo_tree_attn(const halo_block_pool* pool, const void* q, int64_t q_stride_n, int64_t q_stride_h,
                              int N, int H, const int32_t* table, int64_t table_stride, int B, int W,
                              const int32_t* lengths, const int32_t* cu_nodes, int max_nodes, const int64_t* mask,
                              int64_t mask_stride, float scale, void* out, int64_t out_stride_n, int64_t out_stride_h,
                              int out_dtype, float* lse, void* workspace, size_t workspace_bytes, void* stream) {
  HALO_CHECK_ARG(pool && pool->k && pool->v && table && lengths && cu_nodes, "null pointer argument");
  const int dtype = pool->dtype, D = pool->D, H_kv = pool->H_kv;
  HALO_CHECK_ARG(dtype == HALO_BF16 || dtype == HALO_F16 || dtype == HALO_F32, "dtype must be bf16, f16 or f32");
  HALO_CHECK_ARG(out_dtype == HALO_F32 || out_dtype == HALO_BF16 || out_dtype == HALO_F16, "bad out_dtype");
  HALO_CHECK_ARG(pool->layers == 1 && pool->blocks > 0 && pool->block_size > 0 && W > 0, "need a pool of one layer");
  HALO_CHECK_ARG(D == 64 || D == 128, "head_dim must be 64 or 128");
  HALO_CHECK_ARG(N >= 0, "bad number of nodes");
  if (N == 0) return HALO_OK;
  HALO_CHECK_ARG(q && out, "null pointer argument");
  HALO_CHECK_ARG(tree_sizes_ok(B, H, H_kv, D, (int64_t)W * pool->block_size, max_nodes),
                 "need H % H_kv == 0, 1 <= max_nodes <= 512 and positive sizes in 31 bits");
  HALO_CHECK_ARG(table_stride >= W, "rows of the block table overlap");
  HALO_CHECK_ARG(mask == nullptr || mask_stride >= (max_nodes + 63) / 64, "mask rows are shorter than max_nodes bits");
  const int64_t es = elem_size(dtype);
  const int64_t lanes = 16 / es;  // elements of a 16-byte piece
  HALO_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | (uintptr_t)(q_stride_n * es) | (uintptr_t)(q_stride_h * es)) % 16 == 0,
                 "q rows must be 16-byte aligned");
  HALO_CHECK_ARG((reinterpret_cast<uintptr_t>(pool->k) | reinterpret_cast<uintptr_t>(pool->v)) % 16 == 0 &&
                     pool->stride_b % lanes == 0 && pool->stride_h % lanes == 0 && pool->stride_r % lanes == 0,
                 "pool rows must be 16-byte aligned");
  HALO_CHECK_ARG(pool->stride_b >= 0 && pool->stride_h >= 0 && pool->stride_r >= 0, "negative pool strides");
  // places are 32-bit counts of 16-byte pieces, one value of them means "no row"
  const int64_t last = ((int64_t)(pool->blocks - 1) * pool->stride_b + (pool->block_size - 1) * pool->stride_r) / lanes;
  HALO_CHECK_ARG(last < 0xffffffffll && pool->stride_h / lanes * (H_kv - 1) < 0xffffffffll, "pool larger than 64 GiB");
  HALO_CHECK_ARG(scale > 0.f && std::isfinite(scale), "scale must be positive and finite");
  const TreeShape s = tree_shape(dtype, B, H, H_kv, D, (int64_t)W * pool->block_size, max_nodes);
  const size_t need = (size_t)s.partials * (size_t)tree_part_bytes(D);
  HALO_CHECK_ARG(need == 0 || (workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0),
                 "workspace missing or not 16-byte aligned");
  if (workspace_bytes < need) {
    set_error("workspace too small");
    return HALO_E_WORKSPACE;
  }
  TreeParams p;
  p.q = q;
  p.q_stride_n = q_stride_n;
  p.q_stride_h = q_stride_h;
  p.k = static_cast<const char*>(pool->k);
  p.v = static_cast<const char*>(pool->v);
  p.sb = (uint32_t)(pool->stride_b / lanes);
  p.sh = (uint32_t)(pool->stride_h / lanes);
  p.sr = (uint32_t)(pool->stride_r / lanes);
  p.blocks = pool->blocks;
  p.bs = make_div(pool->block_size);
  p.table = table;
  p.table_stride = table_stride;
  p.W = W;
  p.lengths = lengths;
  p.cu = cu_nodes;
  p.mask = reinterpret_cast<const uint32_t*>(mask);
  p.mask_stride = 2 * mask_stride;
  p.B = B;
  p.H = H;
  p.H_kv = H_kv;
  p.rep = H / H_kv;
  p.N = N;
  p.max_nodes = max_nodes;
  p.slots = s.slots;
  p.min_tiles = s.min_tiles;
  p.scale2 = (float)((double)scale * 1.4426950408889634);
  HALO_CHECK_ARG(p.scale2 >= 0x1p-126f && std::isfinite(p.scale2), "scale out of range");
  p.out = out;
  p.o_stride_n = out_stride_n;
  p.o_stride_h = out_stride_h;
  p.out_dtype = out_dtype;
  const int64_t ea = out_dtype == HALO_F32 ? 16 : 8, eo = elem_size(out_dtype);
  p.out_vec4 = reinterpret_cast<uintptr_t>(out) % ea == 0 && (out_stride_n * eo) % ea == 0 && (out_stride_h * eo) % ea == 0;
  p.lse = lse;
  p.part_o = reinterpret_cast<float4*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + s.partials * kTreeRows * (D / 4));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)s.grid), block(64 * kTreeWaves), mgrid((unsigned)s.units, D / 32);
#define HALO_TREE(KERNEL, DV, F32V)                                                                       \
  do {                                                                                                    \
    hipLaunchKernelGGL((KERNEL), grid, block, 0, st, p);                                                  \
    if (s.merge) hipLaunchKernelGGL((tree_merge_kernel<DV, F32V>), mgrid, dim3(256), 0, st, p);           \
  } while (0)
#define HALO_TREE16(DTV)                                                  \
  do {                                                                    \
    if (D == 128) HALO_TREE((tree_attn_kernel<DTV, 128>), 128, false);    \
    else HALO_TREE((tree_attn_kernel<DTV, 64>), 64, false);               \
  } while (0)
  if (dtype == HALO_F32) {
    if (D == 128) HALO_TREE((tree_attn_f32_kernel<128>), 128, true);
    else HALO_TREE((tree_attn_f32_kernel<64>), 64, true);
  } else if (dtype == HALO_BF16) {
    HALO_TREE16(HALO_BF16);
  } else {
    HALO_TREE16(HALO_F16);
  }
#undef HALO_TREE16
#undef HALO_TREE
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
