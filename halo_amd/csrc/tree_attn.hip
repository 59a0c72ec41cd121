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
// A request's key tiles are its rows, committed ones and then the tree's, in
// steps of KT from row 0.  The lengths are on the device only: every workgroup
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
  int slots, min_tiles;  // workgroups aimed at; the least that an item's largest number of tiles may be
  float scale2;
  void* out;
  int64_t o_stride_n, o_stride_h;
  int out_f32;
  float* lse;
  float4* part_o;
  float2* part_ml;
};

// Narrow kernels (up to 32 rows a unit): the columns of one 32x32 product, key
// tiles of 32, four waves with tiles of their own.  Wide: key tiles of 64.
constexpr int kTreeRows = 32, kTreeKT = 32, kTreeWaves = 4;
constexpr int kTreeWideKT = 64;
// Slack (log2 units) by which a tile's max may exceed the running max before
// the running max moves (probabilities stay below 2^8).
constexpr float kTreeLazyMax = 8.0f;
// The running max of the 16-bit kernels is held kTreeLift (log2 units) below the
// one found, which lifts all weights and sums alike and leaves their quotients.
// fp16 has no exponents below 2^-14: as they are, weights of 2^-25 of the
// largest and less would vanish from the products while l still counts them (a
// first row of large score and 9000 rows of 2^-25.6 behind it gave 0 for
// 1.8e-4).  Lifted by 2^7 they are off by 2^-32 of the largest at most, and stay
// below 2^15 for exponents up to 2^30: the tile's max is taken a step up there,
// since an exponent's exact product may lie half a step above its rounded one,
// and the step is 32 at 2^28.  bf16 has fp32's exponents.
template <int DT>
__device__ __forceinline__ float tree_new_max(float m_old, float bm) {
  constexpr float kLift = DT == HALO_F16 ? 7.0f : 0.0f;
  if constexpr (DT == HALO_F16) bm = __builtin_fmaf(fabsf(bm), 0x1.01p-24f, bm);  // of -inf NaN, which is not above
  return bm - m_old > kTreeLazyMax + kLift ? bm - kLift : m_old;
}

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
    if (r.n > 0) r.tiles = (r.ctx + r.n + KT - 1) / KT;
  }
  return r;
}

// One item (or, for the merge, one unit) of the launch.
struct TreeItem {
  int b, lo, ctx, n, rbs, tiles;
  int h, rb, cut, cuts;  // the cut-th of `cuts` cuts of the unit (h, rb)
  int part;              // partial of the unit's first cut
};

// Finds item x, EACH requests a lane at once (one round trip to memory up to 64
// EACH requests).
template <int KT, int R, bool ITEMS, int EACH>
__device__ __forceinline__ bool tree_find_of(const TreeParams& P, int x, TreeItem& it) {
  const int lane = threadIdx.x & 63;
  TreeReq r[EACH];
  auto look = [&](int b0) {
#pragma unroll
    for (int k = 0; k < EACH; ++k) r[k] = tree_req<KT, R>(P, b0 + lane * EACH + k);
  };
  look(0);
  float total = 0.f;
  int units = 0;
  for (int b0 = 0;;) {
    int u = 0;
    float t = 0.f;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      u += P.H_kv * r[k].rbs;
      t += (float)(P.H_kv * r[k].rbs) * (float)r[k].tiles;
    }
    units += lane_of(wave_prefix(u), 63);
    total += lane_of(wave_prefix(t), 63);
    b0 += 64 * EACH;
    if (b0 >= P.B) break;
    look(b0);
  }
  // sum of ceil(tiles / L) <= total / L + units: a share that fills the GPU
  // once if the units leave room.  Items, cut units and partials stay within
  // the launch and the workspace whatever the batch: a rounded sum of terms
  // that are not negative is never below the rounded sum of some of them alone,
  // and of the (at most 2 P.slots, were there more) cut units each goes through
  // 16 roundings in its wave and one for each wave with another of them, so
  // total >= (the cut units' tiles) (1 - 1040 2^-24), which the factor covers.
  const int room = P.slots > 2 * units ? P.slots - units : P.slots / 2;
  const int share = (int)fminf(ceilf(total * (1.f + 0x1p-14f) / (float)room), 1e9f);
  constexpr int EVEN = KT == kTreeKT ? kTreeWaves : 1;  // waves that share an item's tiles: none gets one more
  const int L = max((share + EVEN - 1) / EVEN * EVEN, P.min_tiles);
  int base = 0, part = 0;
  if (P.B > 64 * EACH) look(0);
  for (int b0 = 0;;) {
    int cuts[EACH], mine[EACH], parts[EACH], sum = 0, psum = 0;
#pragma unroll
    for (int k = 0; k < EACH; ++k) {
      cuts[k] = (int)(((uint32_t)r[k].tiles + (uint32_t)L - 1) / (uint32_t)L);
      const int u = P.H_kv * r[k].rbs;
      parts[k] = cuts[k] > 1 ? u * cuts[k] : 0;
      mine[k] = ITEMS ? u * cuts[k] : cuts[k] > 1 ? u : 0;
      sum += mine[k];
      psum += parts[k];
    }
    const int at = wave_prefix(sum), parts_at = wave_prefix(psum);
    const uint64_t past = __ballot(base + at > x);
    if (past != 0) {
      const int w = __builtin_ctzll(past);
      int y = x - (base + lane_of(at, w) - lane_of(sum, w));  // among lane w's requests
      part += lane_of(parts_at, w) - lane_of(psum, w);
      bool found = false;
#pragma unroll
      for (int k = 0; k < EACH; ++k) {
        const int m = lane_of(mine[k], w);
        if (!found && y < m) {
          found = true;
          it.b = b0 + w * EACH + k;
          it.lo = lane_of(r[k].lo, w);
          it.ctx = lane_of(r[k].ctx, w);
          it.n = lane_of(r[k].n, w);
          it.rbs = lane_of(r[k].rbs, w);
          it.tiles = lane_of(r[k].tiles, w);
          it.cuts = lane_of(cuts[k], w);
        }
        if (!found) {
          y -= m;
          part += lane_of(parts[k], w);
        }
      }
      it.cut = 0;
      it.rb = 0;
      uint32_t z = (uint32_t)y;
      if (it.rbs > 1) {
        it.rb = z % (uint32_t)it.rbs;
        z /= (uint32_t)it.rbs;
      }
      if (ITEMS && it.cuts > 1) {
        it.cut = z % (uint32_t)it.cuts;
        z /= (uint32_t)it.cuts;
      }
      it.h = z;
      it.part = part + (it.rb * P.H_kv + it.h) * it.cuts;
      return true;
    }
    base += lane_of(at, 63);
    part += lane_of(parts_at, 63);
    b0 += 64 * EACH;
    if (b0 >= P.B) return false;
    look(b0);
  }
}

// Every lane returns the same; false past the last one.  ITEMS: x counts items
// (head, cut, row block; the row blocks that read the same rows side by side),
// else the units that were cut (head, row block).
template <int KT, int R, bool ITEMS>
__device__ __forceinline__ bool tree_find(const TreeParams& P, int x, TreeItem& it) {
  return P.B <= 64 ? tree_find_of<KT, R, ITEMS, 1>(P, x, it) : tree_find_of<KT, R, ITEMS, 4>(P, x, it);
}

// Staging.  An LDS-DMA instruction fills 1 KiB, lane l its piece l, so RPI rows
// of RB bytes; NJ instructions of a wave fill KEYS rows.  Row key(lane, j) is
// the one that lane reads for instruction j: a lane's rows lie side by side (or
// every other one), so where a block holds them all, one look at the block
// table is enough.  At RB = 128 two rows share the 64 banks; there the parity
// of the LDS row is kept that of the key.  Both swizzles (which 16-byte piece
// of a row lies where) go by the key and put every read pass on distinct banks.
constexpr uint32_t kNoRow = 0xffffffffu;
template <int RB, int NJ>
struct TreeLanes {
  static constexpr int SL = RB / 16, RPI = 64 / SL, KEYS = NJ * RPI;
  static constexpr int STEP = RB == 128 ? 2 : 1;  // keys from one instruction to the next
  static constexpr int SPAN = NJ * STEP;          // keys, aligned to their number, that a lane's rows lie in
  __device__ static __forceinline__ int first(int lane) {
    const int g = lane / SL;
    return RB == 128 ? SPAN * (g >> 1) + (g & 1) : SPAN * g;
  }
  __host__ __device__ static constexpr int lds_row(int key) {  // key < KEYS
    return RB == 128 ? ((key >> 1) % NJ) * RPI + 2 * (key / SPAN) + (key & 1) : (key % NJ) * RPI + key / NJ;
  }
};
template <int RB>
__device__ __forceinline__ int tree_kswz(int key) {
  return RB == 128 ? (key >> 1) & 7 : key & 15;
}
template <int RB>
__device__ __forceinline__ int tree_vswz(int key) {
  return RB == 128 ? 2 * ((key >> 1) & 1) : 2 * (key & 3);
}

// The table entry of position `pos` (-1 past the request's rows or the table), and its row in the block.
struct TreeRow {
  int blk, in_blk;
  __device__ __forceinline__ void load(const TreeParams& P, const TreeItem& it, int pos) {
    const int c = div_by(pos, P.bs);
    // read in any case, from the last column at most: a load behind a branch would be waited for with all others
    blk = P.table[it.b * P.table_stride + min(c, P.W - 1)];
    in_blk = pos < it.ctx + it.n && c < P.W ? pos - c * P.bs.d : -1;
  }
  __device__ __forceinline__ bool there(const TreeParams& P) const {
    return in_blk >= 0 && (uint32_t)blk < (uint32_t)P.blocks;
  }
  // in 16-byte pieces from the pool's first row, which stands in for rows that are not there
  __device__ __forceinline__ uint32_t place(const TreeParams& P) const {
    const uint32_t at = (uint32_t)blk * P.sb + (uint32_t)in_blk * P.sr;
    return there(P) ? at : 0;
  }
};

// What rows that are not there read as, where they are not zeroed in LDS.
__device__ uint4 tree_zeros[1];

// 16 bytes a lane from memory into the 1 KiB of LDS at `st` (lane l's piece at 16 l).
__device__ __forceinline__ void tree_dma(const char* from, char* st) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from),
                                   (__attribute__((address_space(3))) void*)(st), 16, 0, 0);
}

// Bits of the 32 positions from `pos` on that node i of the item's tree sees:
// committed rows all, tree rows by the node's mask.  In two steps, so that the
// mask's words can be on their way during other work.
struct TreeBits {
  uint32_t lo, hi;
  __device__ __forceinline__ void load(const TreeParams& P, const TreeItem& it, int i, int pos) {
    lo = hi = 0xffffffffu;
    if (P.mask == nullptr) return;
    const int w = (pos - it.ctx) >> 5, words = (it.n + 31) >> 5;
    const uint32_t* row = P.mask + (int64_t)(it.lo + i) * P.mask_stride;
    if (w >= 0) lo = w < words ? row[w] : 0u;
    if (w >= -1) hi = w + 1 < words ? row[w + 1] : 0u;
  }
  __device__ __forceinline__ uint32_t at(const TreeParams& P, const TreeItem& it, int i, int pos) const {
    if (P.mask == nullptr) {
      const int d = it.ctx + i - pos;
      return d < 0 ? 0u : d >= 31 ? 0xffffffffu : (2u << d) - 1;
    }
    return (uint32_t)((((uint64_t)hi << 32) | lo) >> ((pos - it.ctx) & 31));
  }
};
__device__ __forceinline__ uint32_t tree_bits(const TreeParams& P, const TreeItem& it, int i, int pos) {
  TreeBits b;
  b.load(P, it, i, pos);
  return b.at(P, it, i, pos);
}

// Bit k set: position pos + k is one of the request's rows (k < 32).
__device__ __forceinline__ uint32_t tree_rows(const TreeItem& it, int pos) {
  const int n = it.ctx + it.n - pos;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
}

// Which halves of a word hold 16-bit values that are not finite, as 0xffff.
template <int DT>
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
  constexpr uint32_t E = DT == HALO_BF16 ? 0x7f80u : 0x7c00u;
  return ((w & E) == E ? 0xffffu : 0u) | ((w & (E << 16)) == (E << 16) ? 0xffff0000u : 0u);
}
template <int DT>
__device__ __forceinline__ uint4 odd_halves(const uint4& v) {
  return make_uint4(odd_halves<DT>(v.x), odd_halves<DT>(v.y), odd_halves<DT>(v.z), odd_halves<DT>(v.w));
}

// Tree rows that some nodes see and others do not: 0 x inf is not 0, so values
// of V that are not finite must not meet the products.  Whether the staged V
// tile (`bytes` of 16-bit values) holds any; all lanes take part.
template <int DT>
__device__ __forceinline__ bool tree_v_odd(const char* sv, int bytes, int lane) {
  bool any = false;
#pragma unroll 1
  for (int x = lane * 16; x < bytes; x += 1024) {
    const uint4 o = odd_halves<DT>(*reinterpret_cast<const uint4*>(sv + x));
    any |= (o.x | o.y | o.z | o.w) != 0;
  }
  return __ballot(any) != 0;
}
// Zeroes them in LDS, from byte `from` in steps of `step`.
template <int DT>
__device__ __forceinline__ void tree_v_clean(char* sv, int bytes, int from, int step) {
#pragma unroll 1
  for (int x = from; x < bytes; x += step) {
    uint4* at = reinterpret_cast<uint4*>(sv + x);
    const uint4 v = *at, o = odd_halves<DT>(v);
    *at = make_uint4(v.x & ~o.x, v.y & ~o.y, v.z & ~o.z, v.w & ~o.w);
  }
}
// Adds them to the rows that see them: bit k of `bits` is this lane's row and
// the tile's key k, whose staged row is at sv + at(k).
template <int DT, int D, typename AT>
__device__ __forceinline__ void tree_v_add_odd(pf32x16* o, const char* sv, uint64_t bits, int keys, int hh, AT at) {
  constexpr int RB = D * 2;
#pragma unroll 1
  for (int k = 0; k < keys; ++k) {
    const bool sees = (bits >> k) & 1;
    const char* row = sv + at(k);
#pragma unroll
    for (int x = 0; x < D / 8; ++x) {
      const int m = 8 * (x & 3) + 4 * hh;
      const int byte = ((m >> 4) * (D / 2) + 16 * (x >> 2) + (m & 15)) * 2;  // see tree_channel
      const uint2 w = *reinterpret_cast<const uint2*>(row + (((byte >> 4) ^ tree_vswz<RB>(k)) << 4) + (byte & 15));
#pragma unroll
      for (int y = 0; y < 4; ++y) {
        const uint32_t half = ((y & 2 ? w.y : w.x) >> (16 * (y & 1))) & 0xffffu;
        const float f = DT == HALO_BF16 ? __uint_as_float(half << 16) : f16_bits_to_f32((uint16_t)half);
        o[x >> 2][4 * (x & 3) + y] += sees && !(fabsf(f) < INFINITY) ? f : 0.f;
      }
    }
  }
}

// Four channels of a row of out, which is of the queries' type or fp32.
template <int DT>
__device__ __forceinline__ void tree_store4(const TreeParams& P, int64_t at, const float* v4) {
  if (DT == HALO_F32 || P.out_f32) store_elem4(P.out, at, HALO_F32, v4);
  else store_elem4(P.out, at, DT, v4);
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


// Waits until at most N of the wave's vector memory instructions are in flight
// (they end in order).
template <int N>
__device__ __forceinline__ void tree_wait() {
  static_assert(N < 64, "6 bits");
  // the builtin, not asm: the compiler then knows what has landed and adds no waits of its own
  __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}

// LDS reads of a tile in one block with their wait.  The compiler orders an
// ordinary LDS read behind every LDS-DMA in flight, since it cannot tell the
// next K tile from this V tile; these are ordered by tree_wait alone.
__device__ __forceinline__ uint32_t lds_addr(const char* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)(p);
}
typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;
typedef __attribute__((ext_vector_type(2))) uint32_t u32x2;
// b128 at a[0 .. N)
__device__ __forceinline__ void lds_read8(u32x4* v, const uint32_t* a) {
  asm volatile(
      "ds_read_b128 %0, %8\n\tds_read_b128 %1, %9\n\tds_read_b128 %2, %10\n\tds_read_b128 %3, %11\n\t"
      "ds_read_b128 %4, %12\n\tds_read_b128 %5, %13\n\tds_read_b128 %6, %14\n\tds_read_b128 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
      : "memory");
}
__device__ __forceinline__ void lds_read4(u32x4* v, const uint32_t* a) {
  asm volatile(
      "ds_read_b128 %0, %4\n\tds_read_b128 %1, %5\n\tds_read_b128 %2, %6\n\tds_read_b128 %3, %7\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
      : "memory");
}
__device__ __forceinline__ void lds_read8_b64(u32x2* v, const uint32_t* a) {
  asm volatile(
      "ds_read_b64 %0, %8\n\tds_read_b64 %1, %9\n\tds_read_b64 %2, %10\n\tds_read_b64 %3, %11\n\t"
      "ds_read_b64 %4, %12\n\tds_read_b64 %5, %13\n\tds_read_b64 %6, %14\n\tds_read_b64 %7, %15\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7])
      : "memory");
}
// V^T operands of N d-blocks: for each, transposed reads at a, a + 256, a + 512 and a + 768.
__device__ __forceinline__ void lds_read_tr2(u32x2* v, const uint32_t* a) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %8\n\tds_read_b64_tr_b16 %1, %8 offset:256\n\t"
      "ds_read_b64_tr_b16 %2, %8 offset:512\n\tds_read_b64_tr_b16 %3, %8 offset:768\n\t"
      "ds_read_b64_tr_b16 %4, %9\n\tds_read_b64_tr_b16 %5, %9 offset:256\n\t"
      "ds_read_b64_tr_b16 %6, %9 offset:512\n\tds_read_b64_tr_b16 %7, %9 offset:768\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
      : "v"(a[0]), "v"(a[1])
      : "memory");
}
__device__ __forceinline__ void lds_read_tr4(u32x2* v, const uint32_t* a) {
  asm volatile(
      "ds_read_b64_tr_b16 %0, %16\n\tds_read_b64_tr_b16 %1, %16 offset:256\n\t"
      "ds_read_b64_tr_b16 %2, %16 offset:512\n\tds_read_b64_tr_b16 %3, %16 offset:768\n\t"
      "ds_read_b64_tr_b16 %4, %17\n\tds_read_b64_tr_b16 %5, %17 offset:256\n\t"
      "ds_read_b64_tr_b16 %6, %17 offset:512\n\tds_read_b64_tr_b16 %7, %17 offset:768\n\t"
      "ds_read_b64_tr_b16 %8, %18\n\tds_read_b64_tr_b16 %9, %18 offset:256\n\t"
      "ds_read_b64_tr_b16 %10, %18 offset:512\n\tds_read_b64_tr_b16 %11, %18 offset:768\n\t"
      "ds_read_b64_tr_b16 %12, %19\n\tds_read_b64_tr_b16 %13, %19 offset:256\n\t"
      "ds_read_b64_tr_b16 %14, %19 offset:512\n\tds_read_b64_tr_b16 %15, %19 offset:768\n\t"
      "s_waitcnt lgkmcnt(0)"
      : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7]),
        "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]), "=&v"(v[14]), "=&v"(v[15])
      : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3])
      : "memory");
}

// Where a wave leaves piece x of its o (1 KiB, in register order): half of them over its K stage, half over its V stage.
template <int D>
__device__ __forceinline__ char* tree_piece(char* k, char* v, int x) {
  return x < D / 16 ? k + x * 1024 : v + (x - D / 16) * 1024;
}

// The four waves of a workgroup hold (m, l, o) of the same 32 rows over
// different tiles; each folds a quarter of the pieces.
template <int D, int DT, int TB>
__device__ __forceinline__ void tree_fold_store(const TreeParams& P, const TreeItem& it, int wave, int lane,
                                                float2 (*s_ml)[32], char (*sK)[TB], char (*sV)[TB]) {
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
      const float4 a = *reinterpret_cast<const float4*>(tree_piece<D>(sK[w], sV[w], x) + lane * 16);
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
      tree_store4<DT>(P, row * P.o_stride_n + head * P.o_stride_h + tree_channel<D, DT == HALO_F32>(x, hh), v);
    }
  }
  if (wave == 0 && hh == 0) {
    if (it.cuts > 1) P.part_ml[pu * 32 + qc] = make_float2(M, l);
    else if (P.lse != nullptr) P.lse[row * P.H + head] = tree_lse(M, l);
  }
}

// A wave's tile in the narrow kernels: where its rows lie and which are there.
template <int RB>
struct TreeTile {
  static constexpr int NJ = kTreeKT * RB / 1024;
  typedef TreeLanes<RB, NJ> L;
  TreeRow row;       // of the lane's first key, where one block holds the lane's rows
  uint32_t pl[NJ];
  uint32_t there;    // bit k: key k of the tile
  __device__ __forceinline__ void look(const TreeParams& P, const TreeItem& it, int t, int lane) {
    row.load(P, it, t * kTreeKT + L::first(lane));
  }
  __device__ __forceinline__ void locate(const TreeParams& P, const TreeItem& it, int t, int lane) {
    constexpr int GROUPS = kTreeKT / L::SPAN;  // lanes whose rows share a block, 64 / GROUPS of them
    if (P.bs.d % L::SPAN == 0) {
      const bool ok = row.there(P);
      const uint32_t p0 = row.place(P), step = ok ? L::STEP * P.sr : 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j) pl[j] = p0 + j * step;
      const uint64_t all = __ballot(ok);
      there = 0xffffffffu;
      if (all != ~0ull) {
        there = 0;
        constexpr uint32_t part = L::SPAN == 32 ? 0xffffffffu : (1u << L::SPAN) - 1;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) there |= (all >> (g * (64 / GROUPS))) & 1 ? part << (g * L::SPAN) : 0u;
      }
    } else {
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int k = L::first(lane) + j * L::STEP;
        TreeRow r;
        r.load(P, it, t * kTreeKT + k);
        pl[j] = r.place(P);
        mine |= r.there(P) ? 1u << k : 0u;
      }
      there = 0;
#pragma unroll
      for (int g = 0; g < L::RPI; ++g) there |= (uint32_t)__builtin_amdgcn_readlane(mine, g * L::SL);
    }
    there &= tree_rows(it, t * kTreeKT);
  }
  // K (swizzled for b128 reads of a row a lane) or V (for transposed reads; fp32 V plain)
  template <bool V, bool F32>
  __device__ __forceinline__ void issue(const char* base, char* st, int lane) const {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int k = L::first(lane) + j * L::STEP;
      const int slot = lane % L::SL;
      const int piece = !V ? slot ^ tree_kswz<RB>(k) : F32 ? slot : slot ^ tree_vswz<RB>(k);
      tree_dma(base + (int64_t)pl[j] * 16 + (piece << 4), st + j * 1024);
    }
  }
};

// Zeroes the rows of a wave's staged V tile that are not there: their weights
// are 0, but what the stand-in row holds need not be finite.
template <int RB>
__device__ __forceinline__ void tree_zero_rows(char* sv, uint32_t there, int lane) {
  typedef typename TreeTile<RB>::L L;
#pragma unroll 1
  for (int j = 0; j < TreeTile<RB>::NJ; ++j) {
    const int k = L::first(lane) + j * L::STEP;
    if (!((there >> k) & 1)) *reinterpret_cast<uint4*>(sv + j * 1024 + lane * 16) = make_uint4(0, 0, 0, 0);
  }
}

// 16-bit queries and pools, products on v_mfma_f32_32x32x16:
//   scores  S^T[key][row] = sum_d K[key][d] Q[row][d]          (A = K tile, B = Q^T)
//   output  O^T[d][row]  += sum_key V^T[d][key] P^T[key][row]  (A = V^T, B = P^T)
// S^T's accumulator gives lane (row, half h) the keys 8i + 4h + j, which are the
// keys of its P^T operands, so p goes to the second product (rounded to the
// pool's type: half a step of it at most, fp16's below 2^-21 of the largest
// off by 2^-32 of that) without a cross-lane move.  Each wave
// streams tiles of its own, every fourth of the item's, through one LDS stage
// of its own: the next K tile is asked for once the scores are there, the next
// V tile once the product is; no barrier in the loop.  One stage leaves room for
// two workgroups a CU, whose loads overlap each other's products.  Long
// requests run at the memory's rate (16 of 8192 rows, 8 KV heads: 106 us,
// 5.0 TB/s; one of 131072: 101); 8 nodes over 4096 rows take 11 us where their
// bytes need 3.3: one chain of launch, item search, table look, K, V, the second
// tile's K and V behind the first's products, and the fold of the four waves.
template <int DT, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) tree_attn_kernel(TreeParams P) {
  constexpr int KS = D / 16, DB = D / 32, RB = D * 2;
  constexpr int TB = kTreeKT * RB;  // bytes of a K or V tile
  typedef TreeTile<RB> Tile;
  typedef typename Tile::L L;
  constexpr int NJ = Tile::NJ;
  __shared__ __attribute__((aligned(16))) char sK[kTreeWaves][TB], sV[kTreeWaves][TB];
  __shared__ float2 s_ml[kTreeWaves][32];
  TreeItem it;
  if (!tree_find<kTreeKT, kTreeRows, true>(P, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int t_end = (int)((int64_t)it.tiles * (it.cut + 1) / it.cuts);
  int t = (int)((int64_t)it.tiles * it.cut / it.cuts) + wave;
  const int tree0 = it.ctx / kTreeKT;  // first tile with tree rows
  char* const stK = sK[wave];
  char* const stV = sV[wave];
  const char* kh = P.k + (int64_t)it.h * P.sh * 16;
  const char* vh = P.v + (int64_t)it.h * P.sh * 16;
  Tile tile;
  tile.look(P, it, t, lane);

  const int r_eff = min(it.rb * kTreeRows + qc, it.n * P.rep - 1);
  const int node = r_eff / P.rep, head = it.h * P.rep + (r_eff - node * P.rep);
  uint4 qb[KS];  // lane (row, half): channels 16 s + 8 half .. + 8
  {
    const char* qrow =
        reinterpret_cast<const char*>(P.q) + ((it.lo + node) * P.q_stride_n + head * P.q_stride_h) * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const uint4*>(qrow + (s * 16 + hh * 8) * 2);
  }
  // the mask bits of the wave's first tile with tree rows
  const int tm = t < tree0 ? t + (tree0 - t + kTreeWaves - 1) / kTreeWaves * kTreeWaves : t;
  TreeBits first_bits = {0, 0};
  if (tm < t_end) first_bits.load(P, it, node, tm * kTreeKT);

  uint32_t ka[KS];  // K operands: key qc, channels 16 s + 8 half
#pragma unroll
  for (int s = 0; s < KS; ++s)
    ka[s] = lds_addr(stK) + L::lds_row(qc) * RB + (((2 * s + hh) ^ tree_kswz<RB>(qc)) << 4);
  // V^T operands of step u, d-block db: keys 16 u + 4 (lane / 32) + (lane % 16) / 4 and 8 more, 512 bytes a step, 256 to the upper keys
  static_assert((L::lds_row(8) - L::lds_row(0)) * RB == 256 && (L::lds_row(16) - L::lds_row(0)) * RB == 512, "offsets of the V reads");
  uint32_t va[DB];
  {
    const int vG = lane >> 4, vei = (lane & 15) >> 2, vai = lane & 3;
    const int k = 4 * (vG >> 1) + vei;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const int byte = ((vG & 1) * (D / 2) + 16 * db + 4 * vai) * 2;
      va[db] = lds_addr(stV) + L::lds_row(k) * RB + (((byte >> 4) ^ tree_vswz<RB>(k)) << 4) + (byte & 15);
    }
  }

  pf32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pf32x16{};
  float m_run = -INFINITY, l_run = 0.f;

  if (t < t_end) {
    tile.locate(P, it, t, lane);
    tile.template issue<false, false>(kh, stK, lane);
    tile.template issue<true, false>(vh, stV, lane);
    // q and the mask bits are waited for here, not in the loop behind the DMA in flight there
#pragma unroll
    for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(qb[s].x), "+v"(qb[s].y), "+v"(qb[s].z), "+v"(qb[s].w));
    asm volatile("" : "+v"(first_bits.lo), "+v"(first_bits.hi));
    const uint32_t bits0 = first_bits.at(P, it, node, tm * kTreeKT);
    tile.look(P, it, t + kTreeWaves, lane);
    for (;;) {
      const uint32_t there = tile.there;
      uint32_t bits = there;
      if (t >= tree0) bits &= t == tm ? bits0 : tree_bits(P, it, node, t * kTreeKT);
      const int tn = t + kTreeWaves;
      tree_wait<NJ>();  // K: this tile's V came after it
      u32x4 kk[KS];
      if constexpr (KS == 8) lds_read8(kk, ka);
      else lds_read4(kk, ka);
      pf32x16 S = pf32x16{};
#pragma unroll
      for (int s = 0; s < KS; ++s) S = PMfma<DT>::run(__builtin_bit_cast(uint4, kk[s]), qb[s], S);
      const bool more = tn < t_end;
      tile.locate(P, it, tn, lane);
      if (more) tile.template issue<false, false>(kh, stK, lane);
      tile.look(P, it, tn + kTreeWaves, lane);
      const uint32_t mine = bits >> (4 * hh);
      if (__ballot(bits != 0xffffffffu)) {
#pragma unroll
        for (int e = 0; e < 16; ++e) S[e] = (mine >> (8 * (e >> 2) + (e & 3))) & 1 ? S[e] : -INFINITY;
      }
      float bm = -INFINITY;
#pragma unroll
      for (int e = 0; e < 16; ++e) bm = fmaxf(bm, S[e]);
      bm = half_max(bm) * P.scale2;  // scale > 0
      const float m_old = m_run;
      m_run = tree_new_max<DT>(m_old, bm);
      const float ms = m_run == -INFINITY ? 0.f : m_run;
      if (__ballot(m_run != m_old)) {
        const float alpha = m_run != m_old ? __builtin_amdgcn_exp2f(m_old - m_run) : 1.f;
        l_run *= alpha;
#pragma unroll
        for (int db = 0; db < DB; ++db) o[db] *= alpha;
      }
      float p[16], ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e], P.scale2, -ms));
        ps[e & 3] += p[e];
      }
      l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      uint4 pb[2];  // step u: keys 16 u + {4 h + j, 8 + 4 h + j}
#pragma unroll
      for (int u = 0; u < 2; ++u)
        pb[u] = make_uint4(PMfma<DT>::pack(p[8 * u], p[8 * u + 1]), PMfma<DT>::pack(p[8 * u + 2], p[8 * u + 3]),
                           PMfma<DT>::pack(p[8 * u + 4], p[8 * u + 5]), PMfma<DT>::pack(p[8 * u + 6], p[8 * u + 7]));
      if (more) tree_wait<NJ>();  // V: the next tile's K came after it
      else tree_wait<0>();
      if (there != 0xffffffffu) {
        tree_zero_rows<RB>(stV, there, lane);
        wave_lds_fence();
      }
      if (t >= tree0 && tree_v_odd<DT>(stV, TB, lane)) {
        tree_v_add_odd<DT, D>(o, stV, bits, kTreeKT, hh, [](int k) { return L::lds_row(k) * RB; });
        wave_lds_fence();
        tree_v_clean<DT>(stV, TB, lane * 16, 1024);
        wave_lds_fence();
      }
      u32x2 vv[4 * DB];
      if constexpr (DB == 4) lds_read_tr4(vv, va);
      else lds_read_tr2(vv, va);
#pragma unroll
      for (int i = 0; i < 2 * DB; ++i) {
        const u32x2 lo = vv[4 * (i % DB) + 2 * (i / DB)], hi = vv[4 * (i % DB) + 2 * (i / DB) + 1];
        o[i % DB] = PMfma<DT>::run(make_uint4(lo.x, lo.y, hi.x, hi.y), pb[i / DB], o[i % DB]);
      }
      t = tn;
      if (!more) break;
      tile.template issue<true, false>(vh, stV, lane);
    }
  }
  const float lt = half_sum(l_run);
  if (hh == 0) s_ml[wave][qc] = make_float2(m_run, lt);
#pragma unroll
  for (int x = 0; x < D / 8; ++x)
    *reinterpret_cast<float4*>(tree_piece<D>(stK, stV, x) + lane * 16) =
        make_float4(o[x / 4][4 * (x & 3)], o[x / 4][4 * (x & 3) + 1], o[x / 4][4 * (x & 3) + 2], o[x / 4][4 * (x & 3) + 3]);
  __syncthreads();
  tree_fold_store<D, DT, TB>(P, it, wave, lane, s_ml, sK, sV);
}

// fp32 queries and pools: the same walk on v_mfma_f32_32x32x2 (fp32 products
// and sums).  Step s of the score product multiplies channel s (lane half 0)
// and D/2 + s (half 1).  3 requests of up to 1500 rows: 10.2 us, the same chain of
// search, loads and fold as in the 16-bit kernel, with eight times its MFMA steps.
template <int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) tree_attn_f32_kernel(TreeParams P) {
  constexpr int DB = D / 32, RB = D * 4;
  constexpr int TB = kTreeKT * RB;
  typedef TreeTile<RB> Tile;
  typedef typename Tile::L L;
  constexpr int NJ = Tile::NJ;
  __shared__ __attribute__((aligned(16))) char sK[kTreeWaves][TB], sV[kTreeWaves][TB];
  __shared__ float2 s_ml[kTreeWaves][32];
  TreeItem it;
  if (!tree_find<kTreeKT, kTreeRows, true>(P, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int t_end = (int)((int64_t)it.tiles * (it.cut + 1) / it.cuts);
  int t = (int)((int64_t)it.tiles * it.cut / it.cuts) + wave;
  const int tree0 = it.ctx / kTreeKT;
  char* const stK = sK[wave];
  char* const stV = sV[wave];
  const char* kh = P.k + (int64_t)it.h * P.sh * 16;
  const char* vh = P.v + (int64_t)it.h * P.sh * 16;
  Tile tile;
  tile.look(P, it, t, lane);

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
  const int tm = t < tree0 ? t + (tree0 - t + kTreeWaves - 1) / kTreeWaves * kTreeWaves : t;
  TreeBits first_bits = {0, 0};
  if (tm < t_end) first_bits.load(P, it, node, tm * kTreeKT);

  typedef __attribute__((ext_vector_type(DB))) float vrow;
  const uint32_t krow = lds_addr(stK) + L::lds_row(qc) * RB;

  pf32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pf32x16{};
  float m_run = -INFINITY, l_run = 0.f;

  if (t < t_end) {
    tile.locate(P, it, t, lane);
    tile.template issue<false, true>(kh, stK, lane);
    tile.template issue<true, true>(vh, stV, lane);
#pragma unroll
    for (int s = 0; s < D / 2; ++s) asm volatile("" : "+v"(qf[s]));
    asm volatile("" : "+v"(first_bits.lo), "+v"(first_bits.hi));
    const uint32_t bits0 = first_bits.at(P, it, node, tm * kTreeKT);
    tile.look(P, it, t + kTreeWaves, lane);
    for (;;) {
      const uint32_t there = tile.there;
      uint32_t bits = there;
      if (t >= tree0) bits &= t == tm ? bits0 : tree_bits(P, it, node, t * kTreeKT);
      const int tn = t + kTreeWaves;
      tree_wait<NJ>();
      pf32x16 S = pf32x16{};
#pragma unroll
      for (int s0 = 0; s0 < D / 8; s0 += 8) {
        uint32_t ka[8];
        u32x4 kk[8];
#pragma unroll
        for (int s = 0; s < 8; ++s) ka[s] = krow + (((hh * (D / 8) + s0 + s) ^ tree_kswz<RB>(qc)) << 4);
        lds_read8(kk, ka);
#pragma unroll
        for (int s = 0; s < 8; ++s)
#pragma unroll
          for (int x = 0; x < 4; ++x)
            S = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(kk[s][x]), qf[4 * (s0 + s) + x], S, 0, 0, 0);
      }
      const bool more = tn < t_end;
      tile.locate(P, it, tn, lane);
      if (more) tile.template issue<false, true>(kh, stK, lane);
      tile.look(P, it, tn + kTreeWaves, lane);
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
      float p[16], ps[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[e], P.scale2, -ms));
        ps[e & 3] += p[e];
      }
      l_run += (ps[0] + ps[1]) + (ps[2] + ps[3]);
      if (more) tree_wait<NJ>();
      else tree_wait<0>();
      if (there != 0xffffffffu) {
        tree_zero_rows<RB>(stV, there, lane);
        wave_lds_fence();
      }
      // tree rows: values that are not finite reach the rows that see them only
      if (t >= tree0) {
        bool bad = false;
#pragma unroll 1
        for (int x = lane * 16; x < TB; x += 1024) {
          const float4 y = *reinterpret_cast<const float4*>(stV + x);
          bad |= (y.x * 0.f + y.y * 0.f) + (y.z * 0.f + y.w * 0.f) != 0.f;  // inf x 0 and NaN x 0 are NaN
        }
        if (__ballot(bad)) {
#pragma unroll 1
          for (int k = 0; k < kTreeKT; ++k) {
            const bool sees = (bits >> k) & 1;
#pragma unroll
            for (int e = 0; e < 16; ++e) {
              const vrow v =
                  *reinterpret_cast<const vrow*>(stV + L::lds_row(k) * RB + (8 * (e >> 2) + 4 * hh + (e & 3)) * DB * 4);
#pragma unroll
              for (int db = 0; db < DB; ++db) o[db][e] += sees && !(fabsf(v[db]) < INFINITY) ? v[db] : 0.f;
            }
          }
          wave_lds_fence();
#pragma unroll 1
          for (int x = lane * 4; x < TB; x += 256) {
            float* y = reinterpret_cast<float*>(stV + x);
            if (!(fabsf(*y) < INFINITY)) *y = 0.f;
          }
          wave_lds_fence();
        }
      }
      // a tile's products are summed by themselves and then added to O: its rounding error stays below one
      // accumulator's over all keys
      pf32x16 sum[DB];
#pragma unroll
      for (int db = 0; db < DB; ++db) sum[db] = pf32x16{};
#pragma unroll
      for (int e0 = 0; e0 < 16; e0 += 8) {
        uint32_t va[8];
        float v[8][DB];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          va[e] = lds_addr(stV) + L::lds_row(8 * ((e0 + e) >> 2) + 4 * hh + (e & 3)) * RB + qc * DB * 4;
        if constexpr (DB == 4) {
          u32x4 w[8];
          lds_read8(w, va);
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int db = 0; db < DB; ++db) v[e][db] = __uint_as_float(w[e][db]);
        } else {
          u32x2 w[8];
          lds_read8_b64(w, va);
#pragma unroll
          for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int db = 0; db < DB; ++db) v[e][db] = __uint_as_float(w[e][db]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int db = 0; db < DB; ++db)
            sum[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(v[e][db], p[e0 + e], sum[db], 0, 0, 0);
      }
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] += sum[db];
      t = tn;
      if (!more) break;
      tile.template issue<true, true>(vh, stV, lane);
    }
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
      *reinterpret_cast<float4*>(tree_piece<D>(stK, stV, i * DB + g) + lane * 16) =
          make_float4(x[0], x[1], x[2], x[3]);
    }
  __syncthreads();
  tree_fold_store<D, HALO_F32, TB>(P, it, wave, lane, s_ml, sK, sV);
}

// More than 32 rows a unit, 16 bits: NW waves of 32 rows each share every K/V
// tile, 64 keys staged in LDS (two stages of K and of V), one barrier a tile.
// K is staged two tiles ahead and V one, so the score products of tile t + 1
// are issued between the exponentials of tile t, and the maximum of tile t + 1
// between the output products of tile t: the matrix core and the VALU overlap
// within a wave.  Lane l of each wave looks up key l of a tile, so one vote gives the
// rows that are there, and hands the places to the lanes that stage them.
// 64 nodes of 4 heads (256 rows a unit) over 32768 rows, 8 KV heads: 57 us (51 to
// 66 by the card), 34.4 GFLOP at 600 TFLOP/s.  The matrix cores are busy 39 % of
// the cycles and the waves wait 39 % of theirs: products and exponentials are one
// instruction stream, and each tile ends in a full wait and a barrier with one
// workgroup a CU.  16 requests of 1024 to 32768 rows, 84 rows a unit: 55 us (52 to
// 63), 4.3 TB/s, the waves waiting 57 % of their cycles.
// Four stages of K and V took 57.7 where two took 55.7; finding a tile's places
// in the step that stages it cost 5 us of 52.
template <int DT, int D, int NW>
__global__ void __launch_bounds__(64 * NW) __attribute__((amdgpu_waves_per_eu(2, 2))) tree_attn_wide_kernel(TreeParams P) {
  constexpr int KT = kTreeWideKT, R = 32 * NW;
  constexpr int KS = D / 16, DB = D / 32, RB = D * 2;
  constexpr int TB = KT * RB;
  constexpr int NJ = TB / 1024 / NW;  // LDS-DMA instructions of a wave and tile
  typedef TreeLanes<RB, NJ> L;
  static_assert(L::KEYS * NW == KT, "the waves stage the tile");
  __shared__ __attribute__((aligned(16))) char sK0[TB], sK1[TB], sV0[TB], sV1[TB];
  TreeItem it;
  if (!tree_find<KT, R, true>(P, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int t_end = (int)((int64_t)it.tiles * (it.cut + 1) / it.cuts);
  const int t0 = (int)((int64_t)it.tiles * it.cut / it.cuts);
  const int tree0 = it.ctx / KT;  // first tile with tree rows
  const char* kh = P.k + (int64_t)it.h * P.sh * 16;
  const char* vh = P.v + (int64_t)it.h * P.sh * 16;

  TreeRow row;  // of key `lane` of the tile looked up last
  row.load(P, it, t0 * KT + lane);

  const int RG = it.n * P.rep;
  const int r_lane = it.rb * R + wave * 32 + qc;
  const bool active = it.rb * R + wave * 32 < RG;  // a wave past the rows only stages tiles
  const int r_eff = min(r_lane, RG - 1);
  const int node = r_eff / P.rep, head = it.h * P.rep + (r_eff - node * P.rep);
  uint4 qb[KS];
  {
    const char* qrow =
        reinterpret_cast<const char*>(P.q) + ((it.lo + node) * P.q_stride_n + head * P.q_stride_h) * 2;
#pragma unroll
    for (int s = 0; s < KS; ++s) qb[s] = *reinterpret_cast<const uint4*>(qrow + (s * 16 + hh * 8) * 2);
  }

  // a tile's staged places (of this wave's rows) and which of its keys are there
  struct Tile {
    uint32_t pl[NJ];
    uint64_t there;
  };
  int my_key = wave * L::KEYS + L::first(lane);
  auto locate = [&](int t) {
    Tile x;
    const bool ok = row.there(P);
    const uint32_t place = ok ? row.place(P) : kNoRow;
    x.there = __ballot(ok);
#pragma unroll
    for (int j = 0; j < NJ; ++j) x.pl[j] = __shfl(place, my_key + j * L::STEP, 64);
    row.load(P, it, (t + 1) * KT + lane);
    return x;
  };
  auto issue = [&](const Tile& x, const char* base, char* st, bool is_v) {
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      const int k = my_key + j * L::STEP, slot = lane % L::SL;
      const int piece = slot ^ (is_v ? tree_vswz<RB>(k) : tree_kswz<RB>(k));
      const char* from = base + (int64_t)x.pl[j] * 16 + (piece << 4);
      tree_dma(x.pl[j] == kNoRow ? reinterpret_cast<const char*>(tree_zeros) : from, st + (wave * NJ + j) * 1024);
    }
  };
  // Operand addresses: the key's LDS row and, xored, the piece.  lds_row takes
  // the bits of a key apart, so the rows of key step u are those of the first
  // by a constant.  kx and vx pass through a register of unknown value in each
  // tile: the xors are cheaper than keeping all their results.
  auto lds_row = [](int k) { return k / L::KEYS * L::KEYS + L::lds_row(k % L::KEYS); };
  const int kx0 = L::lds_row(qc % L::KEYS) * RB + qc / L::KEYS * L::KEYS * RB + ((hh ^ tree_kswz<RB>(qc)) << 4);
  auto kread = [&](const char* sk, int i, int kx) {  // step i: d-step i / 2, key block i % 2
    static_assert(32 % L::KEYS == 0, "key block 1 is 32 LDS rows on");
    return *reinterpret_cast<const uint4*>(sk + (i & 1) * 32 * RB + (kx ^ ((i >> 1) << 5)));
  };
  const int vG = lane >> 4, vkey = 4 * (vG >> 1) + ((lane & 15) >> 2), vai = lane & 3;
  const int vx0 = lds_row(vkey) * RB + ((((vG & 1) * (D / 16) + (vai >> 1)) ^ tree_vswz<RB>(vkey)) << 4) + 8 * (vai & 1);
  auto vread = [&](const char* sv, int i, int vx) {  // step i: key step i / DB, d-block i % DB
    const int u = i / DB;
    const char* at = sv + (vx ^ ((i % DB) << 5));
    const uint2 a0 = pf_tr16(at + lds_row(16 * u) * RB);
    const uint2 a1 = pf_tr16(at + lds_row(16 * u + 8) * RB);
    return make_uint4(a0.x, a0.y, a1.x, a1.y);
  };
  constexpr int NKS = 2 * KS;  // score MFMAs per tile
  constexpr int NPV = 4 * DB;  // output MFMAs per tile
  constexpr int RING = 4;      // operand reads in flight ahead of their MFMA

  pf32x16 o[DB];
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = pf32x16{};
  float m_run = -INFINITY, l_run = 0.f;

  Tile c1, c2;
  uint64_t there;  // of the tile whose scores are next
  {
    const Tile c0 = locate(t0);
    issue(c0, kh, sK0, false);
    issue(c0, vh, sV0, true);
    there = c0.there;
  }
  c1 = locate(t0 + 1);
  if (t0 + 1 < t_end) issue(c1, kh, sK1, false);
  c2 = locate(t0 + 2);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();

  // Masks scores by the keys of the tile that this lane's row sees.
  auto mask_by = [&](uint64_t bits, pf32x16* S) {
    const uint32_t m_lo = (uint32_t)bits >> (4 * hh), m_hi = (uint32_t)(bits >> 32) >> (4 * hh);
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        S[kb][e] = ((kb ? m_hi : m_lo) >> (8 * (e >> 2) + (e & 3))) & 1 ? S[kb][e] : -INFINITY;
  };
  uint64_t bits = 0;  // of the tile whose scores were masked last, where it is a tree tile
  auto mask_tile = [&](int t, pf32x16* S) {
    if (t >= tree0) {
      bits = there & (((uint64_t)tree_bits(P, it, node, t * KT + 32) << 32) | tree_bits(P, it, node, t * KT));
      mask_by(bits, S);
    } else if (there != ~0ull) {
      mask_by(there, S);
    }
  };
  float ms = 0.f;  // exponent offset of the current tile: m_run, or 0 while m_run is -inf
  auto take_max = [&](float bm) {  // the running max takes a tile's max into account, o and l follow
    bm = half_max(bm) * P.scale2;  // scale > 0
    const float m_old = m_run;
    m_run = tree_new_max<DT>(m_old, bm);
    ms = m_run == -INFINITY ? 0.f : m_run;
    if (__ballot(m_run != m_old)) {
      const float alpha = m_run != m_old ? __builtin_amdgcn_exp2f(m_old - m_run) : 1.f;
      l_run *= alpha;
#pragma unroll
      for (int db = 0; db < DB; ++db) o[db] *= alpha;
    }
  };
  auto scores = [&](const char* sk, int t, pf32x16* S) {  // not interleaved: the first tile and tree tiles
    int kx = kx0;
    asm volatile("" : "+v"(kx));
#pragma unroll
    for (int i = 0; i < NKS; ++i) S[i & 1] = PMfma<DT>::run(kread(sk, i, kx), qb[i >> 1], i < 2 ? pf32x16{} : S[i & 1]);
    mask_tile(t, S);
    float bm = -INFINITY;
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
      for (int e = 0; e < 16; ++e) bm = fmaxf(bm, S[kb][e]);
    take_max(bm);
  };

  pf32x16 S[2], S2[2];
  int t = t0;
  if (active) scores(sK0, t, S);
  __syncthreads();  // K stage 0 is refilled below

  // Stages K(t+2) over K(t) and V(t+1), and moves on the places.
  auto stage_next = [&](char* kcur, char* vnxt) {
    asm volatile("" : "+v"(my_key));  // the pieces are worked out anew in each tile
    if (t + 2 < t_end) issue(c2, kh, kcur, false);
    if (t + 1 < t_end) issue(c1, vh, vnxt, true);
    there = c1.there;
    c1 = c2;
    c2 = locate(t + 3);
  };
  auto end_tile = [&]() {
    __builtin_amdgcn_s_waitcnt(0);  // this wave's loads of K(t+2) and V(t+1) have landed
    __syncthreads();                // every wave's have; tile t's stages are free
    ++t;
  };
  // A tile whose next one has committed rows only.
  auto step = [&](auto stage_c, pf32x16* S, pf32x16* Sn) {
    constexpr int stage = decltype(stage_c)::value;
    char* const kcur = stage ? sK1 : sK0;  // K(t), scored; receives K(t+2)
    char* const knxt = stage ? sK0 : sK1;  // K(t+1)
    char* const vcur = stage ? sV1 : sV0;  // V(t)
    char* const vnxt = stage ? sV0 : sV1;  // receives V(t+1)
    stage_next(kcur, vnxt);
    if (active) {
      // Both blocks are issued in source order (a scheduling barrier after
      // each MFMA step): every MFMA's operand was read RING steps earlier, and
      // the VALU work is spread evenly between the MFMAs.
      int kx = kx0, vx = vx0;
      asm volatile("" : "+v"(kx), "+v"(vx));
      uint4 kr[RING], vr[RING];
#pragma unroll
      for (int i = 0; i < RING; ++i) kr[i] = kread(knxt, i, kx);
      constexpr int EPM = 32 / NKS;  // exponentials per score MFMA
      uint32_t pw[16];               // P^T: key step 2 kb + u, words 4 (2 kb + u) .., holds keys 16 u + {4 h + j, 8 + 4 h + j} of block kb
      float psum = 0.f;
#pragma unroll
      for (int i = 0; i < NKS; ++i) {
        Sn[i & 1] = PMfma<DT>::run(kr[i % RING], qb[i >> 1], i < 2 ? pf32x16{} : Sn[i & 1]);
        if (i + RING < NKS) kr[i % RING] = kread(knxt, i + RING, kx);
#pragma unroll
        for (int x = 0; x < EPM; x += 2) {
          const int w = (i * EPM + x) / 2, e = 2 * (w & 7);
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[w >> 3][e], P.scale2, -ms));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(S[w >> 3][e + 1], P.scale2, -ms));
          psum += p0;
          psum += p1;
          pw[w] = PMfma<DT>::pack(p0, p1);
          // keeps the exponentials in this block
          asm volatile("" : "+v"(pw[w]));
        }
        // keeps the additions next to their exponentials
        asm volatile("" : "+v"(psum));
        __builtin_amdgcn_sched_barrier(0);
      }
      l_run += psum;
      if (there != ~0ull) mask_by(there, Sn);

      constexpr int MPM = 32 / NPV;  // score elements folded into the max per output MFMA
      float bm = -INFINITY;
#pragma unroll
      for (int i = 0; i < RING; ++i) vr[i] = vread(vcur, i, vx);
#pragma unroll
      for (int i = 0; i < NPV; ++i) {
        const uint32_t* pb = pw + 4 * (i / DB);
        o[i % DB] = PMfma<DT>::run(vr[i % RING], make_uint4(pb[0], pb[1], pb[2], pb[3]), o[i % DB]);
        if (i + RING < NPV) vr[i % RING] = vread(vcur, i + RING, vx);
#pragma unroll
        for (int x = 0; x < MPM; ++x) {
          const int e = i * MPM + x;
          bm = fmaxf(bm, Sn[e >> 4][e & 15]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      take_max(bm);
    }
    end_tile();
  };
  // Steps in pairs, which leaves the stages and the scores where they were.
  const int t_steps = min(t_end, tree0) - 1;  // tiles before the last one, and before a tree tile
  while (t + 2 <= t_steps) {
    step(std::integral_constant<int, 0>(), S, S2);
    step(std::integral_constant<int, 1>(), S2, S);
  }
  // The last tile or two and the tree tiles, one product behind the other.
  int stage = 0;
  for (; t < t_end; stage ^= 1) {
    char* const vcur = stage ? sV1 : sV0;
    stage_next(stage ? sK1 : sK0, stage ? sV0 : sV1);
    // Tree rows whose values are not finite reach the rows that see them and are zeroed for the product.
    // Every wave finds the same: it reads the tile before any of them changes it.
    if (t >= tree0 && tree_v_odd<DT>(vcur, TB, lane)) {
      if (active) tree_v_add_odd<DT, D>(o, vcur, bits, KT, hh, [&](int k) { return lds_row(k) * RB; });
      __syncthreads();
      tree_v_clean<DT>(vcur, TB, threadIdx.x * 16, NW * 1024);
      __syncthreads();
    }
    if (active) {
      int vx = vx0;
      asm volatile("" : "+v"(vx));
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        uint4 pb[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          float p[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(S[kb][8 * u + e], P.scale2, -ms));
            l_run += p[e];
          }
          pb[u] = make_uint4(PMfma<DT>::pack(p[0], p[1]), PMfma<DT>::pack(p[2], p[3]), PMfma<DT>::pack(p[4], p[5]),
                             PMfma<DT>::pack(p[6], p[7]));
        }
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) o[i % DB] = PMfma<DT>::run(vread(vcur, kb * 2 * DB + i, vx), pb[i / DB], o[i % DB]);
      }
      if (t + 1 < t_end) scores(stage ? sK0 : sK1, t + 1, S);
    }
    end_tile();
  }

  if (r_lane >= RG) return;
  const float lt = half_sum(l_run);
  if (it.cuts > 1) {
    const int64_t pw = (int64_t)(it.part + it.cut) * NW + wave;
    float4* po = P.part_o + pw * (DB * 4 * 64) + lane;
#pragma unroll
    for (int x = 0; x < 4 * DB; ++x)
      po[x * 64] = make_float4(o[x / 4][4 * (x & 3)], o[x / 4][4 * (x & 3) + 1], o[x / 4][4 * (x & 3) + 2],
                               o[x / 4][4 * (x & 3) + 3]);
    if (hh == 0) P.part_ml[pw * 32 + qc] = make_float2(m_run, lt);
    return;
  }
  const float inv = tree_inv(lt);
  const int64_t at = (it.lo + node) * P.o_stride_n + head * P.o_stride_h;
#pragma unroll
  for (int x = 0; x < 4 * DB; ++x) {
    float v4[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) v4[j] = o[x / 4][4 * (x & 3) + j] * inv;
    tree_store4<DT>(P, at + tree_channel<D, false>(x, hh), v4);
  }
  if (P.lse != nullptr && hh == 0) P.lse[(int64_t)(it.lo + node) * P.H + head] = tree_lse(m_run, lt);
}

// Merge of a unit's partials: with M the largest of a row's maxima, out = sum_c
// 2^(m_c - M) o_c / sum_c 2^(m_c - M) l_c.  One workgroup folds four pieces of
// 32 rows, its MW waves every MW-th partial each, in batches of 8 whose loads
// are in flight together; the order is fixed.  Bound by the launch and one or
// two round trips: 8 units of 17 partials 4.0 us, of 29 5.1; 31 partials of 256 rows
// of 8 heads (33 MB) 8.9.  For MW see tree_shape.
constexpr int kMergeBatch = 8;
template <int D, int DT, int KT, int NW, int MW>
__global__ void __launch_bounds__(64 * MW) tree_merge_kernel(TreeParams P) {
  constexpr int PIECES = D / 8, PPW = 4;
  __shared__ float4 s_o[MW][PPW][64];
  __shared__ float2 s_ml[MW][32];
  TreeItem it;
  const int rows32 = NW == 1 ? 0 : blockIdx.x % NW;  // which 32 of the unit's rows
  if (!tree_find<KT, 32 * NW, false>(P, blockIdx.x / NW, it)) return;
  const int row0 = (it.rb * NW + rows32) * 32;
  if (row0 >= it.n * P.rep) return;
  const int lane = threadIdx.x & 63;
  const int wave = uni((int)(threadIdx.x >> 6));
  const int qc = lane & 31, hh = lane >> 5;
  const int x0 = blockIdx.y * PPW;
  const int r = row0 + qc;
  const bool live = r < it.n * P.rep;
  float m = -INFINITY, l = 0.f;
  float4 acc[PPW];
#pragma unroll
  for (int x = 0; x < PPW; ++x) acc[x] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int c0 = wave; live && c0 < it.cuts; c0 += MW * kMergeBatch) {
    float2 ml[kMergeBatch];
    float4 v[kMergeBatch][PPW];
#pragma unroll
    for (int y = 0; y < kMergeBatch; ++y) {
      ml[y].x = -INFINITY;
      if (c0 + y * MW < it.cuts) {
        const int64_t pu = (int64_t)(it.part + c0 + y * MW) * NW + rows32;
        ml[y] = P.part_ml[pu * 32 + qc];
#pragma unroll
        for (int x = 0; x < PPW; ++x) v[y][x] = P.part_o[pu * (PIECES * 64) + (x0 + x) * 64 + lane];
      }
    }
    float mn = m;
#pragma unroll
    for (int y = 0; y < kMergeBatch; ++y) mn = fmaxf(mn, ml[y].x);
    const float wo = tree_weight(m, mn);
    m = mn;
    l *= wo;
#pragma unroll
    for (int x = 0; x < PPW; ++x) acc[x] = make_float4(acc[x].x * wo, acc[x].y * wo, acc[x].z * wo, acc[x].w * wo);
#pragma unroll
    for (int y = 0; y < kMergeBatch; ++y) {
      if (c0 + y * MW < it.cuts) {
        const float w = tree_weight(ml[y].x, mn);
        l = __builtin_fmaf(ml[y].y, w, l);
#pragma unroll
        for (int x = 0; x < PPW; ++x) {
          acc[x].x = __builtin_fmaf(v[y][x].x, w, acc[x].x);
          acc[x].y = __builtin_fmaf(v[y][x].y, w, acc[x].y);
          acc[x].z = __builtin_fmaf(v[y][x].z, w, acc[x].z);
          acc[x].w = __builtin_fmaf(v[y][x].w, w, acc[x].w);
        }
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
  for (int w = 0; w < MW; ++w) M = fmaxf(M, s_ml[w][qc].x);
  float wt[MW];
  l = 0.f;
#pragma unroll
  for (int w = 0; w < MW; ++w) {
    wt[w] = tree_weight(s_ml[w][qc].x, M);
    l += s_ml[w][qc].y * wt[w];
  }
  const float inv = tree_inv(l);
  const int node = r / P.rep, head = it.h * P.rep + (r - node * P.rep);
  const int64_t row = it.lo + node;
#pragma unroll
  for (int x = wave; x < PPW; x += MW) {
    float v4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < MW; ++w) {
      const float4 y = s_o[w][x][lane];
      v4[0] += y.x * wt[w];
      v4[1] += y.y * wt[w];
      v4[2] += y.z * wt[w];
      v4[3] += y.w * wt[w];
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) v4[j] *= inv;
    tree_store4<DT>(P, row * P.o_stride_n + head * P.o_stride_h + tree_channel<D, DT == HALO_F32>(x0 + x, hh), v4);
  }
  if (P.lse != nullptr && blockIdx.y == 0 && wave == 0 && hh == 0) P.lse[row * P.H + head] = tree_lse(M, l);
}

}  // namespace halo

using namespace halo;

namespace {

// How a call is cut: 32-row waves that share a unit's tiles (1: the narrow
// kernel), units at most, workgroups that the GPU holds, launch size, partials
// at most.
struct TreeShape {
  int nw, kt, slots, min_tiles, mw;
  int64_t units, grid, partials;
  bool merge;
};
TreeShape tree_shape(int dtype, int B, int H, int H_kv, int D, int64_t max_rows, int max_nodes) {
  TreeShape s;
  const int64_t rows = (int64_t)max_nodes * (H / H_kv);
  // As few waves as hold the rows.  48 rows, one request of 32768: two waves
  // 40.7 us, four 39.6, two blocks of the narrow kernel 49.4; 64 rows, 16 of
  // 8192: 120, 116 and 156; 48 rows, 64 of 1024: 65.7, 67.6 and 78.7.  128 rows,
  // 16 of 8192: four waves 124, eight 175, two blocks of two 176; 32 rows, 16 of
  // 8192: the narrow kernel 106, two waves 118.
  s.nw = dtype == HALO_F32 || rows <= 32 ? 1 : rows <= 64 ? 2 : rows <= 128 ? 4 : 8;
  s.kt = s.nw == 1 ? kTreeKT : kTreeWideKT;
  s.units = (int64_t)B * H_kv * ((rows + 32 * s.nw - 1) / (32 * s.nw));
  // Two workgroups a CU fit by their LDS (64 KiB at D = 128, 32 KiB at D = 64,
  // the fp32 kernel's twice that) and 2 waves a SIMD, one of 8 waves.  Few units
  // are cut into one a CU: half the partials, and the same bandwidth (8 units of
  // 32768 rows 36.3 -> 34.2 us, of 131072 105 -> 101, 32 units of 8192 34.7 ->
  // 34.0; 128 units of 8192 would go from 106 to 120 by the coarser cuts).
  const bool few = s.nw == 1 && s.units <= 32;
  s.slots = 256 * (few || s.nw == 8 || (dtype == HALO_F32 && D == 128) ? 1 : 2);
  // The least L: a tile a wave, or two for the pipeline.  A unit of more tiles is
  // cut into ceil(tiles / L) even items, which may be about half as long (5 tiles
  // become 2 and 3).  With 4, 8 and 16 in the narrow kernel 1000 rows took 12.2,
  // 12.9 and 14.6 us, in fp32 3 requests of 900 13.4, 15.4 and 20.3.
  s.min_tiles = s.nw == 1 ? kTreeWaves : 2;
  // 8 waves of the merge have 64 partials in one round trip (129 partials of one
  // unit 8.7 us, with four waves 9.5; 52 of 4 units 5.7 and 6.0; 29 of 8 units 5.1
  // both); many units of few partials need the workgroups side by side (128 units
  // of 3 partials of 64 rows: four waves 7.7, eight 12.5).
  s.mw = s.slots >= 16 * s.units ? 8 : 4;
  const int64_t longest = (max_rows + max_nodes + s.kt - 1) / s.kt;
  s.merge = longest > s.min_tiles;
  // tree_find: at most `room` items besides one a unit
  s.grid = s.merge ? (s.slots / 2 + s.units > s.slots ? s.slots / 2 + s.units : s.slots) : s.units;
  s.partials = s.merge ? (int64_t)s.slots * s.nw : 0;
  return s;
}

int64_t tree_part_bytes(int D) { return 32ll * D * 4 + 32 * 8; }

bool tree_sizes_ok(int B, int H, int H_kv, int D, int64_t max_rows, int max_nodes) {
  return B > 0 && H > 0 && H_kv > 0 && H % H_kv == 0 && (D == 64 || D == 128) && max_rows > 0 &&
         max_rows < (1ll << 31) - 1024 && max_nodes > 0 && max_nodes <= 512 && (int64_t)max_nodes * (H / H_kv) < (1 << 24) &&
         (int64_t)B * H_kv * ((int64_t)max_nodes * (H / H_kv) / 32 + 8) < (1ll << 30);
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
  HALO_CHECK_ARG(out_dtype == HALO_F32 || out_dtype == dtype, "out must be of q's type or fp32");
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
  const int64_t ea = 4 * elem_size(out_dtype);
  HALO_CHECK_ARG(reinterpret_cast<uintptr_t>(out) % ea == 0 && out_stride_n % 4 == 0 && out_stride_h % 4 == 0,
                 "out rows must be aligned to four elements");
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
  p.out_f32 = out_dtype == HALO_F32;
  p.lse = lse;
  p.part_o = reinterpret_cast<float4*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + s.partials * 32 * (D / 4));
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)s.grid), block(64 * (s.nw == 1 ? kTreeWaves : s.nw)),
      mgrid((unsigned)((s.units < s.slots / 2 ? s.units : s.slots / 2) * s.nw), D / 32);  // units that can be cut
#define HALO_TREE(KERNEL, DV, DTV, KTV, NWV)                                                                      \
  do {                                                                                                             \
    hipLaunchKernelGGL((KERNEL), grid, block, 0, st, p);                                                           \
    if (s.merge && s.mw == 8)                                                                                      \
      hipLaunchKernelGGL((tree_merge_kernel<DV, DTV, KTV, NWV, 8>), mgrid, dim3(512), 0, st, p);                   \
    else if (s.merge)                                                                                              \
      hipLaunchKernelGGL((tree_merge_kernel<DV, DTV, KTV, NWV, 4>), mgrid, dim3(256), 0, st, p);                   \
  } while (0)
#define HALO_TREE_WIDE(DTV, DV, NWV) HALO_TREE((tree_attn_wide_kernel<DTV, DV, NWV>), DV, DTV, kTreeWideKT, NWV)
#define HALO_TREE16(DTV, DV)                                                                     \
  do {                                                                                           \
    if (s.nw == 1) HALO_TREE((tree_attn_kernel<DTV, DV>), DV, DTV, kTreeKT, 1);                \
    else if (s.nw == 2) HALO_TREE_WIDE(DTV, DV, 2);                                              \
    else if (s.nw == 4) HALO_TREE_WIDE(DTV, DV, 4);                                              \
    else HALO_TREE_WIDE(DTV, DV, 8);                                                             \
  } while (0)
  if (dtype == HALO_F32) {
    if (D == 128) HALO_TREE((tree_attn_f32_kernel<128>), 128, HALO_F32, kTreeKT, 1);
    else HALO_TREE((tree_attn_f32_kernel<64>), 64, HALO_F32, kTreeKT, 1);
  } else if (dtype == HALO_BF16) {
    if (D == 128) HALO_TREE16(HALO_BF16, 128);
    else HALO_TREE16(HALO_BF16, 64);
  } else {
    if (D == 128) HALO_TREE16(HALO_F16, 128);
    else HALO_TREE16(HALO_F16, 64);
  }
#undef HALO_TREE16
#undef HALO_TREE_WIDE
#undef HALO_TREE
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
