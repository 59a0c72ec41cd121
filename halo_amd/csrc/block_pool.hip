// Block-pool operators of batched decoding with drafted trees (gfx950): block
// tables and slot maps from the requests' lengths, rows written to their
// slots, ancestor masks of drafted trees, and the accepted path's rows moved
// behind the committed ones.
//
// A pool is one tier buffer of the cold-KV store: K and V as (layers, blocks,
// H_kv, block_size, D).  Row p of a request lies in row p % block_size of
// block table[p / block_size]; slot = block * block_size + row names a row of
// the pool.  The reference keeps such blocks (halo/memory_tier.py:45-60) but
// gives them to no request; everything here is this library's own.
#include "block_pool.hpp"

namespace halo {
namespace {

// ---------------------------------------------------------------------------
// Block tables and slots.  need_b = ceil(length_b / block_size); surplus
// blocks go back first, then requests take theirs in order.  With R_b, G_b
// and C_b the sums over b' < b of blocks given back, blocks wanted and new rows,
// every moved id and every slot has a place of its own:
//   entry j of b goes to   free[n_free + R - 1 - (R_b + j - need_b)],
//   entry j of b comes from free[n_free + R - 1 - (G_b + j - own_b)],
//   new row r has           b = the last one with C_b <= r.
// (Requests that are served and grow come before those that want blocks and are
// not, so G_b counts no block that stays.)  One workgroup: a call of a few blocks
// is bound by the chain lengths -> sums -> ids -> slots, not by bytes.  The ids of
// 1024 requests are spread over the threads by a search in their sums (of the
// requests that move any), four neighbouring ids a thread for one search, so one
// long request does not hold up the others; the next ids are on their way
// meanwhile.  16 requests with a few blocks each: 5.3 us (an empty launch is about
// 2); the 11 600 blocks of 256 prompts: 11.2 us to hand out, 9.6 to take back,
// where the one CU's moves bound it (with a search for every id 14.4 and 12.4).
// ---------------------------------------------------------------------------
constexpr int kTabThreads = 1024;
constexpr int64_t kTabNone = -(1ll << 62);  // base of a request that was not served

struct TableParams {
  int32_t* table;
  int64_t table_stride;
  int32_t* n_blocks;
  int B, W;
  int32_t* free_blocks;
  int n_cap;
  int32_t* n_free;
  const int32_t* lengths;
  const int32_t* first;
  Div bs;
  int max_rows;
  int32_t* cu_rows;
  int64_t* slots;
  uint8_t* ok;
};

struct TabReq {
  int own, need, rows;  // blocks it has and needs, new rows
  __device__ __forceinline__ int back() const { return max(own - need, 0); }
  __device__ __forceinline__ int grow(int W) const { return need <= W ? max(need - own, 0) : 0; }
};
__device__ __forceinline__ TabReq tab_req(const TableParams& P, int b) {
  TabReq r = {0, 0, 0};
  if (b < P.B) {
    const int len = max(P.lengths[b], 0);
    r.rows = max(len - max(P.first[b], 0), 0);
    r.own = min(max(P.n_blocks[b], 0), P.W);
    r.need = div_by(len, P.bs);
    if (r.need * P.bs.d < len) ++r.need;
  }
  return r;
}

// Exclusive sums over the workgroup's threads, and the whole sums.  Blocks of
// all requests number below 2^31, rows may not.
struct TabSums {
  int back, grow, i_back, i_grow;  // i_: how many requests before this one give back, want blocks
  int all_back, all_grow, n_back, n_grow;
  int64_t rows, all_rows;
};
struct TabWave {
  int back, grow, n;  // n: requests that give back, and in the upper half those that want blocks
  int64_t rows;
};
__device__ __forceinline__ TabSums tab_scan(int back, int grow, int rows, TabWave* s_wave) {
  constexpr int WAVES = kTabThreads / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int xb = wave_prefix(back), xg = wave_prefix(grow);
  const int64_t xr = wave_prefix((int64_t)rows);
  const uint64_t hb = __ballot(back > 0), hg = __ballot(grow > 0), below = (1ull << lane) - 1;
  __syncthreads();  // the sums of an earlier scan have been read
  if (lane == 63) s_wave[wave] = {xb, xg, (int)(__popcll(hb) | __popcll(hg) << 16), xr};
  __syncthreads();
  TabWave t = {0, 0, 0, 0};
  if (lane < WAVES) t = s_wave[lane];
  const int wb = wave_prefix(t.back), wg = wave_prefix(t.grow), wn = wave_prefix(t.n);
  const int64_t wr = wave_prefix(t.rows);
  TabSums s;
  s.all_back = lane_of(wb, WAVES - 1);
  s.all_grow = lane_of(wg, WAVES - 1);
  s.n_back = lane_of(wn, WAVES - 1) & 0xffff;
  s.n_grow = lane_of(wn, WAVES - 1) >> 16;
  s.all_rows = lane_of(wr, WAVES - 1);
  const int n_before = lane_of(wn - t.n, wave);
  s.back = lane_of(wb - t.back, wave) + xb - back;
  s.grow = lane_of(wg - t.grow, wave) + xg - grow;
  s.i_back = (n_before & 0xffff) + (int)__popcll(hb & below);
  s.i_grow = (n_before >> 16) + (int)__popcll(hg & below);
  s.rows = lane_of(wr - t.rows, wave) + xr - rows;
  return s;
}

// The last i in [0, n) with at[i] <= x (at[0] <= x, ascending).
__device__ __forceinline__ int tab_find(const int* at, int n, int x) {
  int i = 0;
  for (int s = 1 << (31 - __clz(n)); s > 0; s >>= 1) {
    const int c = i + s;
    if (at[min(c, n - 1)] <= x && c < n) i = c;
  }
  return i;
}

// Blocks x .. x + 3 of those that the listed requests move: entry i of the list
// moves blocks at[i] .. at[i + 1] - 1, at least one, to or from table[base[i] + x],
// or nowhere where its base is kTabNone.  e: where they stand in the table, less
// than 0 for one that does not move; true where the four lie side by side.
__device__ __forceinline__ bool tab_places(const int* at, const int64_t* base, int n, int all, int x,
                                           int64_t (&e)[4]) {
  int i = tab_find(at, n, x);
  const bool same = x + 3 < all && (i + 1 == n || at[i + 1] > x + 3);
  e[0] = base[i] + x;
  if (!same) {
#pragma unroll
    for (int u = 1; u < 4; ++u) {
      if (i + 1 < n && at[i + 1] <= x + u) ++i;
      e[u] = x + u < all ? base[i] + x + u : -1;
    }
  }
  return same;
}

// Four ids on the stack, the first on top, `left` of them there.
struct TabIds {
  int32_t id[4];
  __device__ __forceinline__ void load(const int32_t* top, int left) {
    if (left >= 4) {
      int32_t v[4];
      __builtin_memcpy(v, top - 3, 16);
#pragma unroll
      for (int u = 0; u < 4; ++u) id[u] = v[3 - u];
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (u < left) id[u] = top[-u];
    }
  }
};

// Slot of new row r: -1 behind the last row and for rows of requests that were not served.
__device__ __forceinline__ int64_t tab_slot(const TableParams& P, const int32_t* cu, int r) {
  if (r >= cu[P.B]) return -1;
  const int b = tab_find(cu, P.B, r);
  if (!P.ok[b]) return -1;
  const int p = max(P.first[b], 0) + (r - cu[b]);
  const int c = div_by(p, P.bs);
  return (int64_t)P.table[b * P.table_stride + c] * P.bs.d + (p - c * P.bs.d);
}

// SLOTS: also the slots, by the same workgroup.
template <bool SLOTS>
__global__ void __launch_bounds__(kTabThreads) update_tables_kernel(TableParams P) {
  __shared__ TabWave s_wave[kTabThreads / 64];
  __shared__ int s_at[kTabThreads], s_cu[kTabThreads + 1], s_taken;
  __shared__ int64_t s_base[kTabThreads];
  const int tid = threadIdx.x;
  const int nf = min(max(*P.n_free, 0), P.n_cap);
  const bool one = P.B <= kTabThreads;  // all requests at once: one look at them, one scan
  TabReq r = tab_req(P, tid);
  TabSums s = tab_scan(r.back(), r.grow(P.W), r.rows, s_wave);
  int all_back = s.all_back;
  for (int b0 = kTabThreads; b0 < P.B; b0 += kTabThreads)
    all_back += tab_scan(tab_req(P, b0 + tid).back(), 0, 0, s_wave).all_back;
  if (tid == 0) s_taken = 0;

  int before = 0;
  for (int b0 = 0; all_back > 0 && b0 < P.B; b0 += kTabThreads) {
    if (!one) {
      r = tab_req(P, b0 + tid);
      s = tab_scan(r.back(), r.grow(P.W), r.rows, s_wave);
    }
    __syncthreads();
    if (r.back() > 0) {
      s_at[s.i_back] = s.back;
      s_base[s.i_back] = (int64_t)(b0 + tid) * P.table_stride + r.need - s.back;
    }
    __syncthreads();
    for (int x0 = tid * 4; x0 < s.all_back; x0 += kTabThreads * 4) {
      int64_t e[4];
      int32_t id[4];
      const bool same = tab_places(s_at, s_base, s.n_back, s.all_back, x0, e);
      const int64_t to = (int64_t)nf + all_back - 1 - (before + x0);  // of the first, the others below it
      if (same) {
        __builtin_memcpy(id, P.table + e[0], 16);
        const int32_t gone[4] = {-1, -1, -1, -1};
        __builtin_memcpy(P.table + e[0], gone, 16);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (e[u] >= 0) id[u] = P.table[e[u]];
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (e[u] >= 0) P.table[e[u]] = -1;
      }
      if (same && to < P.n_cap) {
        const int32_t v[4] = {id[3], id[2], id[1], id[0]};
        __builtin_memcpy(P.free_blocks + to - 3, v, 16);
      } else {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if ((same || e[u] >= 0) && to - u < P.n_cap) P.free_blocks[to - u] = id[u];
      }
    }
    before += s.all_back;
  }

  const int avail = (int)min((int64_t)nf + all_back, (int64_t)P.n_cap);
  int64_t wanted_before = 0, rows_before = 0;
  for (int b0 = 0; b0 < P.B; b0 += kTabThreads) {
    if (!one) {
      r = tab_req(P, b0 + tid);
      s = tab_scan(r.back(), r.grow(P.W), r.rows, s_wave);
    }
    const int grow = r.grow(P.W);
    const bool ok = r.need <= P.W && (grow == 0 || wanted_before + s.grow + grow <= avail);
    __syncthreads();
    if (grow > 0) {
      s_at[s.i_grow] = s.grow;
      s_base[s.i_grow] = ok ? (int64_t)(b0 + tid) * P.table_stride + r.own - s.grow : kTabNone;
    }
    if (b0 + tid < P.B) {
      const int32_t cu = (int32_t)min(rows_before + s.rows, (int64_t)0x7fffffff);
      P.cu_rows[b0 + tid] = cu;
      s_cu[tid] = cu;
      P.ok[b0 + tid] = ok;
      if (ok) P.n_blocks[b0 + tid] = r.need;
      if (ok && grow > 0) atomicMax(&s_taken, (int)(wanted_before + s.grow + grow));
    }
    __syncthreads();
    const int most = (int)min((int64_t)s.all_grow, avail - wanted_before);
    TabIds ids, next;  // the next ones are on their way during the search
    const int32_t* top = P.free_blocks + (avail - 1 - wanted_before);
    ids.load(top - tid * 4, most - tid * 4);
    for (int x0 = tid * 4; x0 < most; x0 += kTabThreads * 4) {
      next.load(top - (x0 + kTabThreads * 4), most - (x0 + kTabThreads * 4));
      int64_t e[4];
      const bool same = tab_places(s_at, s_base, s.n_grow, most, x0, e);
      if (same && e[0] >= 0) {
        __builtin_memcpy(P.table + e[0], ids.id, 16);
      } else if (!same) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (e[u] >= 0) P.table[e[u]] = ids.id[u];
      }
      ids = next;
    }
    wanted_before += s.all_grow;
    rows_before += s.all_rows;
  }
  const int32_t n_rows = (int32_t)min(rows_before, (int64_t)0x7fffffff);
  if (tid == 0) {
    P.cu_rows[P.B] = n_rows;
    *P.n_free = avail - s_taken;
  }
  if constexpr (SLOTS) {
    if (tid == 0 && one) s_cu[P.B] = n_rows;
    __syncthreads();
    for (int x = tid; x < P.max_rows; x += kTabThreads)
      P.slots[x] = one ? tab_slot(P, s_cu, x) : tab_slot(P, P.cu_rows, x);
  }
}

// Slots of long batches, one a thread over the whole GPU: each is a search in
// the sums and one read of the table (183 000 in 3.9 us, 0.4 TB/s of slots
// written: launch and latency).
constexpr int kSlotThreads = 256;
__global__ void __launch_bounds__(kSlotThreads) slots_kernel(TableParams P) {
  __shared__ int s_cu[kTabThreads + 1];
  const int r = blockIdx.x * kSlotThreads + threadIdx.x;
  if (P.B <= kTabThreads) {  // the search is a chain of reads: in LDS
    for (int i = threadIdx.x; i <= P.B; i += kSlotThreads) s_cu[i] = P.cu_rows[i];
    __syncthreads();
    if (r < P.max_rows) P.slots[r] = tab_slot(P, s_cu, r);
  } else if (r < P.max_rows) {
    P.slots[r] = tab_slot(P, P.cu_rows, r);
  }
}

// ---------------------------------------------------------------------------
// Rows to their slots and along an accepted path: copies of whole rows, PB
// bytes a thread (16 where everything is aligned for it).
// ---------------------------------------------------------------------------
struct AppendParams {
  PoolView pool;
  const char* k;
  const char* v;
  int64_t ksl, ksn, ksh, vsl, vsn, vsh;  // strides of the new rows in bytes
  const int64_t* slots;
  int N;
};

constexpr int kAppThreads = 256;

// One piece of one row a thread.  32768 rows of 2 KiB, K and V (268 MB read and
// written): 51 to 56 us by the card (4.8 to 5.3 TB/s; a plain copy of as much
// 50 to 52).  Two, four and eight rows a thread took 51, 56 and 139 where one
// took 49.  203 rows: 2.6 us, the launch.
template <int PB>
__global__ void __launch_bounds__(kAppThreads) append_rows_kernel(AppendParams P) {
  typedef typename Piece<PB>::type T;
  const int per_head = P.pool.D_bytes / PB;
  const int per_row = P.pool.H_kv * per_head;
  const int cols = min(per_row, kAppThreads);
  const int at_once = kAppThreads / cols;  // rows of a workgroup
  const int row_in = threadIdx.x / cols;
  const int r = blockIdx.x * at_once + row_in;
  if (row_in >= at_once || r >= P.N) return;
  const int64_t slot = P.slots[r];
  if (slot < 0 || slot >= (int64_t)P.pool.blocks * P.pool.bs.d) return;
  const int layer = blockIdx.y;
  const bool is_v = blockIdx.z != 0;
  const char* src = is_v ? P.v + layer * P.vsl + r * P.vsn : P.k + layer * P.ksl + r * P.ksn;
  const int64_t sh = is_v ? P.vsh : P.ksh;
  const int blk = div_by((int)slot, P.pool.bs);
  char* dst = (is_v ? P.pool.v : P.pool.k) + layer * P.pool.sl + blk * P.pool.sb +
              (slot - (int64_t)blk * P.pool.bs.d) * P.pool.sr;
  for (int c = threadIdx.x - row_in * cols; c < per_row; c += cols) {
    const int h = c / per_head, x = (c - h * per_head) * PB;
    *reinterpret_cast<T*>(dst + h * P.pool.sh + x) =
        __builtin_nontemporal_load(reinterpret_cast<const T*>(src + h * sh + x));
  }
}

struct CommitParams {
  PoolView pool;
  const int32_t* table;
  int64_t table_stride;
  int W;
  const int32_t* lengths;
  const int32_t* path;
  int64_t path_stride;
  int n_path_max;
  const int32_t* n_path;
  int32_t* new_lengths;
};

constexpr int kMaxPath = 64;
constexpr int kCommitThreads = 256;

// Byte offset of row p of a request in a layer of the pool, or -1.
__device__ __forceinline__ int64_t row_offset(const PoolView& pool, const int32_t* table, int W, int64_t p) {
  if (p < 0 || p > 0x7fffffff) return -1;
  const int c = div_by((int)p, pool.bs);
  if (c >= W) return -1;
  const int blk = table[c];
  if (blk < 0 || blk >= pool.blocks) return -1;
  return blk * pool.sb + (p - (int64_t)c * pool.bs.d) * pool.sr;
}

// Row length + j of request b receives what row length + path[j] held.  A
// path rises, so path[j] >= j and a row is written only after every move that
// reads it: a thread takes one column of all rows in order and needs no other.
// Lane j of each wave finds move j; the path ends at the first entry that does
// not rise or whose rows the table does not hold.  Eight rows are in flight a
// thread.  One request, 32 layers of 2 KiB rows, 5 accepted nodes: 4.0 us, the
// chain path -> table -> rows; 32 requests, 28 layers of 1 KiB rows, up to 8
// nodes: 7.8 us (2.8 TB/s of rows of 256 bytes).
template <int PB>
__global__ void __launch_bounds__(kCommitThreads) commit_path_kernel(CommitParams P) {
  typedef typename Piece<PB>::type T;
  const int b = blockIdx.y;
  const int lane = threadIdx.x & 63;
  const int len = max(P.lengths[b], 0);
  const int np = min(max(P.n_path[b], 0), P.n_path_max);
  int64_t from = -1, to = -1;
  bool good = false;
  {
    const int32_t* path = P.path + b * P.path_stride;
    const int at = lane < np ? path[lane] : -1;
    const int last = __shfl_up(at, 1, 64);
    if (lane < np) {
      from = row_offset(P.pool, P.table + b * P.table_stride, P.W, (int64_t)len + at);
      to = row_offset(P.pool, P.table + b * P.table_stride, P.W, (int64_t)len + lane);
      good = at > (lane == 0 ? -1 : last) && from >= 0 && to >= 0;
    }
  }
  const uint64_t bad = ~__ballot(good);
  const int n = bad == 0 ? 64 : __builtin_ctzll(bad);
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) P.new_lengths[b] = len + n;

  const int per_head = P.pool.D_bytes / PB;
  const int per_layer = P.pool.H_kv * per_head;
  const int64_t x = (int64_t)blockIdx.x * kCommitThreads + threadIdx.x;
  const int layer = (int)(x / per_layer);
  const int c = (int)(x - (int64_t)layer * per_layer);
  const int h = c / per_head;
  const bool live = layer < P.pool.layers;
  char* col = (blockIdx.z != 0 ? P.pool.v : P.pool.k) + layer * P.pool.sl + h * P.pool.sh + (c - h * per_head) * PB;
  constexpr int U = 8;
  for (int j0 = 0; j0 < n; j0 += U) {
    T v[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (live && j0 + u < n) v[u] = *reinterpret_cast<const T*>(col + lane_of(from, min(j0 + u, 63)));
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t f = lane_of(from, min(j0 + u, 63)), t = lane_of(to, min(j0 + u, 63));
      if (live && j0 + u < n && f != t) *reinterpret_cast<T*>(col + t) = v[u];
    }
  }
}

// ---------------------------------------------------------------------------
// Ancestor masks.  With M_i the set of node i and its ancestors at most s - 1
// steps up and a_i the ancestor s steps up, M_i | M_{a_i} reaches 2 s - 1
// steps: log2(depth) rounds, one workgroup per tree, the sets in LDS.  Bound by
// the launch and two reads: 4 trees of 16 nodes 2.9 us, 256 of 200 4.7.
// ---------------------------------------------------------------------------
constexpr int kMaxNodes = 512;
constexpr int kTreeThreads = 256;

template <int WORDS>
__global__ void __launch_bounds__(kTreeThreads)
    tree_layout_kernel(const int32_t* parents, const int32_t* cu, int N, int max_nodes, int words, uint64_t* mask,
                       int64_t mask_stride, int32_t* depth) {
  constexpr int NODES = WORDS * 64;
  constexpr int PER = (NODES + kTreeThreads - 1) / kTreeThreads;  // nodes a thread
  __shared__ uint64_t s_bits[NODES][WORDS];
  __shared__ int s_up[NODES];
  const int lo = max(cu[blockIdx.x], 0);
  const int n = min(min(max(cu[blockIdx.x + 1], 0), N) - lo, max_nodes);
  if (n <= 0) return;
  uint64_t bits[PER][WORDS];
  int up[PER];
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = threadIdx.x + k * kTreeThreads;
    up[k] = -1;
    if (i < n) {
      const int p = parents[lo + i];
      up[k] = p >= 0 && p < i ? p : -1;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        bits[k][w] = (i >> 6) == w ? 1ull << (i & 63) : 0;
        s_bits[i][w] = bits[k][w];
      }
      s_up[i] = up[k];
    }
  }
  bool more = false;
#pragma unroll
  for (int k = 0; k < PER; ++k) more |= up[k] >= 0;
  while (__syncthreads_or(more)) {
#pragma unroll
    for (int k = 0; k < PER; ++k)
      if (up[k] >= 0) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) bits[k][w] |= s_bits[up[k]][w];
        up[k] = s_up[up[k]];
      }
    __syncthreads();
    more = false;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = threadIdx.x + k * kTreeThreads;
      if (i < n) {
#pragma unroll
        for (int w = 0; w < WORDS; ++w) s_bits[i][w] = bits[k][w];
        s_up[i] = up[k];
      }
      more |= up[k] >= 0;
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = threadIdx.x + k * kTreeThreads;
    if (i < n) {
      int ones = 0;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        if (w < words) mask[(int64_t)(lo + i) * mask_stride + w] = bits[k][w];
        ones += __popcll(bits[k][w]);
      }
      depth[lo + i] = ones - 1;
    }
  }
}

}  // namespace
}  // namespace halo

using namespace halo;

extern "C" int halo_update_block_tables(int32_t* table, int64_t table_stride, int32_t* n_blocks, int B, int W,
                                        int32_t* free_blocks, int n_cap, int32_t* n_free, const int32_t* lengths,
                                        const int32_t* first, int block_size, int max_rows, int32_t* cu_rows,
                                        int64_t* slots, uint8_t* ok, void* stream) {
  HALO_CHECK_ARG(table && n_blocks && (free_blocks || n_cap == 0) && n_free && lengths && first && cu_rows && ok,
                 "null pointer argument");
  HALO_CHECK_ARG(B > 0 && W > 0 && n_cap >= 0 && block_size > 0 && max_rows >= 0 && (max_rows == 0 || slots),
                 "bad sizes");
  // counts of blocks, and a step of the loops over them past the last, in 31 bits
  HALO_CHECK_ARG(table_stride >= W && (int64_t)B * W < (1ll << 31) - kTabThreads * 4 &&
                     (int64_t)W * block_size < (1ll << 31),
                 "table too large, or its rows overlap");
  TableParams p = {table, table_stride, n_blocks, B, W, free_blocks, n_cap, n_free, lengths, first,
                   make_div(block_size), max_rows, cu_rows, slots, ok};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  // up to 4 slots a thread of the one workgroup cost less than a second launch
  const bool here = max_rows <= 4 * kTabThreads;
  if (here) hipLaunchKernelGGL(update_tables_kernel<true>, dim3(1), dim3(kTabThreads), 0, st, p);
  else {
    hipLaunchKernelGGL(update_tables_kernel<false>, dim3(1), dim3(kTabThreads), 0, st, p);
    hipLaunchKernelGGL(slots_kernel, dim3((unsigned)(((int64_t)max_rows + kSlotThreads - 1) / kSlotThreads)),
                       dim3(kSlotThreads), 0, st, p);
  }
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}

extern "C" int halo_append_rows(const halo_block_pool* pool, const void* k, int64_t k_stride_l, int64_t k_stride_n,
                                int64_t k_stride_h, const void* v, int64_t v_stride_l, int64_t v_stride_n,
                                int64_t v_stride_h, const int64_t* slots, int N, void* stream) {
  AppendParams p;
  const int rc = check_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  HALO_CHECK_ARG(N >= 0 && (N == 0 || (k && v && slots)), "null pointer argument");
  HALO_CHECK_ARG(pool->layers <= 65535, "at most 65535 layers");
  if (N == 0) return HALO_OK;
  const int64_t es = elem_size(pool->dtype);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.ksl = k_stride_l * es;
  p.ksn = k_stride_n * es;
  p.ksh = k_stride_h * es;
  p.vsl = v_stride_l * es;
  p.vsn = v_stride_n * es;
  p.vsh = v_stride_h * es;
  p.slots = slots;
  p.N = N;
  const int pb = piece_bytes(p.pool, reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                                         (uint64_t)(p.ksl | p.ksn | p.ksh | p.vsl | p.vsn | p.vsh));
  const int per_row = p.pool.H_kv * (p.pool.D_bytes / pb);
  const int rows = kAppThreads / (per_row < kAppThreads ? per_row : kAppThreads);
  const dim3 grid((unsigned)((N + rows - 1) / rows), (unsigned)pool->layers, 2), block(kAppThreads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (pb == 16) hipLaunchKernelGGL(append_rows_kernel<16>, grid, block, 0, st, p);
  else if (pb == 4) hipLaunchKernelGGL(append_rows_kernel<4>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(append_rows_kernel<2>, grid, block, 0, st, p);
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}

extern "C" int halo_commit_path(const halo_block_pool* pool, const int32_t* table, int64_t table_stride, int B, int W,
                                const int32_t* lengths, const int32_t* path, int64_t path_stride, int n_path_max,
                                const int32_t* n_path, int32_t* new_lengths, void* stream) {
  CommitParams p;
  const int rc = check_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  HALO_CHECK_ARG(table && lengths && path && n_path && new_lengths, "null pointer argument");
  HALO_CHECK_ARG(B > 0 && B <= 65535 && W > 0 && n_path_max > 0 && n_path_max <= kMaxPath,
                 "need 1 <= B <= 65535 and paths of at most 64 entries");
  HALO_CHECK_ARG(new_lengths != lengths, "new_lengths must not be lengths: other workgroups still read them");
  p.table = table;
  p.table_stride = table_stride;
  p.W = W;
  p.lengths = lengths;
  p.path = path;
  p.path_stride = path_stride;
  p.n_path_max = n_path_max;
  p.n_path = n_path;
  p.new_lengths = new_lengths;
  const int pb = piece_bytes(p.pool, 0);
  const int64_t cols = (int64_t)pool->layers * pool->H_kv * (p.pool.D_bytes / pb);
  HALO_CHECK_ARG(cols < (1ll << 31), "rows of all layers too long");
  const dim3 grid((unsigned)((cols + kCommitThreads - 1) / kCommitThreads), (unsigned)B, 2), block(kCommitThreads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (pb == 16) hipLaunchKernelGGL(commit_path_kernel<16>, grid, block, 0, st, p);
  else if (pb == 4) hipLaunchKernelGGL(commit_path_kernel<4>, grid, block, 0, st, p);
  else hipLaunchKernelGGL(commit_path_kernel<2>, grid, block, 0, st, p);
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}

extern "C" int halo_tree_layout(const int32_t* parents, const int32_t* cu_nodes, int B, int N, int max_nodes,
                                int64_t* mask, int64_t mask_stride, int32_t* depth, void* stream) {
  HALO_CHECK_ARG(parents && cu_nodes && mask && depth, "null pointer argument");
  HALO_CHECK_ARG(B > 0 && N > 0 && max_nodes > 0 && max_nodes <= kMaxNodes, "need 1 <= max_nodes <= 512");
  const int words = (max_nodes + 63) / 64;
  HALO_CHECK_ARG(mask_stride >= words, "mask rows overlap");
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  uint64_t* m = reinterpret_cast<uint64_t*>(mask);
  const dim3 grid((unsigned)B), block(kTreeThreads);
#define HALO_LAYOUT(WV) \
  hipLaunchKernelGGL(tree_layout_kernel<WV>, grid, block, 0, st, parents, cu_nodes, N, max_nodes, words, m, \
                     mask_stride, depth)
  if (words == 1) HALO_LAYOUT(1);
  else if (words == 2) HALO_LAYOUT(2);
  else if (words <= 4) HALO_LAYOUT(4);
  else HALO_LAYOUT(8);
#undef HALO_LAYOUT
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
