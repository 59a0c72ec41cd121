// Blocks of a paged cache handed from request to request (gfx950): requests
// that go on with another's blocks or give theirs up, and the used blocks of a
// pool moved to its front.
//
// shared[x] counts the requests beyond the first that hold block x, so it is 0
// for the blocks that halo_update_block_tables hands out, and that call needs
// no counts.  The reference keeps blocks (halo/memory_tier.py:45-60) but gives
// them to no request; everything here is this library's own.
#include "block_pool.hpp"

namespace halo {
namespace {

constexpr int kMoveThreads = 256;
constexpr int kPlanThreads = 1024;
constexpr int kMaxRequests = 4096;  // of fork_blocks: their counts lie in LDS

// Sum over the workgroup's threads before this one, and the whole sum.
__device__ __forceinline__ int plan_scan(int x, int* s_wave, int* all) {
  constexpr int WAVES = kPlanThreads / 64;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  const int in = wave_prefix(x);
  __syncthreads();  // the sums of an earlier scan have been read
  if (lane == 63) s_wave[wave] = in;
  __syncthreads();
  const int t = lane < WAVES ? s_wave[lane] : 0;
  const int ws = wave_prefix(t);
  *all = lane_of(ws, WAVES - 1);
  return lane_of(ws - t, wave) + in - x;
}

// ---------------------------------------------------------------------------
// Forks.  Row b of the table goes on with row a = source[b] as it was before
// the call.  With c_a the number of rows that go on with a, a block in a full
// entry of row a gains c_a - 1 holders, one in another entry loses its holder
// if c_a = 0 and else goes to a's heir; the sums of these gains over the rows
// that hold a block are whole numbers, so their order does not matter.  Blocks
// whose holders come to none are pushed in the order of their ids, and the rows
// that need a block for a copy pop theirs in the rows' order.
//
// Four launches, each a few dependent reads: begin 2.8 us, count 4.0 to 4.9, plan
// 6.5, apply 6.8 for 32 beams of 256 to 4096 rows, 28 layers (19 MB of copies would
// take 3.8).  All but the copies in one workgroup took 12.9 us where three
// launches take 13.5, and 17 for 64 rows of 1026 entries.
// ---------------------------------------------------------------------------
// What a row becomes: whose blocks, how many of them, a block for a copy or -1;
// and what that holds: the block to copy and how many of its rows.
struct ForkPlan {
  int from, keep, fresh, ok, old, rows;
};

struct ForkParams {
  PoolView pool;
  int32_t* table;
  int64_t table_stride;
  int32_t* n_blocks;
  int B, W;
  int32_t* free_blocks;
  int n_cap;
  int32_t* n_free;
  int32_t* shared;
  const int32_t* lengths;
  const int32_t* source;
  int32_t* new_lengths;
  uint8_t* ok;
  // workspace
  int32_t* old_table;  // (B, W)
  int32_t* change;     // (blocks)
  int4* rows;          // (B) ForkRow
  ForkPlan* plans;     // (B)
};

// A row as it was: its blocks, the rows it holds in them, how many rows go on
// with it, and the one of them that has its last blocks.
struct ForkRow {
  int own, len, count, heir;
};
__global__ void __launch_bounds__(kPlanThreads) fork_begin_kernel(ForkParams P) {
  const int64_t n = (int64_t)P.B * P.W;
  if (blockIdx.x != 0) {
    const int64_t at = (int64_t)(blockIdx.x - 1) * kPlanThreads + threadIdx.x, step = (int64_t)(gridDim.x - 1) * kPlanThreads;
    for (int64_t i = at; i < P.pool.blocks; i += step) P.change[i] = 0;
    for (int64_t i = at; i < n; i += step) P.old_table[i] = P.table[i / P.W * P.table_stride + i % P.W];
    return;
  }
  __shared__ int s_count[kMaxRequests], s_heir[kMaxRequests];
  for (int b = threadIdx.x; b < P.B; b += kPlanThreads) s_count[b] = 0, s_heir[b] = 0x7fffffff;
  __syncthreads();
  for (int b = threadIdx.x; b < P.B; b += kPlanThreads) {
    const int a = P.source[b];
    if ((uint32_t)a < (uint32_t)P.B) {
      atomicAdd(&s_count[a], 1);
      atomicMin(&s_heir[a], a == b ? -1 : b);  // -1: it stays its own
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < P.B; b += kPlanThreads) {
    const int own = min(max(P.n_blocks[b], 0), P.W);
    const int len = (int)min((int64_t)max(P.lengths[b], 0), (int64_t)own * P.pool.bs.d);
    P.rows[b] = make_int4(own, len, s_count[b], s_heir[b] == -1 ? b : s_heir[b]);
  }
}

__device__ __forceinline__ ForkRow fork_row(const ForkParams& P, int b) {
  const int4 r = P.rows[b];
  return {r.x, r.y, r.z, r.w};
}

// One column of kCountRows rows a thread: rows of one request's samples hold the
// same blocks, whose gains go to memory as one (64 rows of 1024 blocks given up:
// 9.7 us with an addition for each entry, 4.4 so).
constexpr int kCountRows = 16;
__global__ void __launch_bounds__(kMoveThreads) fork_count_kernel(ForkParams P) {
  const int j = blockIdx.x * kMoveThreads + threadIdx.x, b0 = blockIdx.y * kCountRows;
  int x[kCountRows], gain[kCountRows];
#pragma unroll
  for (int k = 0; k < kCountRows; ++k) {
    const int b = min(b0 + k, P.B - 1);
    const ForkRow r = fork_row(P, b);
    gain[k] = b0 + k >= P.B || j >= r.own || r.count == 1 ? 0 : j < div_by(r.len, P.pool.bs) ? r.count - 1 : r.count > 0 ? 0 : -1;
    x[k] = gain[k] != 0 ? P.old_table[(int64_t)b * P.W + j] : -1;
  }
  int sum = 0;
#pragma unroll
  for (int k = 0; k < kCountRows; ++k) {
    sum += gain[k];
    const bool last = k + 1 == kCountRows || x[k + 1] != x[k];
    if (last && sum != 0 && (uint32_t)x[k] < (uint32_t)P.pool.blocks) atomicAdd(&P.change[x[k]], sum);
    if (last) sum = 0;
  }
}

__device__ __forceinline__ bool fork_freed(const ForkParams& P, int x) {
  const int c = P.change[x];
  return c < 0 && P.shared[x] + 1 + c <= 0;
}

// What row b goes on with, as the rows were.
struct ForkFrom {
  int a, full, rows, old;
  bool lives, heir, wants;
  ForkRow r;
};
__device__ __forceinline__ ForkFrom fork_from(const ForkParams& P, int b) {
  ForkFrom f;
  f.a = P.source[b];
  f.lives = (uint32_t)f.a < (uint32_t)P.B;
  f.r = f.lives ? fork_row(P, f.a) : ForkRow{0, 0, 0, -1};
  f.full = div_by(f.r.len, P.pool.bs);
  f.rows = f.r.len - f.full * P.pool.bs.d;
  f.heir = f.lives && f.r.heir == b;
  f.wants = f.lives && !f.heir && f.rows > 0;
  f.old = f.wants ? P.old_table[(int64_t)f.a * P.W + f.full] : -1;
  return f;
}

__global__ void __launch_bounds__(kPlanThreads) fork_plan_kernel(ForkParams P) {
  __shared__ int s_wave[kPlanThreads / 64];
  const int tid = threadIdx.x;
  const int nf = min(max(*P.n_free, 0), P.n_cap);
  // a thread has rows, and blocks, that lie side by side; its first row is on its way with the blocks
  const int per_b = (P.B + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(tid * per_b, P.B), b1 = min(b0 + per_b, P.B);
  const ForkFrom first = fork_from(P, min(b0, P.B - 1));
  const int per = (P.pool.blocks + kPlanThreads - 1) / kPlanThreads;
  const int x0 = (int)min((int64_t)tid * per, (int64_t)P.pool.blocks), x1 = min(x0 + per, P.pool.blocks);
  int mine = 0, freed, wants_all;
#pragma unroll 4
  for (int x = x0; x < x1; ++x) mine += fork_freed(P, x);
  const int before = plan_scan(mine, s_wave, &freed);
  int my_wants = 0;
  for (int b = b0; b < b1; ++b) my_wants += b == b0 ? first.wants : fork_from(P, b).wants;
  const int wants_before = plan_scan(my_wants, s_wave, &wants_all);
  const int top = (int)min((int64_t)nf + freed, (int64_t)P.n_cap);
  const bool ok = wants_all <= top;
  if (ok && mine > 0) {
    int at = nf + before;
    for (int x = x0; x < x1; ++x)
      if (fork_freed(P, x)) {
        if (at < P.n_cap) P.free_blocks[at] = x;
        ++at;
      }
  }
  __threadfence();
  __syncthreads();
  int nth = wants_before;
  for (int b = b0; b < b1; ++b) {
    const ForkFrom f = b == b0 ? first : fork_from(P, b);
    ForkPlan p = {f.lives ? f.a : -1, !f.lives ? 0 : f.heir ? f.r.own : f.full, -1, ok, f.old, f.rows};
    if (ok && f.wants) p.fresh = P.free_blocks[top - 1 - nth++];
    P.new_lengths[b] = ok ? f.r.len : P.lengths[b];
    P.plans[b] = p;
  }
  if (tid == 0) {
    *P.ok = ok;
    if (ok) *P.n_free = top - wants_all;
  }
}

// The first `meta` workgroups write counts and tables, the others copy the rows
// of partly filled blocks, all layers.
template <int PB>
__global__ void __launch_bounds__(kMoveThreads) fork_apply_kernel(ForkParams P, int meta, int splits) {
  typedef typename Piece<PB>::type T;
  if ((int)blockIdx.x < meta) {
    if (!*P.ok) return;
    const int64_t at = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x, step = (int64_t)meta * kMoveThreads;
    for (int64_t x = at; x < P.pool.blocks; x += step) {
      const int c = P.change[x];
      if (c != 0) P.shared[x] = max(P.shared[x] + c, 0);
    }
    for (int64_t i = at; i < (int64_t)P.B * P.W; i += step) {
      const int b = (int)(i / P.W), j = (int)(i - (int64_t)b * P.W);
      const ForkPlan p = P.plans[b];
      if (p.from == b) continue;
      const int last = p.keep + (p.fresh >= 0);
      P.table[b * P.table_stride + j] = j < p.keep ? P.old_table[(int64_t)p.from * P.W + j] : j < last ? p.fresh : -1;
      if (j == 0) P.n_blocks[b] = last;
    }
    return;
  }
  const int item = blockIdx.x - meta;
  const int b = item / splits, split = item - b * splits;
  const ForkPlan p = P.plans[b];
  if (!p.ok || (uint32_t)p.old >= (uint32_t)P.pool.blocks || (uint32_t)p.fresh >= (uint32_t)P.pool.blocks) return;
  const int per_row = P.pool.D_bytes / PB, per_head = p.rows * per_row;
  const int64_t from = p.old * P.pool.sb, to = p.fresh * P.pool.sb;
  for (int u = split; u < 2 * P.pool.layers * P.pool.H_kv; u += splits) {
    const int h = u % P.pool.H_kv, l = u / P.pool.H_kv >> 1, is_v = u / P.pool.H_kv & 1;
    char* base = (is_v ? P.pool.v : P.pool.k) + l * P.pool.sl + h * P.pool.sh;
    for (int x = threadIdx.x; x < per_head; x += kMoveThreads) {
      const int r = x / per_row;
      const int64_t o = r * P.pool.sr + (x - r * per_row) * PB;
      *reinterpret_cast<T*>(base + to + o) = *reinterpret_cast<const T*>(base + from + o);
    }
  }
}

// ---------------------------------------------------------------------------
// Compaction.  Of the blocks that are used or free, in the order of their ids,
// the first U (as many as are used) shall be the used ones: with rank(x) the
// number of such blocks before x, the free blocks of rank below U are gaps and
// the used ones of rank U and above move, the i-th of these into the i-th gap.
// The number of gaps before x is rank(x) - used(x), so one scan places all.
//
// The moves are bound by memory: 480 blocks of 8 layers of 32 KiB, K and V, 0.5 GB
// read and written in 92 to 102 us (a plain copy of as much 99); the three
// launches in front of them take 16 (five blocks of a small pool: 1.4, 1.6, 5.4
// and 5.1 us).
// ---------------------------------------------------------------------------
struct CompactParams {
  PoolView pool;
  int32_t* table;
  int64_t table_stride;
  const int32_t* n_blocks;
  int B, W;
  int32_t* free_blocks;
  int n_cap;
  int32_t* n_free;
  int32_t* shared;
  int32_t* new_id;
  int32_t* n_used;
  // workspace
  int32_t* flag;  // (blocks) 1: used, 2: free
  int32_t* gaps;  // (blocks)
  int32_t* used;  // (blocks) used blocks by rank among them
  int32_t* n_moves;
};

__global__ void __launch_bounds__(kMoveThreads) compact_begin_kernel(CompactParams P) {
  for (int64_t i = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x; i < P.pool.blocks; i += (int64_t)gridDim.x * kMoveThreads) {
    P.flag[i] = 0;
    P.new_id[i] = (int)i;
  }
}

__global__ void __launch_bounds__(kMoveThreads) compact_mark_kernel(CompactParams P) {
  const int64_t at = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x, step = (int64_t)gridDim.x * kMoveThreads;
  const int nf = min(max(*P.n_free, 0), P.n_cap);
  for (int64_t i = at; i < nf; i += step) {
    const int x = P.free_blocks[i];
    if ((uint32_t)x < (uint32_t)P.pool.blocks) atomicOr(&P.flag[x], 2);
  }
  for (int64_t i = at; i < (int64_t)P.B * P.W; i += step) {
    const int b = (int)(i / P.W), j = (int)(i - (int64_t)b * P.W);
    if (j >= P.n_blocks[b]) continue;
    const int x = P.table[b * P.table_stride + j];
    if ((uint32_t)x < (uint32_t)P.pool.blocks) atomicOr(&P.flag[x], 1);
  }
}

__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(CompactParams P) {
  __shared__ int s_wave[kPlanThreads / 64], s_gaps;
  const int tid = threadIdx.x;
  const int per = (P.pool.blocks + kPlanThreads - 1) / kPlanThreads;
  const int x0 = (int)min((int64_t)tid * per, (int64_t)P.pool.blocks), x1 = min(x0 + per, P.pool.blocks);
  int mine = 0, mine_used = 0, there, U;
  for (int x = x0; x < x1; ++x) {
    const int f = P.flag[x];
    mine += f != 0;
    mine_used += f & 1;
  }
  if (tid == 0) s_gaps = 0;
  int rank = plan_scan(mine, s_wave, &there);
  int used = plan_scan(mine_used, s_wave, &U);
  int gaps = 0;
  for (int x = x0; x < x1; ++x) {
    const int f = P.flag[x];
    if (f == 0) continue;
    if (rank >= U) {  // free afterwards, the lowest on top: a free block, or one that a move leaves
      const int at = there - 1 - rank;
      if (at < P.n_cap) P.free_blocks[at] = x;
    }
    if (f & 1) {
      P.used[used++] = x;
    } else if (rank < U) {
      P.gaps[rank - used] = x;
      ++gaps;
    }
    ++rank;
  }
  if (gaps) atomicAdd(&s_gaps, gaps);
  __threadfence();
  __syncthreads();
  const int n = s_gaps;
  for (int i = tid; i < n; i += kPlanThreads) {
    const int from = P.used[U - n + i], to = P.gaps[i];
    P.new_id[from] = to;
    P.shared[to] = P.shared[from];
    P.shared[from] = 0;
  }
  if (tid == 0) {
    *P.n_moves = n;
    *P.n_used = U;
    *P.n_free = min(there - U, P.n_cap);
  }
}

template <int PB>
__global__ void __launch_bounds__(kMoveThreads) compact_apply_kernel(CompactParams P, int meta) {
  typedef typename Piece<PB>::type T;
  if ((int)blockIdx.x < meta) {
    const int64_t at = (int64_t)blockIdx.x * kMoveThreads + threadIdx.x, step = (int64_t)meta * kMoveThreads;
    for (int64_t i = at; i < (int64_t)P.B * P.W; i += step) {
      const int b = (int)(i / P.W), j = (int)(i - (int64_t)b * P.W);
      if (j >= P.n_blocks[b]) continue;
      int32_t* e = P.table + b * P.table_stride + j;
      const int x = *e;
      if ((uint32_t)x < (uint32_t)P.pool.blocks) *e = P.new_id[x];
    }
    return;
  }
  const int per_unit = 2 * P.pool.layers;
  const int64_t units = (int64_t)*P.n_moves * per_unit;
  const int U = *P.n_used, n = *P.n_moves;
  const int per_row = P.pool.D_bytes / PB, per_head = P.pool.bs.d * per_row;
  for (int64_t u = blockIdx.x - meta; u < units; u += gridDim.x - meta) {
    const int i = (int)(u / per_unit), w = (int)(u - (int64_t)i * per_unit);
    const int from = P.used[U - n + i], to = P.gaps[i];
    char* base = (w & 1 ? P.pool.v : P.pool.k) + (w >> 1) * P.pool.sl;
    for (int64_t x = threadIdx.x; x < (int64_t)P.pool.H_kv * per_head; x += kMoveThreads) {
      const int h = (int)(x / per_head), y = (int)(x - (int64_t)h * per_head), r = y / per_row;
      const int64_t o = h * P.pool.sh + r * P.pool.sr + (y - r * per_row) * PB;
      *reinterpret_cast<T*>(base + to * P.pool.sb + o) = *reinterpret_cast<const T*>(base + from * P.pool.sb + o);
    }
  }
}

int64_t align16(int64_t x) { return (x + 15) / 16 * 16; }

unsigned groups(int64_t n, int threads, int most) {
  const int64_t g = (n + threads - 1) / threads;
  return (unsigned)(g < 1 ? 1 : g < most ? g : most);
}

}  // namespace
}  // namespace halo

using namespace halo;

extern "C" size_t halo_fork_workspace_size(int B, int W, int blocks) {
  if (B <= 0 || W <= 0 || blocks <= 0) return 0;
  return (size_t)(align16((int64_t)B * W * 4) + align16((int64_t)blocks * 4) + (int64_t)B * (sizeof(int4) + sizeof(ForkPlan)));
}

extern "C" int halo_fork_blocks(const halo_block_pool* pool, int32_t* table, int64_t table_stride, int32_t* n_blocks,
                                int B, int W, int32_t* free_blocks, int n_cap, int32_t* n_free, int32_t* shared,
                                const int32_t* lengths, const int32_t* source, int32_t* new_lengths, uint8_t* ok,
                                void* workspace, size_t workspace_bytes, void* stream) {
  ForkParams p;
  const int rc = check_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  HALO_CHECK_ARG(table && n_blocks && (free_blocks || n_cap == 0) && n_free && shared && lengths && source && new_lengths && ok,
                 "null pointer argument");
  HALO_CHECK_ARG(B > 0 && B <= kMaxRequests && W > 0 && n_cap >= 0, "need 1 <= B <= 4096 and positive sizes");
  HALO_CHECK_ARG(table_stride >= W && (int64_t)B * W < (1ll << 31) - 4096 && (int64_t)W * pool->block_size < (1ll << 31),
                 "table too large, or its rows overlap");
  HALO_CHECK_ARG(new_lengths != lengths, "new_lengths must not be lengths");
  HALO_CHECK_ARG((int64_t)pool->layers * pool->H_kv < (1 << 30), "too many layers and heads");
  HALO_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace missing or not 16-byte aligned");
  if (workspace_bytes < halo_fork_workspace_size(B, W, pool->blocks)) {
    set_error("workspace too small");
    return HALO_E_WORKSPACE;
  }
  p.table = table;
  p.table_stride = table_stride;
  p.n_blocks = n_blocks;
  p.B = B;
  p.W = W;
  p.free_blocks = free_blocks;
  p.n_cap = n_cap;
  p.n_free = n_free;
  p.shared = shared;
  p.lengths = lengths;
  p.source = source;
  p.new_lengths = new_lengths;
  p.ok = ok;
  char* ws = static_cast<char*>(workspace);
  p.rows = reinterpret_cast<int4*>(ws);
  p.plans = reinterpret_cast<ForkPlan*>(p.rows + B);
  p.old_table = reinterpret_cast<int32_t*>(p.plans + B);
  p.change = p.old_table + align16((int64_t)B * W * 4) / 4;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t entries = (int64_t)B * W;
  const int64_t most = entries > pool->blocks ? entries : pool->blocks;
  hipLaunchKernelGGL(fork_begin_kernel, dim3(1 + groups(most, kPlanThreads, 256)), dim3(kPlanThreads), 0, st, p);
  hipLaunchKernelGGL(fork_count_kernel, dim3((unsigned)((W + kMoveThreads - 1) / kMoveThreads), (unsigned)((B + kCountRows - 1) / kCountRows)),
                     dim3(kMoveThreads), 0, st, p);
  hipLaunchKernelGGL(fork_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
  const int meta = (int)groups(most, kMoveThreads, 512);
  const int64_t units = 2ll * pool->layers * pool->H_kv;
  const int splits = (int)(units < 64 ? units : 64);
  const dim3 grid((unsigned)(meta + B * splits)), block(kMoveThreads);
  const int pb = piece_bytes(p.pool, 0);
  if (pb == 16) hipLaunchKernelGGL(fork_apply_kernel<16>, grid, block, 0, st, p, meta, splits);
  else if (pb == 4) hipLaunchKernelGGL(fork_apply_kernel<4>, grid, block, 0, st, p, meta, splits);
  else hipLaunchKernelGGL(fork_apply_kernel<2>, grid, block, 0, st, p, meta, splits);
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}

extern "C" size_t halo_compact_workspace_size(int blocks) {
  return blocks <= 0 ? 0 : (size_t)(3 * align16((int64_t)blocks * 4) + 16);
}

extern "C" int halo_compact_blocks(const halo_block_pool* pool, int32_t* table, int64_t table_stride,
                                   const int32_t* n_blocks, int B, int W, int32_t* free_blocks, int n_cap, int32_t* n_free,
                                   int32_t* shared, int32_t* new_id, int32_t* n_used, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  CompactParams p;
  const int rc = check_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  HALO_CHECK_ARG(table && n_blocks && (free_blocks || n_cap == 0) && n_free && shared && new_id && n_used,
                 "null pointer argument");
  HALO_CHECK_ARG(B > 0 && W > 0 && n_cap >= 0, "sizes must be positive");
  HALO_CHECK_ARG(table_stride >= W && (int64_t)B * W < (1ll << 31) - 4096, "table too large, or its rows overlap");
  HALO_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace missing or not 16-byte aligned");
  if (workspace_bytes < halo_compact_workspace_size(pool->blocks)) {
    set_error("workspace too small");
    return HALO_E_WORKSPACE;
  }
  p.table = table;
  p.table_stride = table_stride;
  p.n_blocks = n_blocks;
  p.B = B;
  p.W = W;
  p.free_blocks = free_blocks;
  p.n_cap = n_cap;
  p.n_free = n_free;
  p.shared = shared;
  p.new_id = new_id;
  p.n_used = n_used;
  const int64_t part = align16((int64_t)pool->blocks * 4) / 4;
  p.flag = static_cast<int32_t*>(workspace);
  p.gaps = p.flag + part;
  p.used = p.gaps + part;
  p.n_moves = p.used + part;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const int64_t entries = (int64_t)B * W, marks = entries > n_cap ? entries : n_cap;
  hipLaunchKernelGGL(compact_begin_kernel, dim3(groups(pool->blocks, kMoveThreads, 512)), dim3(kMoveThreads), 0, st, p);
  hipLaunchKernelGGL(compact_mark_kernel, dim3(groups(marks, kMoveThreads, 1024)), dim3(kMoveThreads), 0, st, p);
  hipLaunchKernelGGL(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, p);
  const int meta = (int)groups(entries, kMoveThreads, 512);
  const dim3 grid((unsigned)(meta + 2048)), block(kMoveThreads);
  const int pb = piece_bytes(p.pool, 0);
  if (pb == 16) hipLaunchKernelGGL(compact_apply_kernel<16>, grid, block, 0, st, p, meta);
  else if (pb == 4) hipLaunchKernelGGL(compact_apply_kernel<4>, grid, block, 0, st, p, meta);
  else hipLaunchKernelGGL(compact_apply_kernel<2>, grid, block, 0, st, p, meta);
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
