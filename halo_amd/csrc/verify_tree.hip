// Verification of drafted trees (gfx950): the path of drafted tokens that a
// target's probabilities accept, from given random numbers, and the token that
// follows it.
//
// At node c, with p the target's probabilities behind it, its children are
// tried in order.  Child j with token t was drawn from q_j: the draft's
// probabilities q behind c (replacement), q without the tokens rejected before
// (none twice: q_j(t) = q(t) / (1 - Q_j), Q_j their sum in q), or t itself (no
// draft probabilities, q_j(t) = 1).  With R_0 = p and Z_0 = 1,
//   accept iff u q_j(t) Z_j < R_j(t),
//   else R_{j+1}(v) = max(R_j(v) - Z_j q_j(v), 0), Z_{j+1} = sum_v R_{j+1}(v),
// which leaves the target's distribution whatever the draft's.  A rejected
// token has R(t) < Z q(t) and stays at 0, and max(max(a - b, 0) - c, 0) =
// max(a - b - c, 0) for b, c >= 0, so one number says what is left:
//   R_j(v) = max(p(v) - S_j q(v), 0), 0 for rejected tokens,
//   S_{j+1} = S_j + Z_j, or + Z_j / (1 - Q_j) without replacement,
// and without draft probabilities R is p without the rejected tokens.  Where no
// child is accepted the next token is the first v whose R(0) + .. + R(v)
// exceeds u sum R.  Sums and products are in 64 bits: a sum of 100 000 terms in
// 32 would move the borders between tokens.
//
// The reference drafts no tokens; this is the library's own.
#include "block_pool.hpp"

namespace halo {
namespace {

constexpr int kVerMaxNodes = 512, kVerMaxPath = 64;
constexpr int kWalkThreads = 1024, kSumThreads = 256;
constexpr int kEach = 8;                     // tokens of a thread
constexpr int kSlab = kSumThreads * kEach;   // of a workgroup of the sums

// Where a request's walk ended: its last node's row, what is left of that row's
// probabilities, and the tokens rejected there.
struct VerifyEnd {
  double S;
  int32_t row, n_gone;  // row -1: a request without nodes
  int32_t gone[kVerMaxNodes];
};

struct VerifyParams {
  const int64_t* tokens;
  const int32_t* parents;
  const int32_t* cu;
  int B, N, max_nodes, V;
  const void* p;
  int64_t p_stride;
  const void* q;
  int64_t q_stride;
  int replacement;
  const float* accept;
  const float* sample;
  int max_path;
  int32_t* path;
  int32_t* n_path;
  int64_t* token;
  VerifyEnd* ends;
  double2* parts;  // (B, slabs): sums of R and of p
  int slabs;
};

// A probability; NaN and what is below 0 count as 0.
template <int DT>
__device__ __forceinline__ float prob(const void* base, int64_t at) {
  return fmaxf(load_elem(base, at, DT), 0.f);
}
// Those of kEach tokens from v on, 0 from V on.  Rows begin at any element: the
// wide loads need no alignment.
template <int DT>
__device__ __forceinline__ void probs_at(const void* base, int64_t row, int v, int V, float (&f)[kEach]) {
  constexpr int ES = DT == HALO_F32 ? 4 : 2, PIECES = kEach * ES / 16;
  if (v + kEach <= V) {
    uint4 w[PIECES];
    __builtin_memcpy(w, static_cast<const char*>(base) + (row + v) * ES, sizeof(w));
#pragma unroll
    for (int i = 0; i < PIECES; ++i) unpack16<DT>(w[i], f + i * (kEach / PIECES));
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) f[i] = v + i < V ? load_elem(base, row + v + i, DT) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) f[i] = fmaxf(f[i], 0.f);
}
// What is left at one token.
__device__ __forceinline__ double rest_of(float p, float q, double S) { return fmax((double)p - S * (double)q, 0.0); }

// Sum over the workgroup, the same in every thread.
template <int THREADS>
__device__ __forceinline__ double block_sum(double x, double* s_wave) {
  x = wave_prefix(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s_wave[threadIdx.x >> 6] = x;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w) t += s_wave[w];
  return t;
}

// One workgroup a request walks its tree: all waves find the same.  Nodes'
// probabilities are gathered first, all at once.
template <int DT>
__global__ void __launch_bounds__(kWalkThreads) verify_walk_kernel(VerifyParams P) {
  __shared__ double s_wave[kWalkThreads / 64];
  __shared__ float s_p[kVerMaxNodes], s_q[kVerMaxNodes], s_u[kVerMaxNodes];
  __shared__ int s_tok[kVerMaxNodes], s_gone[kVerMaxNodes];
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  const int lo = max(P.cu[b], 0);
  const int n = max(min(min(max(P.cu[b + 1], 0), P.N) - lo, P.max_nodes), 0);
  VerifyEnd* end = P.ends + b;
  int32_t* path = P.path + (int64_t)b * P.max_path;
  if (n == 0) {
    for (int i = threadIdx.x; i < P.max_path; i += kWalkThreads) path[i] = -1;
    if (threadIdx.x == 0) {
      P.n_path[b] = 0;
      end->row = -1;
      end->n_gone = 0;
    }
    return;
  }
  int par[kVerMaxNodes / 64];  // of nodes lane, lane + 64, ..; -1: none
#pragma unroll
  for (int w = 0; w < kVerMaxNodes / 64; ++w) {
    const int i = w * 64 + lane;
    par[w] = -1;
    if (i < n) {
      const int x = P.parents[lo + i];
      par[w] = x >= 0 && x < i ? x : -1;
    }
  }
  for (int i = threadIdx.x; i < n; i += kWalkThreads) {
    const int64_t t = P.tokens[lo + i];
    const int x = P.parents[lo + i];
    const bool there = x >= 0 && x < i && t >= 0 && t < P.V;
    s_tok[i] = there ? (int)t : -1;
    s_u[i] = P.accept[lo + i];
    s_p[i] = there ? prob<DT>(P.p, (lo + x) * P.p_stride + t) : 0.f;
    s_q[i] = there && P.q ? prob<DT>(P.q, (lo + x) * P.q_stride + t) : 1.f;
  }
  __syncthreads();

  // The first child of `node` behind `last`, or n.
  auto next_child = [&](int node, int last) {
#pragma unroll
    for (int w = 0; w < kVerMaxNodes / 64; ++w) {
      uint64_t m = __ballot(par[w] == node);
      const int past = last + 1 - w * 64;  // bits from here on
      m &= past >= 64 ? 0 : past > 0 ? ~0ull << past : ~0ull;
      if (m != 0) return w * 64 + (int)__builtin_ctzll(m);
    }
    return n;
  };

  int node = 0, len = 1, n_gone = 0;
  double S = 0.0, Z = 1.0, Q = 0.0;
  if (threadIdx.x == 0) path[0] = 0;
  int c = P.max_path > 1 ? next_child(0, 0) : n;
  while (c < n) {
    const int t = s_tok[c];
    bool tried = t >= 0, was = false;
    if (tried) {
      for (int i0 = 0; i0 < n_gone; i0 += 64) was |= __ballot(i0 + lane < n_gone && s_gone[i0 + lane] == t) != 0;
      if (P.q == nullptr || !P.replacement) tried = !was && 1.0 - Q > 0.0;
    }
    const double d = P.q != nullptr && !P.replacement ? 1.0 / (1.0 - Q) : 1.0;
    const double r = was ? 0.0 : P.q != nullptr ? rest_of(s_p[c], s_q[c], S) : (double)s_p[c];
    const int after = next_child(node, c);
    if (tried && (double)s_u[c] * (double)s_q[c] * d * Z < r) {
      if (threadIdx.x == 0) path[len] = c;
      node = c;
      ++len;
      n_gone = 0;
      S = 0.0, Z = 1.0, Q = 0.0;
      c = len < P.max_path ? next_child(c, c) : n;
      continue;
    }
    if (tried) {
      __syncthreads();  // the list has been read
      if (!was && threadIdx.x == 0) s_gone[n_gone] = t;
      n_gone += !was;
      __syncthreads();
      if (P.q == nullptr) {
        Z -= (double)s_p[c];
      } else {
        S += Z * d;
        Q += was ? 0.0 : (double)s_q[c];
        if (after < n) {  // what is left counts for the next child
          double sum = 0.0;
          const int64_t pr = (lo + node) * P.p_stride, qr = (lo + node) * P.q_stride;
#pragma unroll 2
          for (int v = threadIdx.x * kEach; v < P.V; v += kWalkThreads * kEach) {
            float p[kEach], q[kEach];
            probs_at<DT>(P.p, pr, v, P.V, p);
            probs_at<DT>(P.q, qr, v, P.V, q);
#pragma unroll
            for (int i = 0; i < kEach; ++i) sum += rest_of(p[i], q[i], S);
          }
          for (int i = threadIdx.x; i < n_gone; i += kWalkThreads)
            sum -= rest_of(prob<DT>(P.p, pr + s_gone[i]), prob<DT>(P.q, qr + s_gone[i]), S);
          Z = block_sum<kWalkThreads>(sum, s_wave);
        }
      }
    }
    c = after;
  }
  for (int i = len + threadIdx.x; i < P.max_path; i += kWalkThreads) path[i] = -1;
  for (int i = threadIdx.x; i < n_gone; i += kWalkThreads) end->gone[i] = s_gone[i];
  if (threadIdx.x == 0) {
    P.n_path[b] = len;
    end->S = S;
    end->row = lo + node;
    end->n_gone = n_gone;
  }
}

// Which of this thread's tokens v0 + kEach t .. were rejected.
__device__ __forceinline__ uint32_t gone_of(const VerifyEnd* end, int n_gone, int v0, uint32_t* s_gone) {
  if (n_gone == 0) return 0;
  if (threadIdx.x < kSlab / 32) s_gone[threadIdx.x] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n_gone; i += kSumThreads) {
    const int x = end->gone[i] - v0;
    if (x >= 0 && x < kSlab) atomicOr(&s_gone[x >> 5], 1u << (x & 31));
  }
  __syncthreads();
  return s_gone[threadIdx.x / 4] >> (threadIdx.x % 4 * kEach) & 0xff;
}

// What is left of this thread's tokens.
template <int DT>
__device__ __forceinline__ void rests(const VerifyParams& P, int row, int v, double S, uint32_t gone, float (&p)[kEach],
                                      double (&r)[kEach]) {
  probs_at<DT>(P.p, row * P.p_stride, v, P.V, p);
  if (S != 0.0) {
    float q[kEach];
    probs_at<DT>(P.q, row * P.q_stride, v, P.V, q);
#pragma unroll
    for (int i = 0; i < kEach; ++i) r[i] = gone >> i & 1 ? 0.0 : rest_of(p[i], q[i], S);
  } else {
#pragma unroll
    for (int i = 0; i < kEach; ++i) r[i] = gone >> i & 1 ? 0.0 : (double)p[i];
  }
}

// Sums of what is left, a slab of tokens a workgroup.
template <int DT>
__global__ void __launch_bounds__(kSumThreads) verify_sum_kernel(VerifyParams P) {
  __shared__ uint32_t s_gone[kSlab / 32];
  __shared__ double s_wave[kSumThreads / 64];
  const int b = blockIdx.y, v0 = blockIdx.x * kSlab;
  const VerifyEnd* end = P.ends + b;
  const int row = end->row, n_gone = end->n_gone;
  if (row < 0) return;
  const uint32_t gone = gone_of(end, n_gone, v0, s_gone);
  float p[kEach];
  double r[kEach], rest = 0.0, all = 0.0;
  rests<DT>(P, row, v0 + threadIdx.x * kEach, end->S, gone, p, r);
#pragma unroll
  for (int i = 0; i < kEach; ++i) rest += r[i], all += (double)p[i];
  rest = block_sum<kSumThreads>(rest, s_wave);
  all = block_sum<kSumThreads>(all, s_wave);
  if (threadIdx.x == 0) P.parts[(int64_t)b * P.slabs + blockIdx.x] = make_double2(rest, all);
}

// Sum over the workgroup's threads before this one.
__device__ __forceinline__ double block_before(double x, double* s_wave) {
  const int wave = threadIdx.x >> 6;
  const double in = wave_prefix(x);
  __syncthreads();
  if ((threadIdx.x & 63) == 63) s_wave[wave] = in;
  __syncthreads();
  double before = __shfl_up(in, 1, 64);
  if ((threadIdx.x & 63) == 0) before = 0.0;
  for (int w = 0; w < wave; ++w) before += s_wave[w];
  return before;
}

// The token: the slab that passes u times the whole sum, then the token in it.
template <int DT>
__global__ void __launch_bounds__(kSumThreads) verify_pick_kernel(VerifyParams P) {
  __shared__ uint32_t s_gone[kSlab / 32];
  __shared__ double s_wave[kSumThreads / 64], s_from;
  __shared__ int s_slab, s_last, s_tok;
  const int b = blockIdx.x, tid = threadIdx.x;
  const VerifyEnd* end = P.ends + b;
  const int row = end->row;
  if (row < 0) {
    if (tid == 0) P.token[b] = -1;
    return;
  }
  // slabs in order, as many a thread as there have to be
  const double2* parts = P.parts + (int64_t)b * P.slabs;
  const int per = (P.slabs + kSumThreads - 1) / kSumThreads;
  const int g0 = min(tid * per, P.slabs), g1 = min(g0 + per, P.slabs);
  if (tid == 0) s_slab = 0x7fffffff, s_last = -1, s_tok = 0x7fffffff;
  double rest = 0.0, all = 0.0;
  for (int g = g0; g < g1; ++g) rest += parts[g].x, all += parts[g].y;
  const double rest_all = block_sum<kSumThreads>(rest, s_wave);
  // where nothing is left (by rounding) the token comes from the target's probabilities
  const bool whole = !(rest_all > 0.0);
  const double T = (double)P.sample[b] * (whole ? block_sum<kSumThreads>(all, s_wave) : rest_all);
  const double start = block_before(whole ? all : rest, s_wave);
  double upto = start;
  for (int g = g0; g < g1; ++g) {
    const double x = whole ? parts[g].y : parts[g].x;
    if (x > 0.0) atomicMax(&s_last, g);
    upto += x;
    if (upto > T) atomicMin(&s_slab, g);
  }
  __syncthreads();
  const int slab = s_slab != 0x7fffffff ? s_slab : max(s_last, 0);
  if (slab >= g0 && slab < g1) {  // one thread: what lies before the slab
    upto = start;
    for (int g = g0; g < slab; ++g) upto += whole ? parts[g].y : parts[g].x;
    s_from = upto;
  }
  const int v0 = slab * kSlab, v = v0 + tid * kEach;
  const uint32_t gone = gone_of(end, whole ? 0 : end->n_gone, v0, s_gone);
  float p[kEach];
  double r[kEach], mine = 0.0;
  rests<DT>(P, row, v, whole ? 0.0 : end->S, gone, p, r);
  int last = -1;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    mine += r[i];
    if (r[i] > 0.0) last = v + i;
  }
  __syncthreads();  // s_from is there, s_last has been read
  if (tid == 0) s_last = -1;
  upto = s_from + block_before(mine, s_wave);
  if (last >= 0) atomicMax(&s_last, last);
  int tok = 0x7fffffff;
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    upto += r[i];
    if (upto > T && r[i] > 0.0) tok = min(tok, v + i);
  }
  if (tok != 0x7fffffff) atomicMin(&s_tok, tok);
  __syncthreads();
  if (tid == 0) P.token[b] = s_tok != 0x7fffffff ? s_tok : max(s_last, 0);
}

int verify_slabs(int V) { return (V + kSlab - 1) / kSlab; }

}  // namespace
}  // namespace halo

using namespace halo;

extern "C" size_t halo_verify_workspace_size(int B, int V) {
  if (B <= 0 || V <= 0) return 0;
  return (size_t)B * sizeof(VerifyEnd) + (size_t)B * verify_slabs(V) * sizeof(double2);
}

extern "C" int halo_verify_tree(const int64_t* tokens, const int32_t* parents, const int32_t* cu_nodes, int B, int N,
                                int max_nodes, int V, int dtype, const void* probs, int64_t probs_stride,
                                const void* draft_probs, int64_t draft_stride, int replacement, const float* accept,
                                const float* sample, int max_path, int32_t* path, int32_t* n_path, int64_t* token,
                                void* workspace, size_t workspace_bytes, void* stream) {
  HALO_CHECK_ARG(cu_nodes && sample && path && n_path && token, "null pointer argument");
  HALO_CHECK_ARG(N >= 0 && (N == 0 || (tokens && parents && probs && accept)), "null pointer argument");
  HALO_CHECK_ARG(dtype == HALO_F32 || dtype == HALO_BF16 || dtype == HALO_F16, "dtype must be bf16, f16 or f32");
  HALO_CHECK_ARG(B > 0 && B <= 65535 && V > 0 && V <= (1 << 24) && max_nodes > 0 && max_nodes <= kVerMaxNodes,
                 "need 1 <= B <= 65535, 1 <= V <= 2^24 and 1 <= max_nodes <= 512");
  HALO_CHECK_ARG(max_path > 0 && max_path <= kVerMaxPath, "need 1 <= max_path <= 64");
  HALO_CHECK_ARG(probs_stride >= 0 && draft_stride >= 0, "negative strides");
  HALO_CHECK_ARG(workspace && reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "workspace missing or not 16-byte aligned");
  if (workspace_bytes < halo_verify_workspace_size(B, V)) {
    set_error("workspace too small");
    return HALO_E_WORKSPACE;
  }
  const int slabs = verify_slabs(V);
  VerifyParams p = {tokens, parents, cu_nodes, B, N, max_nodes, V, probs, probs_stride, draft_probs, draft_stride, replacement,
                    accept, sample, max_path, path, n_path, token, reinterpret_cast<VerifyEnd*>(workspace),
                    reinterpret_cast<double2*>(reinterpret_cast<VerifyEnd*>(workspace) + B), slabs};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define HALO_VERIFY(DTV)                                                                                              \
  do {                                                                                                                \
    hipLaunchKernelGGL((verify_walk_kernel<DTV>), dim3((unsigned)B), dim3(kWalkThreads), 0, st, p);                   \
    hipLaunchKernelGGL((verify_sum_kernel<DTV>), dim3((unsigned)slabs, (unsigned)B), dim3(kSumThreads), 0, st, p);  \
    hipLaunchKernelGGL((verify_pick_kernel<DTV>), dim3((unsigned)B), dim3(kSumThreads), 0, st, p);                    \
  } while (0)
  if (dtype == HALO_F32) HALO_VERIFY(HALO_F32);
  else if (dtype == HALO_BF16) HALO_VERIFY(HALO_BF16);
  else HALO_VERIFY(HALO_F16);
#undef HALO_VERIFY
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
