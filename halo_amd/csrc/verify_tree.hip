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
constexpr int kMaxSlab = 16384;  // tokens of a workgroup of the sums

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
  double* parts;  // (B, slabs, 2): sums of R and of p
  int slabs, slab;
};

// A probability; NaN and what is below 0 count as 0.
template <int DT>
__device__ __forceinline__ double prob(const void* base, int64_t at) {
  return fmax((double)load_elem(base, at, DT), 0.0);
}
// What is left at one token.
__device__ __forceinline__ double rest_of(double p, double q, double S) { return fmax(p - S * q, 0.0); }

template <int THREADS>
__device__ __forceinline__ double block_sum(double x, double* s_wave) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s_wave[threadIdx.x >> 6] = x;
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
  __shared__ double s_p[kVerMaxNodes], s_q[kVerMaxNodes], s_wave[kWalkThreads / 64];
  __shared__ float s_u[kVerMaxNodes];
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
    s_p[i] = there ? prob<DT>(P.p, (lo + x) * P.p_stride + t) : 0.0;
    s_q[i] = there && P.q ? prob<DT>(P.q, (lo + x) * P.q_stride + t) : 1.0;
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
    const double r = was ? 0.0 : P.q != nullptr ? rest_of(s_p[c], s_q[c], S) : s_p[c];
    const int after = next_child(node, c);
    if (tried && (double)s_u[c] * s_q[c] * d * Z < r) {
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
        Z -= s_p[c];
      } else {
        S += Z * d;
        Q += was ? 0.0 : s_q[c];
        if (after < n) {  // what is left counts for the next child
          double sum = 0.0;
          const int64_t pr = (lo + node) * P.p_stride, qr = (lo + node) * P.q_stride;
          for (int v = threadIdx.x; v < P.V; v += kWalkThreads) sum += rest_of(prob<DT>(P.p, pr + v), prob<DT>(P.q, qr + v), S);
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

// Marks the rejected tokens of [v0, v0 + kMaxSlab) in LDS.
__device__ __forceinline__ void mark_gone(const VerifyEnd* end, int n_gone, int v0, uint32_t* s_gone) {
  for (int i = threadIdx.x; i < kMaxSlab / 32; i += kSumThreads) s_gone[i] = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < n_gone; i += kSumThreads) {
    const int x = end->gone[i] - v0;
    if (x >= 0 && x < kMaxSlab) atomicOr(&s_gone[x >> 5], 1u << (x & 31));
  }
  __syncthreads();
}

// Sums of what is left, a slab of tokens a workgroup.
template <int DT>
__global__ void __launch_bounds__(kSumThreads) verify_sum_kernel(VerifyParams P) {
  __shared__ uint32_t s_gone[kMaxSlab / 32];
  __shared__ double s_wave[kSumThreads / 64];
  const int b = blockIdx.y, v0 = blockIdx.x * P.slab, v1 = min(v0 + P.slab, P.V);
  const VerifyEnd* end = P.ends + b;
  const int row = end->row, n_gone = end->n_gone;
  if (row < 0) return;
  const double S = end->S;
  mark_gone(end, n_gone, v0, s_gone);
  const int64_t pr = row * P.p_stride, qr = row * P.q_stride;
  double rest = 0.0, all = 0.0;
  for (int v = v0 + threadIdx.x; v < v1; v += kSumThreads) {
    const double p = prob<DT>(P.p, pr + v), q = S != 0.0 ? prob<DT>(P.q, qr + v) : 0.0;
    const bool gone = s_gone[(v - v0) >> 5] >> ((v - v0) & 31) & 1;
    rest += gone ? 0.0 : rest_of(p, q, S);
    all += p;
  }
  rest = block_sum<kSumThreads>(rest, s_wave);
  all = block_sum<kSumThreads>(all, s_wave);
  if (threadIdx.x == 0) {
    P.parts[2 * ((int64_t)b * P.slabs + blockIdx.x)] = rest;
    P.parts[2 * ((int64_t)b * P.slabs + blockIdx.x) + 1] = all;
  }
}

// Exclusive sums over the workgroup's threads in order.
__device__ __forceinline__ double block_before(double x, double* s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  double in = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const double y = __shfl_up(in, off, 64);
    if (lane >= off) in += y;
  }
  __syncthreads();
  if (lane == 63) s_wave[wave] = in;
  __syncthreads();
  double before = __shfl_up(in, 1, 64);
  if (lane == 0) before = 0.0;
  for (int w = 0; w < wave; ++w) before += s_wave[w];
  return before;
}

// The token: the slab that passes u times the whole sum, then the token in it.
template <int DT>
__global__ void __launch_bounds__(kSumThreads) verify_pick_kernel(VerifyParams P) {
  __shared__ uint32_t s_gone[kMaxSlab / 32];
  __shared__ double s_wave[kSumThreads / 64], s_from;
  __shared__ int s_slab, s_last, s_tok;
  const int b = blockIdx.x, tid = threadIdx.x;
  const VerifyEnd* end = P.ends + b;
  const int row = end->row;
  if (row < 0) {
    if (tid == 0) P.token[b] = -1;
    return;
  }
  const double* parts = P.parts + 2 * (int64_t)b * P.slabs;
  if (tid == 0) s_slab = 0x7fffffff, s_last = -1, s_tok = 0x7fffffff;
  double rest = 0.0, all = 0.0;
  for (int g = tid; g < P.slabs; g += kSumThreads) rest += parts[2 * g], all += parts[2 * g + 1];
  rest = block_sum<kSumThreads>(rest, s_wave);
  all = block_sum<kSumThreads>(all, s_wave);
  // where nothing is left (by rounding) the token comes from the target's probabilities
  const bool whole = !(rest > 0.0);
  const int n_gone = whole ? 0 : end->n_gone;
  const double S = whole ? 0.0 : end->S;
  const double T = (double)P.sample[b] * (whole ? all : rest);
  // slabs in order, as many a thread as there have to be
  const int per = (P.slabs + kSumThreads - 1) / kSumThreads;
  const int g0 = min(tid * per, P.slabs), g1 = min(g0 + per, P.slabs);
  double mine = 0.0;
  for (int g = g0; g < g1; ++g) mine += parts[2 * g + whole];
  double before = block_before(mine, s_wave);
  for (int g = g0; g < g1; ++g) {
    const double x = parts[2 * g + whole];
    if (x > 0.0) atomicMax(&s_last, g);
    if (before + x > T) atomicMin(&s_slab, g);
    before += x;
  }
  __syncthreads();
  const int slab = s_slab != 0x7fffffff ? s_slab : max(s_last, 0);
  // sum before the slab
  mine = 0.0;
  for (int g = tid; g < slab; g += kSumThreads) mine += parts[2 * g + whole];
  const double from = block_sum<kSumThreads>(mine, s_wave);
  const int v0 = slab * P.slab, v1 = min(v0 + P.slab, P.V);
  mark_gone(end, n_gone, v0, s_gone);
  if (tid == 0) s_last = -1;
  __syncthreads();
  const int64_t pr = row * P.p_stride, qr = row * P.q_stride;
  const int each = (v1 - v0 + kSumThreads - 1) / kSumThreads;
  const int a = min(v0 + tid * each, v1), z = min(a + each, v1);
  auto left = [&](int v) {
    const double p = prob<DT>(P.p, pr + v), q = S != 0.0 ? prob<DT>(P.q, qr + v) : 0.0;
    return s_gone[(v - v0) >> 5] >> ((v - v0) & 31) & 1 ? 0.0 : rest_of(p, q, S);
  };
  mine = 0.0;
  int last = -1;
  for (int v = a; v < z; ++v) {
    const double x = left(v);
    mine += x;
    if (x > 0.0) last = v;
  }
  double upto = from + block_before(mine, s_wave);
  if (last >= 0) atomicMax(&s_last, last);
  if (upto + mine > T) {
    for (int v = a; v < z; ++v) {
      upto += left(v);
      if (upto > T) {
        atomicMin(&s_tok, v);
        break;
      }
    }
  }
  __syncthreads();
  if (tid == 0) P.token[b] = s_tok != 0x7fffffff ? s_tok : max(s_last, 0);
}

// Slabs: enough workgroups for the GPU, at least 2048 tokens each.
struct VerifyShape {
  int slabs, slab;
};
VerifyShape verify_shape(int B, int V) {
  int64_t want = 512 / B < 1 ? 1 : 512 / B;
  const int64_t most = (V + 2047) / 2048, least = (V + kMaxSlab - 1) / kMaxSlab;
  want = want > most ? most : want < least ? least : want;
  VerifyShape s;
  s.slab = (int)((V + want - 1) / want + 7) / 8 * 8;
  if (s.slab > kMaxSlab) s.slab = kMaxSlab;
  s.slabs = (V + s.slab - 1) / s.slab;
  return s;
}

}  // namespace
}  // namespace halo

using namespace halo;

extern "C" size_t halo_verify_workspace_size(int B, int V) {
  if (B <= 0 || V <= 0) return 0;
  return (size_t)B * sizeof(VerifyEnd) + (size_t)B * verify_shape(B, V).slabs * 16;
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
  const VerifyShape s = verify_shape(B, V);
  VerifyParams p = {tokens, parents, cu_nodes, B, N, max_nodes, V, probs, probs_stride, draft_probs, draft_stride, replacement,
                    accept, sample, max_path, path, n_path, token, reinterpret_cast<VerifyEnd*>(workspace),
                    reinterpret_cast<double*>(reinterpret_cast<VerifyEnd*>(workspace) + B), s.slabs, s.slab};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define HALO_VERIFY(DTV)                                                                                              \
  do {                                                                                                                \
    hipLaunchKernelGGL((verify_walk_kernel<DTV>), dim3((unsigned)B), dim3(kWalkThreads), 0, st, p);                   \
    hipLaunchKernelGGL((verify_sum_kernel<DTV>), dim3((unsigned)s.slabs, (unsigned)B), dim3(kSumThreads), 0, st, p);  \
    hipLaunchKernelGGL((verify_pick_kernel<DTV>), dim3((unsigned)B), dim3(kSumThreads), 0, st, p);                    \
  } while (0)
  if (dtype == HALO_F32) HALO_VERIFY(HALO_F32);
  else if (dtype == HALO_BF16) HALO_VERIFY(HALO_BF16);
  else HALO_VERIFY(HALO_F16);
#undef HALO_VERIFY
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
