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
// and without draft probabilities R is p without the rejected tokens, and Z_j is
// 1 less their p: no pass over the row, whose sum differs only by what the rounded
// p lack of 1.  Where no child is accepted the next token is the first v whose
// R(0) + .. + R(v) exceeds u sum R.  Sums and products are in 64 bits: a sum of 100 000 terms in
// 32 would move the borders between tokens.
//
// The reference drafts no tokens; this is the library's own.
#include "block_pool.hpp"

namespace halo {
namespace {

constexpr int kVerMaxNodes = 512, kVerMaxPath = 64;
constexpr int kVerThreads = 1024, kVerWaves = kVerThreads / 64;
constexpr int kEach = 8;                    // tokens of a thread in the last scan
constexpr int kStep = 64 * kEach;           // waves' ranges are multiples of this
constexpr int kTurn = kVerThreads * kEach;  // tokens that the last scan takes
constexpr int kMarks = 16384;               // bits that mark groups of kEach tokens, one of which may be rejected

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
};

// A probability; NaN and what is below 0 count as 0.
__device__ __forceinline__ float clean(float x) { return x > 0.f ? x : 0.f; }
// What is left at one token.
__device__ __forceinline__ double rest_of(float p, float q, double S) { return fmax(__builtin_fma(-S, (double)q, (double)p), 0.0); }

// The tokens of a 16-byte piece.  Rows begin at any element: the loads need no alignment.
template <int DT>
struct Piece16 {
  static constexpr int ES = DT == HALO_F32 ? 4 : 2, N = 16 / ES;
  uint4 w;
  __device__ __forceinline__ void load(const void* base, int64_t at) {
    __builtin_memcpy(&w, static_cast<const char*>(base) + at * ES, 16);
  }
  __device__ __forceinline__ void get(float* f) const { unpack16<DT>(w, f); }
};

// A workgroup's view of the row that its request's walk has reached: what is
// left of it goes by S and the rejected tokens (list and marks in LDS).
// The kernel's code is short on purpose: each line of it runs a few times, and
// with every loop unrolled for itself (70 KB) half of the time was instruction fetch.
template <int DT>
struct VerifyRow {
  const void* p;
  const void* q;  // null where S is 0 for good
  int64_t pr, qr;  // first elements
  int V, n_gone;
  double S;
  bool masked;  // without a draft: rejected tokens are left out one by one, found by their marks
  const int* gone;
  const uint32_t* marks;

  static constexpr int EP = Piece16<DT>::N;

  // What is left of the tokens v .. v + N - 1, the rejected ones included.
  template <int N>
  __device__ __forceinline__ void rests(const float (&x)[N], const float (&y)[N], double (&r)[N]) const {
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = rest_of(x[i], clean(y[i]), S);
  }
  // Without those of the tokens v .. that were rejected.
  template <int N>
  __device__ __forceinline__ void leave_out(int v, double (&r)[N]) const {
#pragma unroll 1
    for (int k = 0; k < n_gone; ++k) {
      const int x0 = gone[k] - v;
#pragma unroll
      for (int i = 0; i < N; ++i) r[i] = x0 == i ? 0.0 : r[i];
    }
  }
  __device__ __forceinline__ bool marked(int v) const {
    const int g = v / kEach % kMarks;
    return marks[g >> 5] >> (g & 31) & 1;
  }
  template <int N>
  __device__ static __forceinline__ double sum_of(const double (&r)[N]) {
    const double t = (r[0] + r[1]) + (r[2] + r[3]);
    if constexpr (N == 8) return t + ((r[4] + r[5]) + (r[6] + r[7]));
    else return t;
  }
  // The same for kEach tokens from v on, 0 from V on.
  __device__ __forceinline__ void rests_at(int v, double (&r)[kEach]) const {
    float x[kEach], y[kEach];
    if (v + kEach <= V) {
#pragma unroll
      for (int i = 0; i < kEach; i += EP) {
        Piece16<DT> a, b = {};
        a.load(p, pr + v + i);
        if (S != 0.0) b.load(q, qr + v + i);
        a.get(x + i);
        b.get(y + i);
      }
    } else {
#pragma unroll
      for (int i = 0; i < kEach; ++i) {
        x[i] = v + i < V ? load_elem(p, pr + v + i, DT) : 0.f;
        y[i] = S != 0.0 && v + i < V ? load_elem(q, qr + v + i, DT) : 0.f;
      }
    }
    rests(x, y, r);
    leave_out(v, r);
  }
  // This lane's part of the sum over [v0, v1), a wave's range (v0 a multiple of
  // kStep).  A load of the wave is 1 KiB side by side, and those of BATCH pieces
  // of p and of q are in flight together.
  __device__ __forceinline__ double part(int v0, int v1) const {
    constexpr int BATCH = 32 / EP, STEP = 64 * EP;
    double sum = 0.0, r[EP];
    const int full = min(v1, V) - EP;  // the last place of a whole piece
    const bool two = S != 0.0;
#pragma unroll 1
    for (int v = v0 + (threadIdx.x & 63) * EP; v <= full; v += BATCH * STEP) {
      Piece16<DT> x[BATCH], y[BATCH];
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        const int at = min(v + k * STEP, full);  // (what is read twice is left out below)
        x[k].load(p, pr + at);
        if (two) y[k].load(q, qr + at);
        else y[k] = {};
      }
#pragma unroll
      for (int k = 0; k < BATCH; ++k) {
        float f[EP], g[EP];
        x[k].get(f);
        y[k].get(g);
        rests(f, g, r);
        if (masked && marked(v + k * STEP)) leave_out(v + k * STEP, r);
        sum += v + k * STEP <= full ? sum_of(r) : 0.0;
      }
    }
    // the one piece that the row's end cuts
    const int cut = V / EP * EP;
    if (cut < V && cut >= v0 && cut < v1 && (threadIdx.x & 63) == 0) {
#pragma unroll 1
      for (int v = cut; v < V; ++v) {
        double one = rest_of(load_elem(p, pr + v, DT), two ? clean(load_elem(q, qr + v, DT)) : 0.f, S);
#pragma unroll 1
        for (int k = 0; masked && k < n_gone; ++k) one = gone[k] == v ? 0.0 : one;
        sum += one;
      }
    }
    // Against a draft a rejected token has p - S q < 0 but for rounding: what is above 0 of it is taken back.
    if (!masked && n_gone > 0) {
#pragma unroll 1
      for (int k = threadIdx.x & 63; k < n_gone; k += 64) {
        const int v = gone[k];
        if (v >= v0 && v < v1) sum -= rest_of(load_elem(p, pr + v, DT), two ? clean(load_elem(q, qr + v, DT)) : 0.f, S);
      }
    }
    return sum;
  }
};

// Tokens of each wave's range where the workgroup shares n of them: whole steps.
__device__ __forceinline__ int range_of(int n) { return ((n + kVerWaves - 1) / kVerWaves + kStep - 1) / kStep * kStep; }

struct VerifyNode {
  float p, q, u;
  int tok;  // -1: not tried
};

// One workgroup a request.  All its waves walk the tree alike: the nodes'
// probabilities are gathered first, all at once, and a pass over the vocabulary
// is made only where a rejected child has a sibling behind it (Z), and once for
// the last token.  A pass gives each wave a range of tokens, so the range that
// holds the token is found from 16 sums, and the token in it by one scan.
//
// Bound by chains: gather 0.8 us, walk 2 to 3, a pass, 2 to 3 for the last token;
// and a pass by what one CU reads, 85 to 150 GB/s.  One request of 32768 bf16
// tokens without draft probabilities 9.8 us; 48 chains over 131072 fp32 tokens,
// 38 MB, 22 us (a pass of 1 MB 12, when 4.9 TB/s come from memory in all); 13 trees
// over 50001 with up to 4 siblings 34 us (up to 5 passes of 4.5).  Spreading the
// last sums over the GPU, with two more launches, took 16.4, 32 and 37 us.
template <int DT>
__global__ void __launch_bounds__(kVerThreads) verify_tree_kernel(VerifyParams P) {
  __shared__ double s_sum[kVerWaves];
  __shared__ VerifyNode s_node[kVerMaxNodes];
  __shared__ int s_gone[kVerMaxNodes], s_last, s_found;
  __shared__ uint32_t s_marks[kMarks / 32];
  constexpr int WORDS = kVerMaxNodes / 64;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int lo = max(P.cu[b], 0);
  const int n = max(min(min(max(P.cu[b + 1], 0), P.N) - lo, P.max_nodes), 0);
  int32_t* path = P.path + (int64_t)b * P.max_path;
  const float u_last = P.sample[b];
  int par[WORDS], tok[WORDS];  // of nodes lane, lane + 64, ..; -1: none
#pragma unroll
  for (int w = 0; w < WORDS; ++w) {
    const int i = w * 64 + lane;
    par[w] = tok[w] = -1;
    if (w * 64 < n && i < n) {
      const int64_t t = P.tokens[lo + i];
      const int x = P.parents[lo + i];
      par[w] = x >= 0 && x < i ? x : -1;
      tok[w] = t >= 0 && t < P.V ? (int)t : -1;
      if ((w & (kVerWaves - 1)) == wave) {  // one wave looks the node's probabilities up
        VerifyNode y = {0.f, 1.f, P.accept[lo + i], tok[w]};
        if (par[w] >= 0 && t >= 0 && t < P.V) {
          y.p = clean(load_elem(P.p, (lo + x) * P.p_stride + t, DT));
          if (P.q != nullptr) y.q = clean(load_elem(P.q, (lo + x) * P.q_stride + t, DT));
        }
        s_node[i] = y;
      }
    }
  }
  __syncthreads();

  // The first child of `node` behind `last`, or n.
  auto next_child = [&](int node, int last) {
    int c = n;
#pragma unroll
    for (int w = WORDS - 1; w >= 0; --w) {
      if (w * 64 >= n) continue;
      uint64_t m = __ballot(par[w] == node);
      const int past = last + 1 - w * 64;  // bits from here on
      m &= past >= 64 ? 0 : past > 0 ? ~0ull << past : ~0ull;
      if (m != 0) c = w * 64 + (int)__builtin_ctzll(m);
    }
    return c;
  };
  VerifyRow<DT> R = {P.p, P.q, 0, 0, P.V, 0, 0.0, false, s_gone, s_marks};
  uint32_t gone = 0;  // bit w: node w * 64 + lane was rejected at the node reached
  int node = 0, len = 1, v0 = 0, v1 = P.V;
  double Z = 1.0, Q = 0.0, T = 0.0, from = 0.0;
  if (tid == 0 && n > 0) path[0] = 0;
  int c = n > 0 && P.max_path > 1 ? next_child(0, 0) : n;
  enum { kWalk, kLast, kWhole, kNarrow } mode = kWalk;
  for (;;) {
    if (mode == kWalk) {
      bool left = false;  // whether what is left has to be summed for the next child
#pragma unroll 1
      while (c < n && !left) {
        const VerifyNode y = s_node[c];
        uint64_t same = 0;
#pragma unroll
        for (int w = 0; w < WORDS; ++w)
          if (w * 64 < n) same |= __ballot((gone >> w & 1) && tok[w] == y.tok);
        const bool was = same != 0;
        const double rest = 1.0 - Q;  // 1 with replacement
        const bool tried = y.tok >= 0 && ((P.q != nullptr && P.replacement) || (!was && rest > 0.0));
        const double r = was ? 0.0 : rest_of(y.p, y.q, P.q != nullptr ? R.S : 0.0);
        // u q Z / rest < r, multiplied by rest: one division less on the way
        if (tried && (double)y.u * (double)y.q * Z < r * rest) {
          if (tid == 0) path[len] = c;
          node = c;
          ++len;
          gone = 0;
          R.S = 0.0, Z = 1.0, Q = 0.0;
          c = len < P.max_path ? next_child(c, c) : n;
          continue;
        }
        const int after = next_child(node, c);
        if (tried) {
          if (!was && (c & 63) == lane) gone |= 1u << (c >> 6);
          if (P.q == nullptr) {
            Z -= (double)y.p;
          } else {
            R.S += Z / rest;
            if (!P.replacement) Q += (double)y.q;
            left = after < n;
          }
        }
        c = after;
      }
      if (!left) mode = kLast;
      R.pr = (lo + node) * P.p_stride;
      R.qr = (lo + node) * P.q_stride;
      if (n == 0) break;
    }
    if (mode <= kLast) {  // the rejected tokens, listed and marked
      R.n_gone = 0;
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        if (w * 64 >= n) continue;
        const uint64_t m = __ballot(gone >> w & 1);
        if (wave == 0 && (gone >> w & 1)) s_gone[R.n_gone + __popcll(m & ((1ull << lane) - 1))] = tok[w];
        R.n_gone += __popcll(m);
      }
      R.masked = R.n_gone > 0 && P.q == nullptr;
      if (!R.masked) {
        if (R.n_gone > 0) __syncthreads();
      } else {
        if (tid < kMarks / 32) s_marks[tid] = 0;
        __syncthreads();
        for (int i = tid; i < R.n_gone; i += kVerThreads) {
          const int g = s_gone[i] / kEach % kMarks;
          atomicOr(&s_marks[g >> 5], 1u << (g & 31));
        }
        __syncthreads();
      }
    }
    const int each = range_of(v1 - v0);
    {
      const int a = v0 + wave * each, z = min(a + each, v1);
      double x = R.part(a, z);
      x = wave_prefix(x);
      __syncthreads();  // sums of an earlier pass have been read
      if (lane == 63) s_sum[wave] = x;
      __syncthreads();
    }
    const double mine = lane < kVerWaves ? s_sum[lane] : 0.0, upto = wave_prefix(mine), total = lane_of(upto, 63);
    if (mode == kWalk) {
      Z = total;
      continue;
    }
    if (mode == kLast && !(total > 0.0)) {  // nothing is left (by rounding): the token comes from the target's probabilities
      R.S = 0.0;
      R.n_gone = 0;
      R.masked = false;
      mode = kWhole;
      continue;
    }
    if (mode != kNarrow) T = (double)u_last * total;
    mode = kNarrow;
    // to the range that passes T; the last one with anything if rounding lets none pass
    const uint64_t passed = __ballot(mine > 0.0 && from + upto > T), some = __ballot(mine > 0.0);
    if (passed == 0) T = INFINITY;
    const int w = passed != 0 ? (int)__builtin_ctzll(passed) : some != 0 ? 63 - (int)__builtin_clzll(some) : 0;
    if (w > 0) from += lane_of(upto, w - 1);
    v0 += w * each;
    v1 = min(v0 + each, v1);
    if (each <= kTurn) break;
  }
  for (int i = (n > 0 ? len : 0) + tid; i < P.max_path; i += kVerThreads) path[i] = -1;
  if (n == 0) {
    if (tid == 0) {
      P.n_path[b] = 0;
      P.token[b] = -1;
    }
    return;
  }

  // the range's tokens, kEach a thread, in order
  const int v = v0 + tid * kEach;
  double r[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) r[i] = 0.0;
  if (v < v1) R.rests_at(v, r);
  const double mine = R.sum_of(r), in = wave_prefix(mine);
  int last = -1;
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (r[i] > 0.0) last = v + i;
  const uint64_t some = __ballot(last >= 0);
  __syncthreads();
  if (lane == 63) s_sum[wave] = in;
  if (tid == 0) s_last = 0, s_found = 0x7fffffff;
  __syncthreads();
  double upto = from;
#pragma unroll
  for (int w = 0; w < kVerWaves; ++w) upto += w < wave ? s_sum[w] : 0.0;
  upto += in - mine;
  if (some != 0 && lane == 63 - (int)__builtin_clzll(some)) atomicMax(&s_last, last);
  int found = 0x7fffffff;
#pragma unroll
  for (int i = kEach - 1; i >= 0; --i) {
    double at = upto;
#pragma unroll
    for (int k = 0; k <= i; ++k) at += r[k];
    if (at > T && r[i] > 0.0) found = v + i;
  }
  const uint64_t passes = __ballot(found != 0x7fffffff);
  if (passes != 0 && lane == (int)__builtin_ctzll(passes)) atomicMin(&s_found, found);
  __syncthreads();
  if (tid == 0) {
    P.n_path[b] = len;
    P.token[b] = s_found != 0x7fffffff ? s_found : s_last;
  }
}

}  // namespace
}  // namespace halo

using namespace halo;

extern "C" int halo_verify_tree(const int64_t* tokens, const int32_t* parents, const int32_t* cu_nodes, int B, int N,
                                int max_nodes, int V, int dtype, const void* probs, int64_t probs_stride,
                                const void* draft_probs, int64_t draft_stride, int replacement, const float* accept,
                                const float* sample, int max_path, int32_t* path, int32_t* n_path, int64_t* token,
                                void* stream) {
  HALO_CHECK_ARG(cu_nodes && sample && path && n_path && token, "null pointer argument");
  HALO_CHECK_ARG(N >= 0 && (N == 0 || (tokens && parents && probs && accept)), "null pointer argument");
  HALO_CHECK_ARG(dtype == HALO_F32 || dtype == HALO_BF16 || dtype == HALO_F16, "dtype must be bf16, f16 or f32");
  HALO_CHECK_ARG(B > 0 && B <= 65535 && V > 0 && V <= (1 << 24) && max_nodes > 0 && max_nodes <= kVerMaxNodes,
                 "need 1 <= B <= 65535, 1 <= V <= 2^24 and 1 <= max_nodes <= 512");
  HALO_CHECK_ARG(max_path > 0 && max_path <= kVerMaxPath, "need 1 <= max_path <= 64");
  HALO_CHECK_ARG(probs_stride >= 0 && draft_stride >= 0, "negative strides");
  const VerifyParams p = {tokens, parents, cu_nodes, B, N, max_nodes, V, probs, probs_stride, draft_probs, draft_stride,
                          replacement, accept, sample, max_path, path, n_path, token};
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const dim3 grid((unsigned)B), block(kVerThreads);
#define HALO_VERIFY(DTV) hipLaunchKernelGGL((verify_tree_kernel<DTV>), grid, block, 0, st, p)
  if (dtype == HALO_F32) HALO_VERIFY(HALO_F32);
  else if (dtype == HALO_BF16) HALO_VERIFY(HALO_BF16);
  else HALO_VERIFY(HALO_F16);
#undef HALO_VERIFY
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
