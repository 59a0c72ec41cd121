// Rows on their way into a paged cache (gfx950, wave64): heads of queries and
// keys normed and rotated, keys and values written to their slots of the pool.
//
//   y = x w / sqrt(mean(x^2) + eps)                       (with a weight w, else y = x)
//   (y_i, y_j) -> (y_i c - y_j s, y_j c + y_i s)          c, s: cosine and sine of the row's position and the pair
// for the pairs (i, i + R/2), or (2i, 2i + 1), of a head's first R channels;
// all of it in fp32, rounded once.  The model library rounds after the norm and
// after the rotation; here the row is read and written once.  The reference
// leaves both to the model and attends what it is handed.
//
// A head's D channels are D / 16 lanes of two 8-channel pieces.  For the pairs
// (i, i + R/2) the pieces of a lane are R/2 channels apart, so both of a pair
// are in one lane, and its cosines and sines are 8 floats in a row either way.
#include <type_traits>

#include "block_pool.hpp"

namespace halo {
namespace {

struct RotateParams {
  PoolView pool;
  const char* q;
  const char* k;
  const char* v;
  char* out;
  int64_t qsn, qsh, ksn, ksh, vsn, vsh, osn, osh;  // strides in bytes
  int H, H_kv, N, parts;
  Div per_row;  // parts
  const void* positions;
  int pos64;
  const float* cos;
  const float* sin;
  int64_t trig_stride;
  int64_t trig_rows;
  int R, interleaved;
  const void* q_norm;
  const void* k_norm;
  int q_norm_f32, k_norm_f32;
  float eps;
  const int64_t* slots;
};

constexpr int kRotThreads = 256;

typedef __attribute__((ext_vector_type(4))) uint32_t u32x4;

template <int DT>
__device__ __forceinline__ void store8(char* p, const float* f) {
  if constexpr (DT == HALO_F32) {
    store_elem4(p, 0, DT, f);
    store_elem4(p, 4, DT, f + 4);
  } else {
    typedef std::conditional_t<DT == HALO_BF16, __bf16, _Float16> T;
    typedef __attribute__((ext_vector_type(2))) T T2;
    auto two = [](float x, float y) { return __builtin_bit_cast(uint32_t, T2{(T)x, (T)y}); };  // to nearest even
    *reinterpret_cast<uint4*>(p) = make_uint4(two(f[0], f[1]), two(f[2], f[3]), two(f[4], f[5]), two(f[6], f[7]));
  }
}

// Sum over the G = 4 or 8 lanes of a head.
template <int G>
__device__ __forceinline__ float head_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, false));  // lane ^ 1
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, false));  // lane ^ 2
  if (G == 8) v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, false));  // 7 - lane
  return v;
}

// Eight elements of a weight, which may begin anywhere.
template <int DT>
__device__ __forceinline__ void weights8(const void* at, bool f32, int i, float* w) {
  if (f32) {
    __builtin_memcpy(w, reinterpret_cast<const float*>(at) + i, 32);
  } else if constexpr (DT != HALO_F32) {
    uint4 x;
    __builtin_memcpy(&x, reinterpret_cast<const uint16_t*>(at) + i, 16);
    unpack16<DT>(x, w);
  }
}

// A group of lanes takes UB heads of a row, `parts` apart, whose loads are in
// flight together; position, cosines and sines are loaded once for them.  Bound
// by memory: 32768 rows of 32 + 8 + 8 heads of 128 in bf16, normed, 822 MB: 170
// to 176 us by the card (4.7 to 4.8 TB/s; a plain copy reaches 5.1).  One head a
// group 263, two 198, four 179; a wave for a whole row 261 to 291, for its
// reads and writes lie far apart.  Few heads are bound by the chain position ->
// cosines -> store, which one head a group has shortest: 768 heads 5.0 us with one
// and 6.3 with three, 12288 heads 6.2 and 6.8, 49152 heads 11.6 and 9.2.
// PART: R < D, and channels behind R stay as they are (with c = 1 and s = 0 an infinity
// among them would make a neighbour NaN); where all turn that test cost 2 us of 171.
constexpr int64_t kRotFew = 16384;
template <int DT, int D, int UB, bool PART>
__global__ void __launch_bounds__(kRotThreads) rotate_rows_kernel(RotateParams P) {
  constexpr int G = D / 16;  // lanes of a head
  constexpr int ES = DT == HALO_F32 ? 4 : 2, PIECES = ES / 2;
  const int unit = blockIdx.x * (kRotThreads / G) + threadIdx.x / G;
  const int n = div_by(unit, P.per_row);
  if (n >= P.N) return;
  const int part = unit - n * P.parts, lane = threadIdx.x & (G - 1);
  const int R = P.R, heads = P.H + 2 * P.H_kv;
  const bool turns = !PART || 16 * lane < R, halves = turns && !P.interleaved;
  const int ca = halves ? 8 * lane : 16 * lane, cb = halves ? R / 2 + 8 * lane : 16 * lane + 8;
  u32x4 w[UB][2 * PIECES];
#pragma unroll
  for (int u = 0; u < UB; ++u) {
    const int h = part + u * P.parts;
    if (h >= heads) break;
    const bool is_q = h < P.H, is_v = h >= P.H + P.H_kv;
    const int hk = h - P.H - (is_v ? P.H_kv : 0);
    const char* src = is_q ? P.q + n * P.qsn + h * P.qsh : is_v ? P.v + n * P.vsn + hk * P.vsh : P.k + n * P.ksn + hk * P.ksh;
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      w[u][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + ca * ES) + i);
      w[u][PIECES + i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + cb * ES) + i);
    }
  }
  const int64_t slot = P.slots[n];
  const bool kept = slot >= 0 && slot < (int64_t)P.pool.blocks * P.pool.bs.d;
  const int blk = kept ? div_by((int)slot, P.pool.bs) : 0;
  const int64_t place = blk * P.pool.sb + (slot - (int64_t)blk * P.pool.bs.d) * P.pool.sr;
  int64_t pos = P.pos64 ? reinterpret_cast<const int64_t*>(P.positions)[n] : reinterpret_cast<const int32_t*>(P.positions)[n];
  const bool there = pos >= 0 && pos < P.trig_rows;
  pos = there ? pos : 0;
  float c[8] = {}, s[8] = {};
  if (turns) {
    const float* cr = P.cos + pos * P.trig_stride + 8 * lane;
    const float* sr = P.sin + pos * P.trig_stride + 8 * lane;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      c[i] = there ? cr[i] : __uint_as_float(0x7fc00000u);
      s[i] = sr[i];
    }
  }
#pragma unroll
  for (int u = 0; u < UB; ++u) {
    const int h = part + u * P.parts;
    const bool is_q = h < P.H, is_v = h >= P.H + P.H_kv;
    const int hk = h - P.H - (is_v ? P.H_kv : 0);
    if (h >= heads || !(is_q || kept)) break;
    char* dst = is_q ? P.out + n * P.osn + h * P.osh : (is_v ? P.pool.v : P.pool.k) + place + hk * P.pool.sh;
    if (is_v) {
#pragma unroll
      for (int i = 0; i < PIECES; ++i) {
        *(reinterpret_cast<u32x4*>(dst + ca * ES) + i) = w[u][i];
        *(reinterpret_cast<u32x4*>(dst + cb * ES) + i) = w[u][PIECES + i];
      }
      continue;
    }
    float a[8], b[8];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      unpack16<DT>(__builtin_bit_cast(uint4, w[u][i]), a + i * (8 / PIECES));
      unpack16<DT>(__builtin_bit_cast(uint4, w[u][PIECES + i]), b + i * (8 / PIECES));
    }
    const void* norm = is_q ? P.q_norm : P.k_norm;
    if (norm != nullptr) {
      const bool f32 = DT == HALO_F32 || (is_q ? P.q_norm_f32 : P.k_norm_f32);
      float wa[8], wb[8], sum = 0.f;
      weights8<DT>(norm, f32, ca, wa);
      weights8<DT>(norm, f32, cb, wb);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = __builtin_fmaf(a[i], a[i], __builtin_fmaf(b[i], b[i], sum));
      const float inv = 1.f / sqrtf(head_sum<G>(sum) * (1.f / D) + P.eps);
#pragma unroll
      for (int i = 0; i < 8; ++i) a[i] = a[i] * inv * wa[i], b[i] = b[i] * inv * wb[i];
    }
    if (PART && !turns) {
    } else if (P.interleaved) {
#pragma unroll
      for (int i = 0; i < 8; i += 2) {
        const float a0 = a[i], a1 = a[i + 1], b0 = b[i], b1 = b[i + 1];
        a[i] = a0 * c[i / 2] - a1 * s[i / 2];
        a[i + 1] = a1 * c[i / 2] + a0 * s[i / 2];
        b[i] = b0 * c[4 + i / 2] - b1 * s[4 + i / 2];
        b[i + 1] = b1 * c[4 + i / 2] + b0 * s[4 + i / 2];
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float x = a[i], y = b[i];
        a[i] = x * c[i] - y * s[i];
        b[i] = y * c[i] + x * s[i];
      }
    }
    store8<DT>(dst + ca * ES, a);
    store8<DT>(dst + cb * ES, b);
  }
}

}  // namespace
}  // namespace halo

using namespace halo;

extern "C" int halo_rotate_rows(const halo_block_pool* pool, const void* q, int64_t q_stride_n, int64_t q_stride_h, int H,
                                const void* k, int64_t k_stride_n, int64_t k_stride_h, const void* v,
                                int64_t v_stride_n, int64_t v_stride_h, void* out, int64_t out_stride_n,
                                int64_t out_stride_h, int N, const void* positions, int pos64, const float* cos,
                                const float* sin, int64_t trig_stride, int64_t trig_rows, int R, int interleaved,
                                const void* q_norm, int q_norm_f32, const void* k_norm, int k_norm_f32, float eps,
                                const int64_t* slots, void* stream) {
  RotateParams p;
  const int rc = check_pool(pool, &p.pool);
  if (rc != HALO_OK) return rc;
  HALO_CHECK_ARG(pool->layers == 1, "need a pool of one layer");
  HALO_CHECK_ARG(pool->D == 64 || pool->D == 128, "head_dim must be 64 or 128");
  HALO_CHECK_ARG(R > 0 && R <= pool->D && R % 16 == 0, "need 16 <= R <= D in steps of 16");
  HALO_CHECK_ARG(N >= 0 && H > 0, "bad sizes");
  HALO_CHECK_ARG(eps >= 0.f && std::isfinite(eps), "eps must be finite and not negative");
  if (N == 0) return HALO_OK;
  HALO_CHECK_ARG(q && k && v && out && positions && cos && sin && slots, "null pointer argument");
  HALO_CHECK_ARG(trig_rows > 0 && trig_stride >= R / 2 && trig_stride % 4 == 0 &&
                     (reinterpret_cast<uintptr_t>(cos) | reinterpret_cast<uintptr_t>(sin)) % 16 == 0,
                 "rows of cosines and sines must be 16-byte aligned and not overlap");
  const int64_t es = elem_size(pool->dtype);
  HALO_CHECK_ARG(piece_bytes(p.pool, 0) == 16, "pool rows must be 16-byte aligned");
  p.q = static_cast<const char*>(q);
  p.k = static_cast<const char*>(k);
  p.v = static_cast<const char*>(v);
  p.out = static_cast<char*>(out);
  p.qsn = q_stride_n * es, p.qsh = q_stride_h * es, p.ksn = k_stride_n * es, p.ksh = k_stride_h * es;
  p.vsn = v_stride_n * es, p.vsh = v_stride_h * es, p.osn = out_stride_n * es, p.osh = out_stride_h * es;
  HALO_CHECK_ARG((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v) |
                  reinterpret_cast<uintptr_t>(out) | (uint64_t)(p.qsn | p.qsh | p.ksn | p.ksh | p.vsn | p.vsh | p.osn | p.osh)) %
                         16 == 0,
                 "rows must be 16-byte aligned");
  const int64_t heads = (int64_t)H + 2 * (int64_t)pool->H_kv;
  HALO_CHECK_ARG(heads * N < (1ll << 31) - kRotThreads, "heads of all rows in 31 bits");
  p.H = H;
  p.H_kv = pool->H_kv;
  p.N = N;
  p.positions = positions;
  p.pos64 = pos64;
  p.cos = cos;
  p.sin = sin;
  p.trig_stride = trig_stride;
  p.trig_rows = trig_rows;
  p.R = R;
  p.interleaved = interleaved;
  p.q_norm = q_norm;
  p.k_norm = k_norm;
  p.q_norm_f32 = q_norm_f32;
  p.k_norm_f32 = k_norm_f32;
  p.eps = eps;
  p.slots = slots;
  const int ub = heads * N < kRotFew ? 1 : 3;
  p.parts = (int)((heads + ub - 1) / ub);
  p.per_row = make_div(p.parts);
  const int per = kRotThreads / (pool->D / 16);
  const dim3 grid((unsigned)(((int64_t)p.parts * N + per - 1) / per)), block(kRotThreads);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
#define HALO_ROTATE_PART(DTV, DV, UBV)                                                                                 \
  do {                                                                                                                 \
    if (R < DV) hipLaunchKernelGGL((rotate_rows_kernel<DTV, DV, UBV, true>), grid, block, 0, st, p);                   \
    else hipLaunchKernelGGL((rotate_rows_kernel<DTV, DV, UBV, false>), grid, block, 0, st, p);                         \
  } while (0)
#define HALO_ROTATE(DTV)                                                                                               \
  do {                                                                                                                 \
    if (pool->D == 128 && ub == 3) HALO_ROTATE_PART(DTV, 128, 3);                                                      \
    else if (pool->D == 128) HALO_ROTATE_PART(DTV, 128, 1);                                                            \
    else if (ub == 3) HALO_ROTATE_PART(DTV, 64, 3);                                                                    \
    else HALO_ROTATE_PART(DTV, 64, 1);                                                                                 \
  } while (0)
  if (pool->dtype == HALO_F32) HALO_ROTATE(HALO_F32);
  else if (pool->dtype == HALO_BF16) HALO_ROTATE(HALO_BF16);
  else HALO_ROTATE(HALO_F16);
#undef HALO_ROTATE
#undef HALO_ROTATE_PART
  HALO_CHECK_HIP(hipGetLastError());
  return HALO_OK;
}
