// 8-bit integer linear layer: tokens quantised row by row,
//   s_n = max_k |x_nk| / 127, q_nk = rint(x_nk / s_n) (a zero row: s_n = 0, q = 0),
//   y_no = s_n w_o sum_k q_nk W_ok (+ bias_o),
// sums in 32-bit integers (exact up to K = 2^31 / (127 * 128)), scales FP32.  A row that holds an
// infinity or a NaN has the scale NaN and comes out NaN.
#include <hip/hip_runtime.h>

#include "sd_skinny.cuh"
#include "../../include/solvedelta_mixer.h"

namespace sd {

struct EpiScaled : EpiNothing {
  static constexpr bool DOWN = true;
  OutBf o;
  const float *row, *col;
  const __bf16* bias;
  int64_t M, N;
  EpiScaled(OutBf o_, const float* row_, const float* col_, const __bf16* bias_, int64_t M_, int64_t N_)
      : o(o_), row(row_), col(col_), bias(bias_), M(M_), N(N_) {}
  struct Cols {
    float c[16], b[16];
  };
  __device__ __forceinline__ Cols cols(int64_t nb) const {
    Cols k;
    const int64_t n0 = nb + 4 * (lane_id() >> 5);
    if (nb + 32 <= N) {
      typedef float f4u __attribute__((ext_vector_type(4), aligned(4)));
      typedef __bf16 b4u __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f4 c = *reinterpret_cast<const f4u*>(col + n0 + 8 * g);
        b4u b = {};
        if (bias) b = *reinterpret_cast<const b4u*>(bias + n0 + 8 * g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          k.c[4 * g + e] = c[e];
          k.b[4 * g + e] = (float)b[e];
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const int64_t n = n0 + 8 * (e >> 2) + (e & 3);
        k.c[e] = n < N ? col[n] : 0.f;
        k.b[e] = bias && n < N ? bf2f(bias[n]) : 0.f;
      }
    }
    return k;
  }
  __device__ __forceinline__ float pre(int64_t mb, int64_t) const {
    const int64_t m = mb + (lane_id() & 31);
    return m < M ? row[m] : 0.f;
  }
  __device__ __forceinline__ void operator()(int64_t mb, int64_t nb, const Cols& k, float s, const i16v& a) const {
    if (mb >= M || nb >= N) return;
    const int64_t m = mb + (lane_id() & 31);
    float v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) v[e] = __builtin_fmaf((float)a[e] * s, k.c[e], k.b[e]);
    store_block(o, m, m < M, nb, N, v);
  }
};

// A row's scale from its largest magnitude m (NaN if `odd`: not all are finite), and a value
// in 8 bits.
__device__ __forceinline__ float quant_scale(float m, bool odd) { return odd ? __builtin_nanf("") : m / 127.f; }
__device__ __forceinline__ int quant(float x, float s) {
  const float v = s > 0.f ? rintf(x / s) : 0.f;
  return (int)fminf(fmaxf(v, -127.f), 127.f);
}
__device__ __forceinline__ float wave_fmax(float m) {
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  return m;
}

// A wave a row of up to 512 NV values, which stay in its registers: one trip to memory, no
// barrier.  x / s is x r, r = 1 / s, and one correction by the exact remainder, which rounds
// as the division does (Markstein); of scales so small that the remainder would not be exact
// it is the division.  8192 bf16 rows of
// 2048 take 14 us, 24 with a workgroup a row.
template <class E, int NV>
__global__ __launch_bounds__(256) void k_quant_rows(int64_t N, int K, const E* x, int64_t x_st, int8_t* q,
                                                    int64_t q_st, int q_end, float* scale) {
  typedef E e8 __attribute__((ext_vector_type(8)));
  typedef E e8u __attribute__((ext_vector_type(8), aligned(2)));
  const int64_t n = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(wave_id());
  if (n >= N) return;
  const int l = lane_id();
  const E* row = x + n * x_st;
  e8 v[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = i * 512 + l * 8;
    if (k + 8 <= K) {
      v[i] = *reinterpret_cast<const e8u*>(row + k);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[i][e] = k + e < K ? row[k + e] : (E)0.f;
    }
  }
  float m = 0.f;
  bool odd = false;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf((float)v[i][e]);
      odd |= !(a < __builtin_inff());
      m = fmaxf(m, a);
    }
  const float s = quant_scale(wave_fmax(m), __any(odd));
  if (l == 0) scale[n] = s;
  const bool exact = s > 0x1p-100f;
  const float r = exact ? 1.f / s : 0.f;
  const bool vec = ((q_st | (int64_t)(uintptr_t)q) & 7) == 0;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = i * 512 + l * 8;
    unsigned w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = (float)v[i][e], y = a * r;
      const int b = exact ? (int)rintf(__builtin_fmaf(__builtin_fmaf(-y, s, a), r, y)) : quant(a, s);
      w[e >> 2] |= (unsigned)(unsigned char)(int8_t)b << (8 * (e & 3));
    }
    if (vec && k + 8 <= q_end) {
      *reinterpret_cast<i2v*>(q + n * q_st + k) = i2v{(int)w[0], (int)w[1]};
    } else {
      for (int e = 0; e < 8 && k + e < q_end; ++e) q[n * q_st + k + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// Longer rows: a workgroup each, 8 values a thread at a time; columns up to q_end are zeros.
template <class E>
__global__ __launch_bounds__(256) void k_quant(int K, const E* x, int64_t x_st, int8_t* q,
                                               int64_t q_st, int q_end, float* scale) {
  __shared__ float red[4];
  __shared__ int bad[4];
  const int64_t n = blockIdx.x;
  const E* row = x + n * x_st;
  float m = 0.f;
  bool odd = false;
  typedef E e8 __attribute__((ext_vector_type(8)));
  typedef E e8u __attribute__((ext_vector_type(8), aligned(2)));
  for (int k = threadIdx.x * 8; k < K; k += 2048) {
    e8 v;
    if (k + 8 <= K) {
      v = *reinterpret_cast<const e8u*>(row + k);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = k + e < K ? row[k + e] : (E)0.f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float a = fabsf((float)v[e]);
      odd |= !(a < __builtin_inff());
      m = fmaxf(m, a);
    }
  }
  m = wave_fmax(m);
  const bool any = __any(odd);
  if (lane_id() == 0) { red[wave_id()] = m; bad[wave_id()] = any; }
  __syncthreads();
  m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const float s = quant_scale(m, bad[0] | bad[1] | bad[2] | bad[3]);
  if (threadIdx.x == 0) scale[n] = s;
  const bool vec = ((q_st | (int64_t)(uintptr_t)q) & 7) == 0;
  for (int k = threadIdx.x * 8; k < q_end; k += 2048) {
    unsigned w[2] = {0u, 0u};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      w[e >> 2] |= (unsigned)(unsigned char)(int8_t)(k + e < K ? quant((float)row[k + e], s) : 0) << (8 * (e & 3));
    if (vec && k + 8 <= q_end) {
      *reinterpret_cast<i2v*>(q + n * q_st + k) = i2v{(int)w[0], (int)w[1]};
    } else {
      for (int e = 0; e < 8 && k + e < q_end; ++e) q[n * q_st + k + e] = (int8_t)(w[e >> 2] >> (8 * (e & 3)));
    }
  }
}

// y of few tokens
struct SkinnyScaled {
  OutBf o;
  const float *row, *col;
  const __bf16* bias;
  int cols;
  __device__ __forceinline__ void put(int n, int c, const i4v& a, float s) const {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int k = c + e < cols ? c + e : cols - 1;
      v[e] = __builtin_fmaf((float)a[e] * s, col[k], bias ? bf2f(bias[k]) : 0.f);
    }
    store4(o, n, c, cols, v);
  }
  __device__ __forceinline__ void operator()(int n, int c, const i4v& a) const { put(n, c, a, row[n]); }
};

// The product of up to 8 bf16 tokens: every workgroup quantises them for itself, into LDS,
// while its first weights are on their way.  Each wave looks at the whole rows for their
// scales, so that one barrier is enough.
template <int R, int U, bool HALF>
__global__ __launch_bounds__(512) void k_int8_few(SkinnyArgs a, const __bf16* x, int64_t x_st, int K, SkinnyScaled epi) {
  constexpr int WAVES = 8;
  typedef Skinny<int8_t, R, 1, WAVES, U, HALF, true> S;
  extern __shared__ __align__(16) char few_smem[];
  __shared__ __align__(16) i4v red[WAVES][R][64];
  __shared__ float scale[8];
  const int w = __builtin_amdgcn_readfirstlane(wave_id()), l = lane_id();
  const int c0 = blockIdx.x * (HALF ? 8 : 16 * R);
  S s;
  s.init(a, c0, 0, false, few_smem);
  i4v acc[R][1] = {};
  s.run(a, w, acc, [&] {
    typedef __bf16 b8 __attribute__((ext_vector_type(8)));
    typedef __bf16 b8u __attribute__((ext_vector_type(8), aligned(2)));
    for (int n = 0; n < a.N; ++n) {
      const __bf16* row = x + n * x_st;
      float m = 0.f;
      bool odd = false;
      for (int k = l * 8; k < K; k += 512) {
        b8 v = {};
        if (k + 8 <= K) {
          v = *reinterpret_cast<const b8u*>(row + k);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = k + e < K ? row[k + e] : (__bf16)0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float f = fabsf(bf2f(v[e]));
          odd |= !(f < __builtin_inff());
          m = fmaxf(m, f);
        }
      }
      const float sc = quant_scale(wave_fmax(m), __any(odd));
      if (threadIdx.x == 0) scale[n] = sc;
      // the workgroup's threads quantise a part of the row each, zeros up to its stride
      for (int k = threadIdx.x * 4; k < a.x_ld; k += 2048) {
        unsigned q = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (k + e < K) q |= (unsigned)(unsigned char)(int8_t)quant(bf2f(row[k + e]), sc) << (8 * e);
        *reinterpret_cast<unsigned*>(few_smem + n * a.x_ld + k) = q;
      }
    }
    __syncthreads();
  });
#pragma unroll
  for (int r = 0; r < R; ++r) red[w][r][l] = acc[r][0];
  __syncthreads();
  for (int r = w; r < R; r += WAVES) {
    const int n = l & 15, c = c0 + 16 * r + 4 * (l >> 4);
    const i4v v = skinny_sum<i4v, R, 1, WAVES>(red, r, 0, l);
    if (n < a.N && c < a.cols && (!HALF || l < 32)) epi.put(n, c, v, scale[n]);
  }
}

namespace {

template <int TILE>
using Tile = GemmTile<int8_t, 2, TILE == 0 ? 4 : TILE == 3 ? 1 : 2, TILE == 0 ? 4 : TILE == 3 ? 1 : 2, 2,
                      TILE == 3 ? 8 : TILE == 2 ? 4 : 2, false, false>;

GemmPlan plan_int8(int64_t N, int K, int O) { return plan_gemm(N, O, (K + 127) / 128); }

constexpr int kMaxK = 132104;       // 2^31 / (127 * 128): a weight may be -128
constexpr int64_t kMaxRow = 1 << 22;  // bytes between a weight's rows: a tile's offsets stay in 31 bits
bool int8_shape_ok(int64_t N, int K, int O) {
  return N > 0 && K > 0 && O > 0 && K <= kMaxK && N < (int64_t(1) << 30) &&
         (N / 128 + 1) * ((int64_t)O / 128 + 1) < (1 << 23);
}

// Columns a workgroup of few tokens: 64, 16 or 8, the most that leave a workgroup for each of 256
// CUs.  One token, with the weights in memory: K=1024 O=32000 10.3 us with 64, 18.8 with 16; O=5632 5.6
// with 16, 6.4 with 64, 8.2 with 8; K=2048 O=2048 5.7 with 8, 8.9 with 64; O=11264 12.0 with 16
// (10.3 with 64, which would leave 80 CUs idle: the cut is a little late there).
int few_cols(int O) { return O >= 64 * 512 / 2 ? 64 : O >= 16 * 256 ? 16 : 8; }

// Tokens that every workgroup quantises for itself, where that costs less than the launch of
// k_quant: one token of K=2048 O=11264 takes 11.5 us so and 13.5 else, four 21.9 and 13.4.  (In a
// graph, where launches cost less, two take 15.3 so, and four take 11.0 by the launch.)
bool fused(int64_t N, int K) { return N <= 2 && N * (up(K, 128) + 16) <= 8192 + 32; }
// Quantised tokens straight from memory to MFMA: up to 32, up to 64 where O is narrow.  In a graph,
// with the weights in memory, so and by the 64x64 tile: 16 of K=1024 O=32000 12.3 and 15.3 us, 32 15.9
// and 15.6; 32 of K=1024 O=5632 8.6 and 11.5; 64 of K=2048 O=2048 11.8 and 15.1.  The tile is ahead
// where the tokens' own reads weigh more: 32 of K=2048 O=11264 18.3 and 15.4, 64 of K=5632 O=2048 27.2
// and 24.7.
bool few(int64_t N, int O) { return N <= 32 || (N <= 64 && O < 4096); }

template <int R, int U, bool HALF>
void launch_few(const SkinnyArgs& a, const void* x, int64_t x_st, int K, const SkinnyScaled& e, hipStream_t st) {
  SD_LAUNCH("k_int8_few", (k_int8_few<R, U, HALF>), dim3((unsigned)a.tiles), dim3(512), (size_t)a.N * a.x_ld, st, a,
            (const __bf16*)x, x_st, K, e);
}
template <int NT>
void launch_skinny(int cols, const SkinnyArgs& a, const SkinnyScaled& e, hipStream_t st) {
  const dim3 grid(skinny_grid(a)), block(512);
  if (cols == 64) SD_LAUNCH("k_linear_int8", (k_skinny<int8_t, 4, NT, 8, 1, false, false, SkinnyScaled>), grid, block, 0, st, a, e);
  else if (cols == 16) SD_LAUNCH("k_linear_int8", (k_skinny<int8_t, 1, NT, 8, 2, false, false, SkinnyScaled>), grid, block, 0, st, a, e);
  else SD_LAUNCH("k_linear_int8", (k_skinny<int8_t, 1, NT, 8, 2, true, false, SkinnyScaled>), grid, block, 0, st, a, e);
}

struct Int8Ws { int8_t *q, *w; float* scale; void* parts; int64_t ld; size_t bytes; };
// w: a copy of the weight in rows of whole 16-byte chunks, where its own are not
Int8Ws carve_int8(int64_t N, int K, int O, const void* w, int64_t w_st, char* base) {
  Int8Ws s;
  size_t off = 0;
  auto take = [&](size_t b) { char* p = base + off; off = (off + b + 255) & ~size_t(255); return p; };
  s.ld = up(K, 16);
  s.q = (int8_t*)take((size_t)N * s.ld);
  s.scale = (float*)take((size_t)N * 4);
  s.w = nullptr;
  if (!few(N, O) && (K % 16 || (O > 1 && w_st % 16) || ((uintptr_t)w & 15))) s.w = (int8_t*)take((size_t)O * s.ld);
  s.parts = take(few(N, O) ? 0 : plan_int8(N, K, O).parts);
  s.bytes = off + 256;
  return s;
}

template <class E>
void quantize(int64_t N, int K, const E* x, int64_t x_st, int8_t* q, int64_t q_st, int q_end, float* scale,
              hipStream_t st) {
  const dim3 rows((unsigned)((N + 3) / 4)), block(256);
  if (K <= 1024) SD_LAUNCH("k_quant", (k_quant_rows<E, 2>), rows, block, 0, st, N, K, x, x_st, q, q_st, q_end, scale);
  else if (K <= 2048) SD_LAUNCH("k_quant", (k_quant_rows<E, 4>), rows, block, 0, st, N, K, x, x_st, q, q_st, q_end, scale);
  else if (K <= 4096) SD_LAUNCH("k_quant", (k_quant_rows<E, 8>), rows, block, 0, st, N, K, x, x_st, q, q_st, q_end, scale);
  else if (K <= 8192) SD_LAUNCH("k_quant", (k_quant_rows<E, 16>), rows, block, 0, st, N, K, x, x_st, q, q_st, q_end, scale);
  else SD_LAUNCH("k_quant", k_quant<E>, dim3((unsigned)N), block, 0, st, K, x, x_st, q, q_st, q_end, scale);
}
}
}  // namespace sd

using namespace sd;

extern "C" {

int sd_quantize_int8(int64_t N, int K, int is_fp32, const void* x, int64_t x_st, int8_t* q,
                     int64_t q_st, float* scale, void* stream) {
  if (N <= 0 || K <= 0 || N >= (1 << 24)) return SD_ERR_SHAPE;
  if (!x || !q || !scale || x_st < K || q_st < K) return SD_ERR_ARG;
  if (is_fp32) quantize(N, K, (const float*)x, x_st, q, q_st, K, scale, (hipStream_t)stream);
  else quantize(N, K, (const __bf16*)x, x_st, q, q_st, K, scale, (hipStream_t)stream);
  return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
}

size_t sd_linear_int8_workspace_bytes(int64_t N, int K, int O, const void* w, int64_t w_st) {
  return int8_shape_ok(N, K, O) ? carve_int8(N, K, O, w, w_st, nullptr).bytes : 0;
}

int sd_linear_int8(int64_t N, int K, int O, const void* x, int64_t x_st, const int8_t* w,
                   int64_t w_st, const float* w_scale, const void* bias, void* y, void* workspace,
                   size_t workspace_bytes, void* stream) {
  if (!int8_shape_ok(N, K, O) || N >= (1 << 24)) return SD_ERR_SHAPE;
  if (!x || !w || !w_scale || !y || !workspace || x_st < K || w_st < K || (O > 1 && w_st > kMaxRow))
    return SD_ERR_ARG;
  const Int8Ws s = carve_int8(N, K, O, w, w_st, (char*)up((int64_t)(uintptr_t)workspace, 256));
  if (workspace_bytes < s.bytes) return SD_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const OutBf o{(__bf16*)y, O};
  const bool some = few(N, O);
  const int cols = few_cols(O);
  const SkinnyScaled se{o, s.scale, w_scale, (const __bf16*)bias, O};
  SkinnyArgs sa{(const char*)w, nullptr, w_st, (const char*)s.q, s.ld, (int)N, K, O, (O + cols - 1) / cols, 1};
  if (some && fused(N, K)) {
    sa.x_ld = up(K, 128) + 16;
    if (cols == 64) launch_few<4, 1, false>(sa, x, x_st, K, se, st);
    else if (cols == 16) launch_few<1, 4, false>(sa, x, x_st, K, se, st);
    else launch_few<1, 4, true>(sa, x, x_st, K, se, st);
    return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
  }
  quantize(N, K, (const __bf16*)x, x_st, s.q, s.ld, (int)s.ld, s.scale, st);
  if (some) {
    if (N > 16) sa.groups = (int)((N + 31) / 32);
    if (N <= 16) launch_skinny<1>(cols, sa, se, st);
    else launch_skinny<2>(cols, sa, se, st);
    return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
  }
  if (s.w)
    SD_LAUNCH("k_gemm_pack", k_gemm_pack<int8_t>, dim3((unsigned)(O < 8192 ? O : 8192)), dim3(256), 0, st, w, w_st,
              (int64_t)O, K, s.w, s.ld);
  const int64_t ld = s.w || O == 1 ? s.ld : w_st, wide = s.w ? s.ld : K;
  GemmArgs g{};
  g.A = {(const char*)s.q, s.ld, N * s.ld, nullptr, 0};
  g.B = {(const char*)(s.w ? s.w : w), ld, (O - 1) * ld + wide, nullptr, 0};
  g.M = N; g.N = O; g.kbytes = (int)s.ld; g.steps = (K + 127) / 128;
  g.parts = s.parts;
  const EpiScaled e(o, s.scale, w_scale, (const __bf16*)bias, N, O);
  const GemmPlan p = plan_int8(N, K, O);
  const char *name = "k_linear_int8", *join = "k_linear_int8_join";
  if (p.tile == 0) launch_gemm<Tile<0>>(name, join, g, p, e, st);
  else if (p.tile == 1) launch_gemm<Tile<1>>(name, join, g, p, e, st);
  else if (p.tile == 2) launch_gemm<Tile<2>>(name, join, g, p, e, st);
  else launch_gemm<Tile<3>>(name, join, g, p, e, st);
  return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
}

}  // extern "C"
