// One token per row of logits from given uniform numbers.  With L the row's maximum and
// z_v = (l_v - L) / temperature, tokens are ranked by (logit descending, index ascending).
// Kept: the first top_k; of these the ones whose predecessors hold less than top_p of the
// mass sum exp(z) of the top_k; of these the ones with z >= log(min_p).  The token is the
// kept one with the largest z_v - log(-log u_v), the lowest index of equals: that is the
// smallest -log(u_v) exp(-z_v), an exponential race, exactly a draw from the kept tokens'
// renormalised softmax.
//
// One workgroup a row, and no sort.  One pass over logits and random numbers holds the race,
// the maximum and a histogram of masses (or numbers) over 4096 bins of z; the bins tell
// which one holds the cut.  The winner of the race over all tokens is the token wherever it
// lies before that bin, as it does with the probability of what is kept.  If it lies
// behind it, the fastest of the tokens that are kept is looked for among the threads' two
// fastest each (a thread that may hold a faster one, not kept in mind, reads its tokens
// again).  Only a winner inside the cut's bin needs the cut itself: the bin's tokens are
// listed and ranked against each other, or cut by radix selection on (logit, index) where
// they are more than the list holds (runs of equal logits).
// For top_k <= 256 one atomic a thread is enough: the k-th largest of the threads' own maxima
// bounds the k-th largest logit from below, and what reaches it is listed and ranked.
//
// Masses are whole numbers, summed in any order to the same bits: every call gives the
// same token.  Each octave of masses has a unit of its own, in which an FP32 exponential is
// exact: a light token weighs what it does, however many there are.  As -log u >= 1 - u, a token whose (1 - u) exp(-z) is more than 8 times the
// workgroup's best so far needs no logarithm, and as -log u <= 2 (1 - u) for u >= 1/4 that
// best is bounded before the first one is taken.
#include <hip/hip_runtime.h>

#include "sd_common.cuh"
#include "sd_internal.h"
#include "../../include/solvedelta_mixer.h"

namespace sd {

typedef unsigned long long u64;
constexpr int SMP_BINS = 4096, SMP_SMALL_K = 256;
constexpr int SMP_FIRST = 512;  // threads whose first tokens give R, however many a row has
constexpr int kMaxVocab = 1 << 22;
constexpr float kInf = __builtin_inff();
// Masses are 2^((l - R) c): R is the maximum of the row's first tokens, and the row's own may
// be up to 2^12 masses above it (else the pass is run again with R the maximum).
constexpr float kOver = 12.f;

// ranks: a larger key is drawn from first
__device__ __forceinline__ u64 rank_key(float l, int v) {
  if (l == 0.f) l = 0.f;  // -0 and +0 are equal
  const unsigned b = __float_as_uint(l);
  const unsigned k = b & 0x80000000u ? ~b : b | 0x80000000u;
  return ((u64)k << 32) | (0xffffffffu - (unsigned)v);
}
__device__ __forceinline__ int key_index(u64 key) { return (int)(0xffffffffu - (unsigned)key); }
__device__ __forceinline__ float key_logit(u64 key) {
  const unsigned k = (unsigned)(key >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

struct SampleArgs {
  int V;
  const void* logits; int64_t l_st;
  const float* noise; int64_t n_st;
  sd_sample_setting temperature, top_k, top_p, min_p;
  int64_t* token;
};
__device__ __forceinline__ double setting_f(const sd_sample_setting& s, int b) {
  return s.rows ? (double)((const float*)s.rows)[b] : s.value;
}
__device__ __forceinline__ long long setting_i(const sd_sample_setting& s, int b) {
  return s.rows ? ((const long long*)s.rows)[b] : (long long)s.value;
}

// 16 bytes of logits at any alignment of their type
typedef unsigned u4v __attribute__((ext_vector_type(4)));
template <class E> struct LogitVec;
template <> struct LogitVec<float> {
  static constexpr int N = 4;
  typedef unsigned v __attribute__((ext_vector_type(4), aligned(4)));
  static __device__ __forceinline__ float at(const u4v& q, int e) { return __uint_as_float(q[e]); }
};
template <> struct LogitVec<__bf16> {
  static constexpr int N = 8;
  typedef unsigned v __attribute__((ext_vector_type(4), aligned(2)));
  static __device__ __forceinline__ float at(const u4v& q, int e) {
    return __uint_as_float(e & 1 ? q[e >> 1] & 0xffff0000u : q[e >> 1] << 16);
  }
};

// A row's logits.  Of a row whose maximum is +infinity only the infinities count, all alike:
// `top` reads them as 0 and the others as -infinity.
template <class E, int T> struct LogitRow {
  typedef LogitVec<E> L;
  static constexpr int N = L::N;
  const E* p;
  int V;
  bool top;
  __device__ __forceinline__ float value(float l) const { return !top ? l : l == kInf ? 0.f : -kInf; }
  // f(index, vectors, how many are inside) for the thread's vectors, G at a time, then
  // g(index, logit) for the up to N - 1 tokens behind the last whole vector
  template <int G, class F, class H> __device__ __forceinline__ void groups(F f, H g) const {
    const int full = V - V % N;
    for (int v0 = (int)threadIdx.x * N; v0 < full; v0 += G * T * N) {
      u4v y[G];
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const int v = v0 + i * T * N;
        y[i] = *reinterpret_cast<const typename L::v*>(p + (v < full ? v : v0));
      }
      const int n = (full - v0 + T * N - 1) / (T * N);
      f(v0, y, n < G ? n : G);
    }
    const int v = full + (int)threadIdx.x;
    if (v < V) g(v, value((float)p[v]));
  }
  // f(index, logit) for each of the thread's tokens
  template <class F> __device__ __forceinline__ void each(F f) const {
    groups<4>(
        [&](int v0, const u4v(&y)[4], int n) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (i < n) {
#pragma unroll
              for (int e = 0; e < N; ++e) f(v0 + i * T * N + e, value(L::at(y[i], e)));
            }
        },
        f);
  }
};

// kept tokens' keys are at least this one's
struct SampleCut {
  float l;
  int v;
  __device__ __forceinline__ bool keeps(float x, int i) const { return x > l || (x == l && i <= v); }
};

template <int T> struct SampleLds {
  u64 hist[SMP_BINS];
  u64 key[T], mass[T];
  u64 red[T / 64];
  u64 rest, cut;
  int bin, n;
  unsigned bound;  // the race's best time so far
};
template <int T> __device__ __forceinline__ SampleLds<T>& smp_lds() {
  __shared__ SampleLds<T> s;
  return s;
}

// x of the lane that the DPP control names, 0 where there is none or its row is masked out
template <int CTRL, int ROWS> __device__ __forceinline__ u64 dpp(u64 x) {
  const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)x, CTRL, ROWS, 0xf, false);
  const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(x >> 32), CTRL, ROWS, 0xf, false);
  return (u64)hi << 32 | lo;
}
struct OpMax {
  static __device__ __forceinline__ u64 of(u64 a, u64 b) { return a > b ? a : b; }
};
struct OpSum {
  static __device__ __forceinline__ u64 of(u64 a, u64 b) { return a + b; }
};
// Inclusive scan over the 16 lanes of a row, and over the wave (0 is neutral): shifts within
// the rows, then a row's last lane to the next row, and lane 31 to the upper half.  Right for
// the wave's first lanes too where only those run.
template <class Op> __device__ __forceinline__ u64 row_scan(u64 x) {
  x = Op::of(x, dpp<0x111, 0xf>(x));
  x = Op::of(x, dpp<0x112, 0xf>(x));
  x = Op::of(x, dpp<0x114, 0xf>(x));
  return Op::of(x, dpp<0x118, 0xf>(x));
}
template <class Op> __device__ __forceinline__ u64 wave_scan(u64 x) {
  x = row_scan<Op>(x);
  x = Op::of(x, dpp<0x142, 0xa>(x));
  return Op::of(x, dpp<0x143, 0xc>(x));
}
__device__ __forceinline__ u64 lane_of(u64 x, int l) {
  return (u64)(unsigned)__builtin_amdgcn_readlane((int)(unsigned)(x >> 32), l) << 32 |
         (unsigned)__builtin_amdgcn_readlane((int)(unsigned)x, l);
}
// over the workgroup, for every thread
template <int T, class Op> __device__ __forceinline__ u64 block_reduce(u64 x) {
  SampleLds<T>& s = smp_lds<T>();
  static_assert(T / 64 <= 16, "one row of waves");
  x = wave_scan<Op>(x);
  __syncthreads();
  if (lane_id() == 63) s.red[wave_id()] = x;
  __syncthreads();
  return lane_of(row_scan<Op>(s.red[lane_id() & (T / 64 - 1)]), T / 64 - 1);
}
template <int T> __device__ __forceinline__ u64 block_max(u64 x) { return block_reduce<T, OpMax>(x); }
template <int T> __device__ __forceinline__ u64 block_min(u64 x) { return ~block_max<T>(~x); }
template <int T> __device__ __forceinline__ u64 block_sum(u64 x) { return block_reduce<T, OpSum>(x); }

template <int T> __device__ __forceinline__ void clear_hist() {
  SampleLds<T>& s = smp_lds<T>();
  for (int i = threadIdx.x; i < SMP_BINS; i += T) s.hist[i] = 0;
  if (threadIdx.x == 0) s.n = 0;
}

// Masses of the d-th octave from the peak's are whole numbers up to 2^31 in units of its own;
// up to 2^22 of them, in units that all octaves share (2^-41 of the largest mass there can be in the
// peak's octave), sum to less than 2^64.  What is cut off is less than one unit a bin: 2^-28 of the
// peak's mass in all.
constexpr int SMP_SHARED = 10;
__device__ __forceinline__ u64 to_shared(u64 sum, int d) {
  return d <= SMP_SHARED ? sum << (SMP_SHARED - d) : sum >> (d - SMP_SHARED);
}
// the least sum in the octave's own units that is x or more in shared ones
__device__ __forceinline__ u64 to_own(u64 x, int d) {
  const int k = SMP_SHARED - d;
  return k >= 0 ? (x + ((u64)1 << k) - 1) >> k : x << -k;
}

// The first bin whose inclusive sum, counted from bin 0, reaches target(sum of all): s.bin,
// and what is left of the target there in s.rest.  Returns the target; 0 where the sum of all is
// less.  first: the peak's octave where the bins hold masses, -1 where they hold numbers.
template <int T, class F> __device__ __forceinline__ u64 find_bin(int first, F target_of) {
  SampleLds<T>& s = smp_lds<T>();
  constexpr int PER = SMP_BINS / T;
  static_assert(64 % PER == 0, "a thread's bins are of one octave");
  const int octave = (int)threadIdx.x * PER >> 6, d = octave > first ? octave - first : 0;
  u64 h[PER], own = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    h[i] = s.hist[threadIdx.x * PER + i];
    if (first >= 0) h[i] = to_shared(h[i], d);
    own += h[i];
  }
  const u64 inc = wave_scan<OpSum>(own);
  __syncthreads();  // s.red may still be read by a wave behind
  if (lane_id() == 63) s.red[wave_id()] = inc;
  __syncthreads();
  u64 acc = inc - own, all = 0;
#pragma unroll
  for (int w = 0; w < T / 64; ++w) {
    const u64 r = s.red[w];
    if (w < wave_id()) acc += r;
    all += r;
  }
  const u64 target = target_of(all);
  if (acc < target && acc + own >= target) {
    int i = 0;
#pragma unroll
    for (int e = 0; e < PER - 1; ++e)
      if (i == e && acc + h[e] < target) { acc += h[e]; i = e + 1; }
    s.bin = threadIdx.x * PER + i;
    s.rest = first >= 0 ? to_own(target - acc, d) : target - acc;
  }
  __syncthreads();
  return all < target ? 0 : target;
}
__device__ __forceinline__ u64 target_of(double p, u64 total) {
  const u64 m = (u64)(fmax(p, 0.) * (double)total);
  return m ? m : 1ull;
}

__device__ __forceinline__ float clamp_u(float u) { return fminf(fmaxf(u, 0x1p-25f), 1.f - 0x1p-24f); }
// -log u.  Near 1, where the winners lie, the hardware's logarithm keeps only its absolute
// error: there the series in t = 1 - u (exact), through t^8, t < 1/16: 2^-35 of it is left out.
__device__ __forceinline__ float neg_log(float u) {
  const float t = 1.f - u;
  float p = 0.125f;
  p = __builtin_fmaf(p, t, 1.f / 7.f);
  p = __builtin_fmaf(p, t, 1.f / 6.f);
  p = __builtin_fmaf(p, t, 0.2f);
  p = __builtin_fmaf(p, t, 0.25f);
  p = __builtin_fmaf(p, t, 1.f / 3.f);
  p = __builtin_fmaf(p, t, 0.5f);
  p = __builtin_fmaf(p, t, 1.f);
  return t < 0.0625f ? t * p : -0.693147181f * __builtin_amdgcn_logf(u);
}

// a time no kept token loses to: rank 0 takes at most -log 2^-25 = 17.4
constexpr u64 kNobody = 0x41900000ffffffffull;  // 18, no token
constexpr float kPass = 8.f;   // tokens slower than this many best times are passed over
__device__ __forceinline__ float time_of(u64 key) { return __uint_as_float((unsigned)(key >> 32)); }

// A thread's two fastest tokens.
struct TwoBest {
  u64 k1, k2;
  float l1, l2;
  __device__ __forceinline__ void meet(u64 k, float l) {
    if (k < k2) {
      const bool first = k < k1;
      k2 = first ? k1 : k;
      l2 = first ? l1 : l;
      k1 = first ? k : k1;
      l1 = first ? l : l1;
    }
  }
};

// What is kept: tokens of bins up to `bin` (4096: all), in the order of ranks up to `cut`, and
// by min_p.
struct SampleKept {
  int bin;
  SampleCut cut;
  float peak, dmax;  // the maximum; min_p keeps peak - l <= dmax
};

enum { HIST_NONE, HIST_COUNT, HIST_MASS };

// A row with its settings.
template <class E, int T> struct SampleRow {
  LogitRow<E, T> row;
  const float* noise;
  float R, c;   // masses are 2^((l - R) c)
  static constexpr int N = LogitVec<E>::N, G = 16 / N;
  __device__ __forceinline__ float expo(float l) const { return (l - R) * c; }
  // 64 bins an octave of the mass, from 2^12 down to 2^-52; the last takes what is behind.  A
  // token is looked for in the bin where it was counted: the multiply-add is written out, since
  // the compiler would fuse kOver - expo in one place and not in another, which at a bin's edge
  // are different bins (20 of 10^6 FP32 logits).
  __device__ __forceinline__ int bin(float l) const {
    const int b = (int)fminf(__builtin_fmaf(expo(l), -64.f, kOver * 64.f), (float)(SMP_BINS - 1));
    return b < 0 ? 0 : b;
  }
  // A mass x in bin b, in units of its octave's, from 2^30 to 2^31 of them (the last octave has the
  // lighter ones too): FP32's 24 bits are all whole ones.
  static __device__ __forceinline__ unsigned units(float x, int b) {
    return (unsigned)__builtin_amdgcn_ldexpf(x, 31 - (int)kOver + (b >> 6));
  }
  __device__ __forceinline__ float mass(float l) const { return fmaxf(__builtin_amdgcn_exp2f(expo(l)), 0.f); }
  __device__ __forceinline__ unsigned term(int hist, float l, int b) const {
    return hist == HIST_MASS ? units(mass(l), b) : l > -kInf ? 1u : 0u;
  }
  // the race's time as a key, smaller is better, with the index behind it
  __device__ __forceinline__ u64 time(int v, float l, float u) const {
    return ((u64)__float_as_uint(neg_log(clamp_u(u)) * __builtin_amdgcn_exp2f(-expo(l))) << 32) | (unsigned)v;
  }
  // a time that the token's own is not below (1e-5 of it: the rounding), whatever u is
  __device__ __forceinline__ float least(float l, float u) const {
    return fminf(fmaxf(1.f - u, 0x1p-24f), 17.f) * __builtin_amdgcn_exp2f(-expo(l));
  }
  __device__ __forceinline__ bool keeps(const SampleKept& k, float l, int v) const {
    return k.cut.keeps(l, v) && k.peak - l <= k.dmax && bin(l) <= k.bin;
  }
  // The pass over all tokens that `in` keeps (CUT; else the whole row): the thread's two
  // fastest and its maximum; and the histogram.
  template <bool CUT>
  __device__ __forceinline__ TwoBest pass(int hist, const SampleCut in, float* top) const {
    SampleLds<T>& s = smp_lds<T>();
    TwoBest b{kNobody, kNobody, 0.f, 0.f};
    float mx = -kInf;
    auto one = [&](int v, float l, float u) {
      if (CUT ? in.keeps(l, v) : l > -kInf) b.meet(time(v, l, u), l);
    };
    auto count = [&](int v, float l, float x) {
      if (CUT && !in.keeps(l, v)) return;
      const int at = bin(l);
      const unsigned m = hist == HIST_MASS ? units(x, at) : l > -kInf ? 1u : 0u;
      if (m) atomicAdd(&s.hist[at], (u64)m);
    };
    row.template groups<G>(
        [&](int v0, const u4v(&y)[G], int n) {
          typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
          v4 u[G][N / 4];
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int h = 0; h < N / 4; ++h)
              u[i][h] = *reinterpret_cast<const v4*>(noise + v0 + (i < n ? i * T * N : 0) + 4 * h);
#pragma unroll
          for (int i = 0; i < G; ++i) {
            if (i >= n) break;
            // -log u >= 1 - u (of u as it is read), and <= 2 (1 - u) from u = 1/4 on
            float lower[N], far = __uint_as_float(__hip_atomic_load(&s.bound, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP));
            float near = kInf;
#pragma unroll
            for (int e = 0; e < N; ++e) {
              const float l = row.value(LogitVec<E>::at(y[i], e)), w = u[i][e >> 2][e & 3];
              mx = fmaxf(mx, l);
              lower[e] = least(l, w);
              if (CUT && !in.keeps(l, v0 + i * T * N + e)) lower[e] = kInf;
              near = fminf(near, w >= 0.25f ? lower[e] : kInf);
            }
            if (hist) {
#pragma unroll
              for (int e = 0; e < N; ++e) {
                const float l = row.value(LogitVec<E>::at(y[i], e));
                count(v0 + i * T * N + e, l, hist == HIST_MASS ? mass(l) : 0.f);
              }
            }
            // a better bound on the race's best time, before any logarithm (at a row's end the
            // wave's first lanes are left: the scan's last of them has it)
            near *= 2.0001f;
            if (__any(near < far)) {
              const int last = __popcll(__ballot(1)) - 1;
              const unsigned b32 = (unsigned)~lane_of(wave_scan<OpMax>(~(u64)__float_as_uint(near)), last);
              if (lane_id() == 0) atomicMin(&s.bound, b32);
              far = fminf(far, __uint_as_float(b32));
            }
            // no time below the bound but of these (1e-5: the rounding)
            const float bound = fminf(time_of(b.k2), far * kPass) * 1.00001f;
            bool may = false;
#pragma unroll
            for (int e = 0; e < N; ++e) may |= lower[e] <= bound;
            if (may) {
              const u64 old = b.k1;
#pragma unroll
              for (int e = 0; e < N; ++e)
                if (lower[e] <= bound) one(v0 + i * T * N + e, row.value(LogitVec<E>::at(y[i], e)), u[i][e >> 2][e & 3]);
              if (b.k1 < old) atomicMin(&s.bound, (unsigned)(b.k1 >> 32));
            }
          }
        },
        [&](int v, float l) {
          mx = fmaxf(mx, l);
          if (hist) count(v, l, mass(l));
          one(v, l, noise[v]);
        });
    *top = mx;
    return b;
  }
  // the thread's two fastest of its kept tokens, all looked at but those slower than `lim`
  __device__ __forceinline__ TwoBest again(const SampleKept k, float lim) const {
    TwoBest b{kNobody, kNobody, 0.f, 0.f};
    lim *= 1.00001f;
    auto one = [&](int v, float l, float u) {
      if (least(l, u) <= lim && keeps(k, l, v)) b.meet(time(v, l, u), l);
    };
    row.template groups<G>(
        [&](int v0, const u4v(&y)[G], int n) {
          typedef float v4 __attribute__((ext_vector_type(4), aligned(4)));
          v4 u[G][N / 4];
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int h = 0; h < N / 4; ++h)
              u[i][h] = *reinterpret_cast<const v4*>(noise + v0 + (i < n ? i * T * N : 0) + 4 * h);
#pragma unroll
          for (int i = 0; i < G; ++i) {
            if (i >= n) break;
#pragma unroll
            for (int e = 0; e < N; ++e) one(v0 + i * T * N + e, row.value(LogitVec<E>::at(y[i], e)), u[i][e >> 2][e & 3]);
          }
        },
        [&](int v, float l) { one(v, l, noise[v]); });
    return b;
  }
  // The fastest kept token over the workgroup; *l: its logit.  over: no token that the thread
  // has passed over is faster.
  __device__ __forceinline__ u64 fastest(const SampleKept& k, TwoBest& two, float& over, float* l) const {
    const bool v1 = two.k1 != kNobody && keeps(k, two.l1, (int)(unsigned)two.k1);
    const bool v2 = two.k2 != kNobody && keeps(k, two.l2, (int)(unsigned)two.k2);
    u64 mine = v1 ? two.k1 : v2 ? two.k2 : kNobody;
    u64 best = block_min<T>(mine);
    // a thread without one of its two has those behind them left; any has what it passed over
    const float least = v1 || v2 ? over : fminf(time_of(two.k2), over);
    const bool look = least < time_of(best) || (least == time_of(best) && !v1 && !v2);
    if (__syncthreads_or(look)) {
      if (look) {
        two = again(k, time_of(best));
        over = time_of(best);
        mine = two.k1;
      }
      best = block_min<T>(mine);
    }
    SampleLds<T>& s = smp_lds<T>();
    if (mine == best) s.cut = __float_as_uint(mine == two.k1 ? two.l1 : two.l2);
    __syncthreads();
    *l = __uint_as_float((unsigned)s.cut);
    return best;
  }
};

// The smallest of the keys in [lo, hi], all of one bin, whose inclusive sum of `term` over larger
// keys reaches `rest`: 8 bits at a time from the first in which lo and hi differ.
template <class E, int T>
__device__ __forceinline__ u64 radix_cut(const SampleRow<E, T> r, int hist, int bin, u64 lo, u64 hi, u64 rest) {
  SampleLds<T>& s = smp_lds<T>();
  int top = lo == hi ? 0 : 64 - __clzll((long long)(lo ^ hi));  // bits that may differ
  u64 prefix = top >= 64 ? 0 : hi >> top;
  while (top > 0) {
    const int nbits = top < 8 ? top : 8, shift = top - nbits;
    if (threadIdx.x < 256) s.hist[threadIdx.x] = 0;
    __syncthreads();
    r.row.each([&](int v, float l) {
      const u64 key = rank_key(l, v);
      if (key < lo || key > hi || (top < 64 && key >> top != prefix)) return;
      const unsigned m = r.term(hist, l, bin);
      if (m) atomicAdd(&s.hist[(key >> shift) & ((1 << nbits) - 1)], (u64)m);
    });
    __syncthreads();
    if (threadIdx.x == 0) {
      int d = (1 << nbits) - 1;
      u64 acc = 0;
      while (d > 0 && acc + s.hist[d] < rest) acc += s.hist[d--];
      s.bin = d;
      s.rest = rest - acc;
    }
    __syncthreads();
    prefix = (prefix << nbits) | (u64)s.bin;
    rest = s.rest;
    top = shift;
    __syncthreads();
  }
  return prefix;
}

// The key inside `bin` of the tokens that `in` keeps at which the sum of their terms reaches
// `rest`.
template <class E, int T>
__device__ __forceinline__ SampleCut exact_cut(const SampleRow<E, T> r, int hist, const SampleCut in, int bin, u64 rest) {
  SampleLds<T>& s = smp_lds<T>();
  __syncthreads();
  if (threadIdx.x == 0) s.n = 0;
  __syncthreads();
  u64 lo = ~0ull, hi = 0;
  r.row.each([&](int v, float l) {
    if (r.bin(l) != bin || !in.keeps(l, v)) return;
    const unsigned m = r.term(hist, l, bin);
    if (!m) return;
    const u64 key = rank_key(l, v);
    lo = key < lo ? key : lo;
    hi = key > hi ? key : hi;
    const int at = atomicAdd(&s.n, 1);
    if (at < T) { s.key[at] = key; s.mass[at] = m; }
  });
  __syncthreads();
  const int n = s.n;
  u64 key;
  if (n <= T) {
    if ((int)threadIdx.x < n) {
      const u64 own = s.key[threadIdx.x];
      u64 acc = 0;
#pragma unroll 4
      for (int j = 0; j < n; ++j) acc += s.key[j] > own ? s.mass[j] : 0;
      if (acc < rest && acc + s.mass[threadIdx.x] >= rest) s.cut = own;
    }
    __syncthreads();
    key = s.cut;
    __syncthreads();
  } else {
    lo = ~block_max<T>(~lo);
    hi = block_max<T>(hi);
    key = radix_cut(r, hist, bin, lo, hi, rest);
  }
  return {key_logit(key), key_index(key)};
}

// 128 bins an octave of d = L - l from 2^-12 to 2^20, monotone, whatever the temperature; the
// first and the last take what lies outside
constexpr int kBinOff = 115 << 7;
__device__ __forceinline__ int octave_bin(float d) {
  const int b = (int)(__float_as_uint(d) >> 16) - kBinOff;
  return b < 0 ? 0 : b > SMP_BINS - 1 ? SMP_BINS - 1 : b;
}

// k <= 256: the tokens that reach the k-th largest of the threads' maxima (`own`), all where
// fewer threads than k have a token, listed and ranked against each other; the winner's key,
// or 0 if they are more than the list holds.  r.R is the maximum.
template <class E, int T>
__device__ __forceinline__ u64 draw_listed(const SampleRow<E, T> r, float own, int k, double p, float dmax) {
  SampleLds<T>& s = smp_lds<T>();
  clear_hist<T>();
  __syncthreads();
  if (own > -kInf) atomicAdd(&s.hist[octave_bin(r.R - own)], 1ull);
  __syncthreads();
  // bin b holds edge(b) <= d < edge(b + 1)
  const bool some = find_bin<T>(-1, [&](u64) { return (u64)k; }) != 0;
  const float to = some && s.bin < SMP_BINS - 1 ? __uint_as_float((unsigned)(s.bin + 1 + kBinOff) << 16) : kInf;
  auto list = [&](int v, float l) {
    if (!(r.R - l < to)) return;
    const int at = atomicAdd(&s.n, 1);
    // masses up to 1, of which 2^-52 is left
    if (at < T) { s.key[at] = rank_key(l, v); s.mass[at] = (u64)(r.mass(l) * 0x1p52f); }
  };
  typedef LogitVec<E> L;
  r.row.template groups<4>(
      [&](int v0, const u4v(&y)[4], int n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (i >= n) break;
          bool any = false;
#pragma unroll
          for (int e = 0; e < L::N; ++e) any |= r.R - r.row.value(L::at(y[i], e)) < to;
          if (any) {
#pragma unroll
            for (int e = 0; e < L::N; ++e) list(v0 + i * T * L::N + e, r.row.value(L::at(y[i], e)));
          }
        }
      },
      list);
  __syncthreads();
  const int n = s.n;
  __syncthreads();
  if (n > T) return 0;
  // ranks and the masses before each, by as many lanes of a wave as there are for every token
  int lanes = 1;
  while (lanes < 64 && 2 * lanes * n <= T) lanes *= 2;
  const int item = (int)threadIdx.x / lanes, part = (int)threadIdx.x % lanes;
  u64 key = 0, m = 0, before = 0, best = kNobody;
  int rank = 0;
  if (item < n) {
    key = s.key[item];
    m = s.mass[item];
#pragma unroll 4
    for (int j = part; j < n; j += lanes) {
      const bool first = s.key[j] > key;
      rank += first;
      before += first ? s.mass[j] : 0;
    }
  }
  for (int d = 1; d < lanes; d *= 2) {
    rank += __shfl_xor(rank, d);
    before += __shfl_xor(before, d);
  }
  const bool in = item < n && part == 0 && rank < k;
  const u64 total = p < 1. ? block_sum<T>(in ? m : 0) : 0;
  if (in && (!(p < 1.) || before < target_of(p, total))) {
    const int v = key_index(key);
    const float l = key_logit(key);
    if (r.R - l <= dmax) best = r.time(v, l, r.noise[v]);
  }
  return block_min<T>(best);
}

template <class E, int T>
__global__ __launch_bounds__(T, 4) void k_sample(SampleArgs a) {
  SampleLds<T>& s = smp_lds<T>();
  const int b = blockIdx.x, V = a.V;
  SampleRow<E, T> r{{(const E*)a.logits + (int64_t)b * a.l_st, V, false}, a.noise + (int64_t)b * a.n_st, 0.f, 0.f};
  const float t = (float)setting_f(a.temperature, b), mp = (float)setting_f(a.min_p, b);
  const double p = setting_f(a.top_p, b);
  const long long k = setting_i(a.top_k, b);
  const bool greedy = !(t > 0.f), by_k = k > 0 && k < V, by_p = p < 1.;
  r.c = fminf(1.44269504f / t, 3e38f);
  const float dmax = mp > 0.f ? -logf(fminf(mp, 1.f)) * t : 3.40282347e38f;

  // the maximum of the row, or of its first vectors
  const bool small = by_k && k <= SMP_SMALL_K, whole = greedy || small;
  float own = -kInf;
  if (whole) {
    r.row.each([&](int, float l) { own = fmaxf(own, l); });  // the larger of a number and NaN is the number
  } else {
    const int v0 = (int)threadIdx.x * LogitVec<E>::N;
    if ((int)threadIdx.x < SMP_FIRST && v0 + LogitVec<E>::N <= V) {
      const u4v y = *reinterpret_cast<const typename LogitVec<E>::v*>(r.row.p + v0);
#pragma unroll
      for (int e = 0; e < LogitVec<E>::N; ++e) own = fmaxf(own, LogitVec<E>::at(y, e));
    }
  }
  r.R = key_logit(block_max<T>(rank_key(own, -1)));
  if (whole && r.R == -kInf) {  // every token is ruled out
    if (threadIdx.x == 0) a.token[b] = -1;
    return;
  }
  if (greedy) {
    u64 first = 0;
    if (own == r.R) r.row.each([&](int v, float l) {
      if (l == r.R) {
        const u64 key = 0xffffffffu - (unsigned)v;
        if (key > first) first = key;
      }
    });
    first = block_max<T>(first);
    if (threadIdx.x == 0) a.token[b] = key_index(first);
    return;
  }
  if (small) {
    if (r.R == kInf) {
      r.row.top = true;
      own = r.row.value(own);
      r.R = 0.f;
    }
    const u64 best = draw_listed(r, own, (int)k, p, dmax);
    if (best) {
      if (threadIdx.x == 0) a.token[b] = (int)(unsigned)best;
      return;
    }
  }
  // with both filters, the first one's cut and then the pass for the second among what it keeps
  const SampleCut all{-kInf, -1};  // everything but -infinity
  SampleCut in = all;
  TwoBest two;
  u64 target = 0;
  float peak;
  for (int stage = by_k ? 0 : 1; stage < 2; ++stage) {
    const int hist = stage == 0 ? HIST_COUNT : by_p ? HIST_MASS : HIST_NONE;
    if (stage == 1 && by_k && !by_p) break;
    for (;;) {
      __syncthreads();
      if (hist) clear_hist<T>();
      if (threadIdx.x == 0) s.bound = (unsigned)(kNobody >> 32);
      __syncthreads();
      float mx;
      two = in.v == -1 && in.l == -kInf ? r.template pass<false>(hist, in, &mx) : r.template pass<true>(hist, in, &mx);
      peak = key_logit(block_max<T>(rank_key(mx, -1)));
      if (peak == -kInf) {
        if (threadIdx.x == 0) a.token[b] = -1;
        return;
      }
      if (peak == kInf) {
        r.row.top = true;
        r.R = 0.f;
      } else if (!((peak - r.R) * r.c <= kOver)) {
        r.R = peak;
      } else {
        break;
      }
    }
    const int first = hist == HIST_MASS ? r.bin(peak) >> 6 : -1;
    target = hist ? find_bin<T>(first, [&](u64 total) { return hist == HIST_COUNT ? (u64)k : target_of(p, total); }) : 0;
    if (stage == 0 && by_p && target) in = exact_cut(r, HIST_COUNT, all, s.bin, s.rest);
  }
  SampleKept kept{SMP_BINS, in, peak, dmax};
  const u64 rest = s.rest;
  if (target) kept.bin = s.bin;
  float over = __uint_as_float(s.bound) * kPass, l;
  u64 best = r.fastest(kept, two, over, &l);
  if (target && r.bin(l) == kept.bin) {
    kept.cut = exact_cut(r, by_p ? HIST_MASS : HIST_COUNT, in, kept.bin, rest);
    best = r.fastest(kept, two, over, &l);
  }
  if (threadIdx.x == 0) a.token[b] = (int)(unsigned)best;
}

// Rows of 1024 threads have a CU to themselves; of 512, two share one, and one's loads and
// arithmetic run in the other's waits.  512 x 50001 FP32, in a graph: 40.9 and 35.1 us without a
// filter, 39.0 and 34.5 at top_k 50, 54.8 and 50.4 at top_p 0.9; 2048 x 32000 bf16: 108 and 81, 85 and
// 57, 149 and 107; 257 x 50001: 32 and 26, 31 and 24, 43 and 36 (32 and 32 at min_p).  The token
// is the same.
template <class E> void launch_sample(int B, const SampleArgs& a, hipStream_t st) {
  if (B > 256) SD_LAUNCH("k_sample", (k_sample<E, 512>), dim3(B), dim3(512), 0, st, a);
  else SD_LAUNCH("k_sample", (k_sample<E, 1024>), dim3(B), dim3(1024), 0, st, a);
}

}  // namespace sd

using namespace sd;

extern "C" int sd_sample_tokens(int B, int V, int is_fp32, const void* logits, int64_t logits_st,
                                const float* noise, int64_t noise_st,
                                const sd_sample_setting* settings, int64_t* token, void* stream) {
  if (B <= 0 || V <= 0 || V > kMaxVocab) return SD_ERR_SHAPE;
  if (!logits || !noise || !settings || !token) return SD_ERR_ARG;
  SampleArgs a{V, logits, logits_st, noise, noise_st, settings[0], settings[1], settings[2],
               settings[3], token};
  hipStream_t st = (hipStream_t)stream;
  if (is_fp32) launch_sample<float>(B, a, st);
  else launch_sample<__bf16>(B, a, st);
  return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
}
