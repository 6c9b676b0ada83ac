// Gated feed-forward block of the causal LM (reference: causallsso/modeling_solvedelta.py:31-100),
// forward and backward, over N tokens:
//   g = x Wg^T, u = x Wu^T, s = sigmoid(g), a = g s u, y = a Wd^T
//   da = dy Wd, du = da g s, dg = da u s (1 + g (1 - s))
//   dx = [dg du] [Wg; Wu], d[Wg; Wu] = [dg du]^T x, dWd = dy^T a
// bf16 operands, FP32 sums.  a, dg and du are rounded to bf16 once, as operands of the
// products that read them; the activation and its derivative are formed from FP32 sums in
// the products' own kernels:
//   k_ffn_gate_up  both projections of a tile, a, and for a backward g and u
//   k_ffn_down     y
//   k_ffn_da       da of a tile, then dg and du
//   k_ffn_dx, k_ffn_dgate_up, k_ffn_ddown
// g and u are kept for the backward as FP16 with one power-of-two scale per 32x32 block (the
// block's largest value at the top of FP16's range): 11 significant bits for all values down
// to 2^-29 of the block's largest, in the 4 bytes a pair that bf16 would take with 8.  a is
// kept as the down projection read it.
#include <hip/hip_runtime.h>

#include "sd_skinny.cuh"
#include "../../include/solvedelta_mixer.h"

namespace sd {

// s = sigmoid(g); 1 / inf = 0 where the exponential overflows
__device__ __forceinline__ float ffn_sigm(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// The kept blocks: 16 FP16 values a lane in the MFMA result's order, g's 2 KiB then u's;
// scales [block][2].
struct FfnSaved {
  _Float16* v;
  float* scale;
  int64_t nb;  // blocks a row of blocks
};
typedef _Float16 f16x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ void keep_block(_Float16* p, float* scale, const float (&v)[16]) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const float a = fabsf(v[e]);
    m = fmaxf(m, a < __builtin_inff() ? a : 0.f);  // infinities and NaN stay what they are
  }
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) m = fmaxf(m, __shfl_xor(m, d));
  // 2^(14 - floor(log2 m)), kept away from the ends of FP32's range
  const int ex = max((int)(__float_as_uint(m) >> 23), 27) - 127;
  const float up = __uint_as_float((unsigned)(127 + 14 - ex) << 23);
  f16x16 h;
#pragma unroll
  for (int e = 0; e < 16; ++e) h[e] = (_Float16)(v[e] * up);
  *reinterpret_cast<f16x16*>(p + lane_id() * 16) = h;
  if (lane_id() == 0) *scale = __uint_as_float((unsigned)(127 - 14 + ex) << 23);
}

struct EpiGateUp : EpiNothing {
  OutBf a;      // [M][a.ld], a.ld >= N: zeros behind N
  FfnSaved s;   // s.v null: nothing is kept
  int64_t M, N;
  EpiGateUp(OutBf a_, FfnSaved s_, int64_t M_, int64_t N_) : a(a_), s(s_), M(M_), N(N_) {}
  __device__ __forceinline__ void operator()(int64_t mb, int64_t nb, None, None, const f16v& g_, const f16v& u_) const {
    if (mb >= M || nb >= N) return;
    const int64_t m = mb + (lane_id() & 31);
    float g[16], u[16], v[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool in = nb + 8 * (e >> 2) + 4 * (lane_id() >> 5) + (e & 3) < N;
      g[e] = in ? g_[e] : 0.f;
      u[e] = in ? u_[e] : 0.f;
      v[e] = g[e] * ffn_sigm(g[e]) * u[e];
    }
    store_block(a, m, m < M, nb, a.ld, v);
    if (s.v) {
      const int64_t b = (mb >> 5) * s.nb + (nb >> 5);
      keep_block(s.v + b * 2048, s.scale + b * 2, g);
      keep_block(s.v + b * 2048 + 1024, s.scale + b * 2 + 1, u);
    }
  }
};

struct EpiDact : EpiNothing {
  OutBf dg, du;  // [M][ld]; du lies behind dg's N columns, with zeros up to its row's end
  FfnSaved s;
  int64_t M, N;
  EpiDact(OutBf dg_, OutBf du_, FfnSaved s_, int64_t M_, int64_t N_) : dg(dg_), du(du_), s(s_), M(M_), N(N_) {}
  struct Kept {
    f16x16 g, u;
    float gs, us;
  };
  __device__ __forceinline__ Kept pre(int64_t mb, int64_t nb) const {
    if (mb >= M || nb >= N) return {};
    const int64_t b = (mb >> 5) * s.nb + (nb >> 5);
    const _Float16* v = s.v + b * 2048 + lane_id() * 16;
    return {*reinterpret_cast<const f16x16*>(v), *reinterpret_cast<const f16x16*>(v + 1024), s.scale[b * 2],
            s.scale[b * 2 + 1]};
  }
  __device__ __forceinline__ void operator()(int64_t mb, int64_t nb, None, const Kept& k, const f16v& d) const {
    if (mb >= M || nb >= N) return;
    const int64_t m = mb + (lane_id() & 31);
    float vg[16], vu[16];
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const bool in = nb + 8 * (e >> 2) + 4 * (lane_id() >> 5) + (e & 3) < N;
      const float g = (float)k.g[e] * k.gs, u = (float)k.u[e] * k.us, sg = ffn_sigm(g), x = in ? d[e] : 0.f;
      vu[e] = x * g * sg;
      vg[e] = x * u * sg * (1.f + g * (1.f - sg));
    }
    const bool ok = m < M;
    store_block(dg, m, ok, nb, N, vg);
    store_block(du, m, ok, nb, du.ld - N, vu);
    // the row's end may lie up to 3 columns behind the last block (N = 29 to 31 of 32)
    if (ok && nb + 32 >= N)
      for (int64_t n = nb + 32 + (lane_id() >> 5); n < du.ld - N; n += 2) du.p[m * du.ld + n] = f2bf(0.f);
  }
};

// few tokens: a, and y
struct SkinnyGateUp {
  OutBf a;      // [N][a.ld], zeros behind `cols`
  int cols;
  __device__ __forceinline__ void operator()(int n, int c, const f4& g, const f4& u) const {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = c + e < cols ? g[e] * ffn_sigm(g[e]) * u[e] : 0.f;
    store4(a, n, c, (int)a.ld, v);
  }
};
struct SkinnyOut {
  OutBf o;
  int cols;
  __device__ __forceinline__ void operator()(int n, int c, const f4& a) const {
    const float v[4] = {a[0], a[1], a[2], a[3]};
    store4(o, n, c, cols, v);
  }
};

namespace {

typedef __bf16 bf;
// Straight from memory to MFMA each workgroup of 8 columns reads all tokens, N I (D + O) / 4 bytes
// in all.  Up to 64 tokens and 100 MB of such reads that is the faster way, beyond it the 64x64 tile
// is.  In a graph, with the weights in memory and (in brackets) in the caches, straight and tile:
// one token of D=2048 I=5632 23.4 and 31.3 us (19.1, 28.2), 16 (92 MB) 29.3 and 31.6 (26.3, 28.3), 24
// (138 MB) 35.0 and 31.9 (32.2, 28.5); 64 of D=1024 I=2816 (92 MB) 22.2 and 23.9 (20.3, 22.1).
bool few(const sd_ffn& f) { return f.N <= 64 && f.N * f.I * ((int64_t)f.D + f.O) <= 400000000; }

template <int NT>
void few_tokens(const sd_ffn& f, bf* a, int64_t la, void* y, hipStream_t st) {
  const int groups = ((int)f.N + 16 * NT - 1) / (16 * NT);
  const OutBf oa{a, la}, oy{(bf*)y, f.O};
  const int64_t gu_ld = f.gate_up_st * 2;
  const SkinnyArgs up{(const char*)f.gate_up, (const char*)f.gate_up + f.I * gu_ld, gu_ld, (const char*)f.x,
                      f.x_st * 2, (int)f.N, f.D * 2, f.I, (f.I + 7) / 8, groups};
  SD_LAUNCH("k_ffn_gate_up", (k_skinny<bf, 1, NT, 8, NT == 1 ? 4 : 2, true, true, SkinnyGateUp>), dim3(skinny_grid(up)),
            dim3(512), 0, st, up, (SkinnyGateUp{oa, f.I}));
  const SkinnyArgs dn{(const char*)f.down, nullptr, f.down_st * 2, (const char*)a, la * 2, (int)f.N, f.I * 2, f.O,
                      (f.O + 7) / 8, groups};
  SD_LAUNCH("k_ffn_down", (k_skinny<bf, 1, NT, 16, NT == 1 ? 4 : 2, true, false, SkinnyOut>), dim3(skinny_grid(dn)),
            dim3(1024), 0, st, dn, (SkinnyOut{oy, f.O}));
}

template <bool AT, bool BT, bool P> using Tile0 = GemmTile<bf, 2, 4, 4, 2, 2, AT, BT, P>;
template <bool AT, bool BT, bool P> using Tile1 = GemmTile<bf, 2, 2, 2, 2, 2, AT, BT, P>;
template <bool AT, bool BT, bool P> using Tile2 = GemmTile<bf, 2, 2, 2, 2, 4, AT, BT, P>;
template <bool AT, bool BT, bool P> using Tile3 = GemmTile<bf, 2, 1, 1, 2, 8, AT, BT, P>;

template <bool AT, bool BT, bool P, class Epi>
void product(const char* name, const char* join, const GemmArgs& g, const GemmPlan& p, const Epi& e, hipStream_t st) {
  if (p.tile == 0) launch_gemm<Tile0<AT, BT, P>>(name, join, g, p, e, st);
  else if (p.tile == 1) launch_gemm<Tile1<AT, BT, P>>(name, join, g, p, e, st);
  else if (p.tile == 2) launch_gemm<Tile2<AT, BT, P>>(name, join, g, p, e, st);
  else launch_gemm<Tile3<AT, BT, P>>(name, join, g, p, e, st);
}

int64_t steps_of(int64_t K) { return (K + 63) / 64; }
OutBf out_bf(void* p, int64_t ld) { return {(bf*)p, ld}; }

// An operand's rows as the products read them: in place where they are whole aligned
// 16-byte chunks, else from a padded copy.
struct Rows {
  const bf* p;
  int64_t ld, rows;
  int width;
  bool packed;
  GemmOperand op(int64_t first = 0, int64_t n = -1) const {
    if (n < 0) n = rows;
    const int64_t w = packed ? ld : width;
    return {(const char*)(p + first * ld), ld * 2, ((n - 1) * ld + w) * 2, nullptr, 0};
  }
};
struct Carver {
  char* base;
  size_t off = 0;
  template <class T> T* take(size_t bytes) {
    T* p = (T*)(base + off);
    off = (off + bytes + 255) & ~size_t(255);
    return p;
  }
};
Rows rows_of(const void* p, int64_t st, int64_t rows, int width, Carver& c) {
  if (rows == 1) st = up(width, 8);  // one row has no stride
  if (width % 8 == 0 && st % 8 == 0 && ((uintptr_t)p & 15) == 0) return {(const bf*)p, st, rows, width, false};
  const int64_t ld = up(width, 8);
  return {c.take<bf>((size_t)rows * ld * 2), ld, rows, width, true};
}
void pack(const Rows& r, const void* src, int64_t st, hipStream_t s) {
  if (!r.packed) return;
  SD_LAUNCH("k_gemm_pack", k_gemm_pack<bf>, dim3((unsigned)(r.rows < 8192 ? r.rows : 8192)), dim3(256), 0, s,
            (const bf*)src, st, r.rows, r.width, (bf*)r.p, r.ld);
}

FfnSaved carve_saved(const sd_ffn& f, void* base) {
  const int64_t mb = up(f.N, 32) / 32, nb = up(f.I, 32) / 32;
  return {(_Float16*)base, (float*)((char*)base + (size_t)mb * nb * 4096), nb};
}
size_t saved_blocks_bytes(const sd_ffn& f) {
  return (size_t)up((up(f.N, 32) / 32) * (up(f.I, 32) / 32) * (4096 + 8), 256);
}
size_t a_bytes(const sd_ffn& f) { return (size_t)f.N * up(f.I, 8) * 2; }

GemmPlan plan_gate_up(const sd_ffn& f) { return plan_gemm(f.N, 2 * (int64_t)f.I, steps_of(f.D)); }
GemmPlan plan_down(const sd_ffn& f) { return plan_gemm(f.N, f.O, steps_of(f.I)); }
GemmPlan plan_da(const sd_ffn& f) { return plan_gemm(f.N, f.I, steps_of(f.O)); }
GemmPlan plan_dx(const sd_ffn& f) { return plan_gemm(f.N, f.D, steps_of(2 * (int64_t)f.I)); }
GemmPlan plan_dgate_up(const sd_ffn& f) { return plan_gemm(2 * (int64_t)f.I, f.D, steps_of(f.N)); }
GemmPlan plan_ddown(const sd_ffn& f) { return plan_gemm(f.O, f.I, steps_of(f.N)); }
size_t most(size_t a, size_t b) { return a > b ? a : b; }

// The parts' region is used by one product after another.
struct FfnFwdWs { Rows x, gu, down; bf* a; void* parts; size_t bytes; };
FfnFwdWs carve_ffn_fwd(const sd_ffn& f, char* base) {
  Carver c{base};
  FfnFwdWs w;
  w.x = rows_of(f.x, f.x_st, f.N, f.D, c);
  w.gu = rows_of(f.gate_up, f.gate_up_st, 2 * (int64_t)f.I, f.D, c);
  w.down = rows_of(f.down, f.down_st, f.O, f.I, c);
  w.a = c.take<bf>(a_bytes(f));
  w.parts = c.take<char>(most(plan_gate_up(f).parts, plan_down(f).parts));
  w.bytes = c.off + 256;
  return w;
}

struct FfnBwdWs { Rows x, gu, down, dy; bf* dgu; void* parts; size_t bytes; };
FfnBwdWs carve_ffn_bwd(const sd_ffn& f, const void* dy, int64_t dy_st, char* base) {
  Carver c{base};
  FfnBwdWs w;
  w.x = rows_of(f.x, f.x_st, f.N, f.D, c);
  w.gu = rows_of(f.gate_up, f.gate_up_st, 2 * (int64_t)f.I, f.D, c);
  w.down = rows_of(f.down, f.down_st, f.O, f.I, c);
  w.dy = rows_of(dy, dy_st, f.N, f.O, c);
  w.dgu = c.take<bf>((size_t)f.N * up(2 * (int64_t)f.I, 8) * 2);
  w.parts = c.take<char>(most(most(plan_da(f).parts, plan_dx(f).parts),
                              most(plan_dgate_up(f).parts, plan_ddown(f).parts)));
  w.bytes = c.off + 256;
  return w;
}

// Widths up to 2^19 (rows up to 4 times as far apart) keep a tile's offsets within 31 bits; a
// launch takes less than 2^23 tiles (2^32 threads).
constexpr int64_t kMaxWidth = 1 << 19;
bool ffn_shape_ok(const sd_ffn* f) {
  if (!f || f->N <= 0 || f->D <= 0 || f->I <= 0 || f->O <= 0 || f->N >= (int64_t(1) << 30)) return false;
  int64_t w = f->D > f->O ? f->D : f->O;
  if (f->I > w) w = f->I;
  return w <= kMaxWidth && (f->N / 128 + 1) * (2 * w / 128 + 1) < (1 << 23) &&
         (2 * w / 128 + 1) * (w / 128 + 1) < (1 << 20);
}
bool ffn_args_ok(const sd_ffn* f) {
  return f->x && f->gate_up && f->down && f->x_st >= f->D && f->gate_up_st >= f->D && f->down_st >= f->I &&
         (f->N == 1 || f->x_st <= 4 * kMaxWidth) && f->gate_up_st <= 4 * kMaxWidth && f->down_st <= 4 * kMaxWidth;
}

}  // namespace
}  // namespace sd

using namespace sd;

extern "C" {

int sd_product_plan(int64_t M, int64_t N, int64_t k_bytes, int plan[3]) {
  if (M <= 0 || N <= 0 || k_bytes <= 0 || M > INT32_MAX || N > INT32_MAX || k_bytes > INT32_MAX) return SD_ERR_SHAPE;
  if (!plan) return SD_ERR_ARG;
  const GemmPlan p = plan_gemm(M, N, (k_bytes + 127) / 128);
  plan[0] = p.tile; plan[1] = p.whole; plan[2] = p.workers;
  return SD_OK;
}

size_t sd_ffn_saved_bytes(const sd_ffn* f) {
  if (!ffn_shape_ok(f)) return 0;
  return saved_blocks_bytes(*f) + a_bytes(*f);
}
size_t sd_ffn_fwd_workspace_bytes(const sd_ffn* f) {
  return ffn_shape_ok(f) ? carve_ffn_fwd(*f, nullptr).bytes : 0;
}
size_t sd_ffn_bwd_workspace_bytes(const sd_ffn* f, const void* dy, int64_t dy_st) {
  return ffn_shape_ok(f) ? carve_ffn_bwd(*f, dy, dy_st, nullptr).bytes : 0;
}

int sd_ffn_fwd(const sd_ffn* f, void* y, void* saved, void* workspace, size_t workspace_bytes,
               void* stream) {
  if (!ffn_shape_ok(f)) return SD_ERR_SHAPE;
  if (!ffn_args_ok(f) || !y || !workspace || ((uintptr_t)saved & 31)) return SD_ERR_ARG;
  const FfnFwdWs w = carve_ffn_fwd(*f, (char*)up((int64_t)(uintptr_t)workspace, 256));
  if (workspace_bytes < w.bytes) return SD_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  if (!saved && few(*f)) {
    if (f->N <= 16) few_tokens<1>(*f, w.a, up(f->I, 8), y, st);
    else few_tokens<2>(*f, w.a, up(f->I, 8), y, st);
    return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
  }
  pack(w.x, f->x, f->x_st, st);
  pack(w.gu, f->gate_up, f->gate_up_st, st);
  pack(w.down, f->down, f->down_st, st);
  const int64_t la = up(f->I, 8);
  bf* a = saved ? (bf*)((char*)saved + saved_blocks_bytes(*f)) : w.a;
  GemmArgs g{};
  g.parts = w.parts;
  g.A = w.x.op(); g.B = w.gu.op();
  const GemmOperand second = w.gu.op(f->I, f->I);
  g.B.p2 = second.p; g.B.bytes2 = second.bytes;
  g.M = f->N; g.N = f->I; g.kbytes = (int)up(f->D, 8) * 2; g.steps = (int)steps_of(f->D);
  const FfnSaved s = saved ? carve_saved(*f, saved) : FfnSaved{nullptr, nullptr, 0};
  product<false, false, true>("k_ffn_gate_up", "k_ffn_gate_up_join", g, plan_gate_up(*f),
                              EpiGateUp(out_bf(a, la), s, f->N, f->I), st);
  g.A = Rows{a, la, f->N, (int)la, true}.op(); g.B = w.down.op();
  g.N = f->O; g.kbytes = (int)la * 2; g.steps = (int)steps_of(f->I);
  product<false, false, false>("k_ffn_down", "k_ffn_down_join", g, plan_down(*f),
                               EpiBf(out_bf(y, f->O), f->N, f->O), st);
  return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
}

int sd_ffn_bwd(const sd_ffn* f, const void* saved, const void* dy, int64_t dy_st, void* dx,
               void* dgate_up, void* ddown, void* workspace, size_t workspace_bytes,
               void* stream) {
  if (!ffn_shape_ok(f)) return SD_ERR_SHAPE;
  if (!ffn_args_ok(f) || !saved || !dy || dy_st < f->O || (f->N > 1 && dy_st > 4 * kMaxWidth) || !workspace ||
      ((uintptr_t)saved & 31))
    return SD_ERR_ARG;
  const FfnBwdWs w = carve_ffn_bwd(*f, dy, dy_st, (char*)up((int64_t)(uintptr_t)workspace, 256));
  if (workspace_bytes < w.bytes) return SD_ERR_WORKSPACE;
  hipStream_t st = (hipStream_t)stream;
  const int64_t I = f->I, I2 = 2 * I, la = up(I, 8), lg = up(I2, 8);
  pack(w.dy, dy, dy_st, st);
  pack(w.down, f->down, f->down_st, st);
  const bf* a = (const bf*)((const char*)saved + saved_blocks_bytes(*f));
  GemmArgs g{};
  g.parts = w.parts;
  // da[n,i] = sum_o dy[n,o] Wd[o,i]
  g.A = w.dy.op(); g.B = w.down.op();
  g.M = f->N; g.N = I; g.kbytes = (int)up(f->O, 8) * 2; g.steps = (int)steps_of(f->O);
  const EpiDact e(out_bf(w.dgu, lg), out_bf(w.dgu + I, lg), carve_saved(*f, (void*)saved), f->N, I);
  product<false, true, false>("k_ffn_da", "k_ffn_da_join", g, plan_da(*f), e, st);
  const Rows dgu{w.dgu, lg, f->N, (int)lg, true};
  if (dx) {
    pack(w.gu, f->gate_up, f->gate_up_st, st);
    g.A = dgu.op(); g.B = w.gu.op();
    g.N = f->D; g.kbytes = (int)lg * 2; g.steps = (int)steps_of(I2);
    product<false, true, false>("k_ffn_dx", "k_ffn_dx_join", g, plan_dx(*f), EpiBf(out_bf(dx, f->D), f->N, f->D), st);
  }
  g.steps = (int)steps_of(f->N);
  if (dgate_up) {
    pack(w.x, f->x, f->x_st, st);
    g.A = dgu.op(); g.B = w.x.op();
    g.M = I2; g.N = f->D;
    product<true, true, false>("k_ffn_dgate_up", "k_ffn_dgate_up_join", g, plan_dgate_up(*f),
                               EpiBf(out_bf(dgate_up, f->D), I2, f->D), st);
  }
  if (ddown) {
    g.A = w.dy.op(); g.B = Rows{a, la, f->N, (int)la, true}.op();
    g.M = f->O; g.N = I;
    product<true, true, false>("k_ffn_ddown", "k_ffn_ddown_join", g, plan_ddown(*f),
                               EpiBf(out_bf(ddown, I), f->O, I), st);
  }
  return hipGetLastError() == hipSuccess ? SD_OK : SD_ERR_LAUNCH;
}

}  // extern "C"
