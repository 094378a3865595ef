// Gated linear recurrence: a recurrent layer whose step has no product with the state, so that a sequence is a scan.
//   u[t] = (z | n | o) pre-activations, z' = sigmoid(z), n' = tanh(n), o' = sigmoid(o)   (2 gates: o' = 1)
//   h[t] = z' h[t-1] + (1 - z') n',   y[t] = o' h[t]
// Row b walks its own steps: t >= len[b] carries the state (y = 0, no gradient); `reverse` walks t downwards.
//
// Every channel (b, j) is a scan of the maps h -> a h + x, and two maps compose into one of the same form:
// (a2, x2) after (a1, x1) = (a1 a2, a2 x1 + x2).  The backward pass is the same scan from the other end,
//   delta[t] = dy[t] o' + c,   c -> z' delta[t]      (c -> a c + z' dy o': the same a),
// and it rebuilds h from the state saved once per 64 steps instead of reading a saved h[t] (which 16-bit
// storage would have to round): the backward pass reads u and dy and writes du, nothing else of that size.
//
// A block owns 64*VW channels; its waves each hold LR_C consecutive steps of those channels in registers, exchange
// their maps through LDS, and finish with the carry they get: one read of u, whatever the length.  Where the
// channels alone are too few blocks for 256 CUs, the time axis is cut into segments: a first launch computes every
// segment's map (z and n are read twice then), and a block starts from the composition of the segments before it.
// The state, the maps and all sums are fp32 for every storage type.
#include "common.hpp"
#include "misc.hpp"
#include "dtype.hpp"

namespace cvae {

constexpr int LR_C = 8;           // steps a wave holds in registers
constexpr int LR_W = 8;           // waves of a block at most: LR_C * LR_W steps (64) between saved states

struct LinRnnArgs {
  int T, B, H, gates, reverse;
  long n;                         // B * H channels
  const void* u; const float* h0; const int64_t* len;
  void* y; float* h_last;
  float* bounds;                  // [ceil(T / 64)][n] state before steps 0, 64, ... (in walking order)
  const void* dy; const float* dlast;
  void* du; float* dh0;
  float* agg;                     // [nseg][2][n] maps of the segments (nseg > 1)
  int nseg, seg;                  // segments and their steps (a multiple of 64)
};

// sigmoid(x) and 1 - sigmoid(x) (1 - z is formed from e^-|x|, not by subtraction: forget gates near 1 decide how much enters a
// long-lived state).  The larger of the two is good to ~2 ulp.  The smaller one is e^-|x| nearly, and as the exponent is rounded
// before it is raised, off by up to (2 + |x|) 2^-24 of itself: 16-bit storage stops there, as |x| 2^-24 is nothing beside what its
// own rounding of x does.  fp32 storage takes the rounding back: with t = |x| log2 e as rounded, e^-|x| = 2^-t e^-(|x| - t ln 2),
// ~2 ulp.  (r is a NaN at an infinity, where 2^-t = 0 has the last word.)  For 16-bit types that would be 650 us in place of 635
// for both passes of 2000 x 32 x 2048.
template <typename T> __device__ __forceinline__ void sigmoid_pair(float x, float& s, float& c) {
  const float a = fabsf(x), t = 1.4426950408889634f * a;
  float e = __builtin_amdgcn_exp2f(-t);
  if (sizeof(T) == 4) {
    const float r = fminf(fmaf(t, 1.9046542999577679e-9f, fmaf(t, -0.693147182464599609f, a)), 1.0f);   // -ln 2 in two parts
    e = fmaf(-r, e, e);
  }
  const float big = __builtin_amdgcn_rcpf(1.0f + e), small = e * big;
  s = x >= 0.f ? big : small;
  c = x >= 0.f ? small : big;
}
// the output gate: sigmoid(x) to the same bounds
template <typename T> __device__ __forceinline__ float sigmoid_of(float x) {
  if (sizeof(T) != 4) return sigmoid_fast(x);
  float s, c;
  sigmoid_pair<T>(x, s, c);
  return s;
}
// tanh: its series to x^9 below 0.3 (next term < 6e-8 relative), else from exp (1 - 2 / (1 + e^2x) keeps only an
// absolute 1e-7, too little near zero)
__device__ __forceinline__ float tanh_full(float x) {
  const float q = x * x;
  const float p = x * fmaf(q, fmaf(q, fmaf(q, fmaf(q, 62.f / 2835.f, -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
  return fabsf(x) < 0.3f ? p : tanh_fast(x);
}

template <typename T, int VW> __device__ __forceinline__ Packed<T, VW> ld(const T* p) {
  return *reinterpret_cast<const Packed<T, VW>*>(p);
}

// where a lane's channels sit, and which of its steps are live
template <int VW> struct Lane {
  long c;            // first channel (b * H + j)
  bool valid;
  int base, hbase;   // offset of (b, j) inside a step of u / of y (below 2^31: checked by the launchers)
  int len;
  __device__ Lane(const LinRnnArgs& p, int lane) {
    c = ((long)blockIdx.x * 64 + lane) * VW;
    valid = c < p.n;
    if (!valid) c = 0;
    const long b = c / p.H, j = c - b * p.H;
    base = (int)(b * p.gates * p.H + j);
    hbase = (int)c;
    long l = p.len ? p.len[b] : (long)p.T;
    len = (int)(l < 0 ? 0 : (l > p.T ? p.T : l));
  }
};

// step s in walking order -> time index; rows past their length read their last live row instead (in cache by then)
__device__ __forceinline__ int time_of(const LinRnnArgs& p, int s) { return p.reverse ? p.T - 1 - s : s; }
__device__ __forceinline__ int clamp_time(int t, int len, int T) {
  t = t < len ? t : len - 1;
  return t < 0 ? 0 : (t >= T ? T - 1 : t);
}

// state (or backward carry) that enters segment `seg`: the maps of the segments on the way there, composed by the
// block's waves in slices and joined through LDS.  `back`: segments are passed from the last one down.
template <int VW>
__device__ __forceinline__ void enter_segment(const LinRnnArgs& p, const Lane<VW>& L, int seg, bool back, int wave,
                                              int nw, int lane, float (*lds)[2][64 * VW], float (&carry)[VW]) {
  const int count = back ? p.nseg - 1 - seg : seg;
  const int per = (count + nw - 1) / nw;
  float a[VW], x[VW];
#pragma unroll
  for (int v = 0; v < VW; ++v) { a[v] = 1.f; x[v] = 0.f; }
  const int i0 = wave * per, i1 = min(count, i0 + per);
#pragma unroll 4
  for (int i = i0; i < i1; ++i) {
    const long s = back ? p.nseg - 1 - i : i;
    const float* g = p.agg + s * 2 * p.n + L.c;
#pragma unroll
    for (int v = 0; v < VW; ++v) {
      const float a2 = g[v], x2 = g[p.n + v];
      x[v] = fmaf(a2, x[v], x2);
      a[v] *= a2;
    }
  }
#pragma unroll
  for (int v = 0; v < VW; ++v) { lds[wave][0][lane * VW + v] = a[v]; lds[wave][1][lane * VW + v] = x[v]; }
  __syncthreads();
  for (int w = 0; w < nw; ++w)
#pragma unroll
    for (int v = 0; v < VW; ++v) carry[v] = fmaf(lds[w][0][lane * VW + v], carry[v], lds[w][1][lane * VW + v]);
  __syncthreads();
}

// What a wave finds in its LR_C steps: every lane inside its row (addresses are then one scalar row pointer plus a lane
// offset, nothing is masked), no lane (nothing is read), or a mixture.  The same for all lanes of the wave.
enum Steps { ST_FULL, ST_MIXED, ST_DEAD };
template <int VW> __device__ __forceinline__ Steps steps_of(const LinRnnArgs& p, const Lane<VW>& L, int w0, int w1) {
  if (w0 >= w1) return ST_DEAD;
  const int ta = time_of(p, w0), tb = time_of(p, w1 - 1), lo = ta < tb ? ta : tb, hi = ta < tb ? tb : ta;
  if (w1 - w0 == LR_C && __all(hi < L.len)) return ST_FULL;
  return __any(lo < L.len) ? ST_MIXED : ST_DEAD;
}
// rows of steps w0 .. w0 + LR_C of `src` (a lane's channels at `off` of a step): where not all are live, a step past a
// row's end reads the row's last live step instead (in cache by then) and is masked by its reader
template <typename T, int VW>
__device__ __forceinline__ void load_steps(const LinRnnArgs& p, const Lane<VW>& L, bool full, const void* src,
                                           long step, int off, int w0, Packed<T, VW> (&r)[LR_C]) {
  const T* q = static_cast<const T*>(src);
  if (full) {
#pragma unroll
    for (int i = 0; i < LR_C; ++i) r[i] = ld<T, VW>(q + (long)time_of(p, w0 + i) * step + (unsigned)off);
  } else {
#pragma unroll
    for (int i = 0; i < LR_C; ++i) r[i] = ld<T, VW>(q + (long)clamp_time(time_of(p, w0 + i), L.len, p.T) * step + off);
  }
}

// The maps of every segment.  BACK: of the backward carry (z, o, dy), else of the state (z, n).  Only where channels are
// few: 8192 steps x 2 rows x 1000 bf16, 25 us before the pass itself (36 forward, 51 backward).
template <typename T, int VW, int G, bool BACK>
__global__ __launch_bounds__(64 * LR_W) void linrnn_maps_kernel(LinRnnArgs p) {
  __shared__ float lds[LR_W][2][64 * VW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const Lane<VW> L(p, lane);
  const int seg = blockIdx.y;
  const int s0 = seg * p.seg, s1 = min(p.T, s0 + p.seg);
  const int per = ((s1 - s0 + nw - 1) / nw + LR_C - 1) / LR_C * LR_C;
  const int w0 = s0 + wave * per, w1 = min(s1, w0 + per);
  const long ustep = (long)p.B * G * p.H;
  float a[VW], x[VW];
#pragma unroll
  for (int v = 0; v < VW; ++v) { a[v] = 1.f; x[v] = 0.f; }
  const int rounds = w1 > w0 ? (w1 - w0 + LR_C - 1) / LR_C : 0;
  for (int r = 0; r < rounds; ++r) {
    const int c0 = w0 + (BACK ? rounds - 1 - r : r) * LR_C, c1 = min(w1, c0 + LR_C);
    const Steps st = steps_of<VW>(p, L, c0, c1);
    if (st == ST_DEAD) continue;
    Packed<T, VW> rz[LR_C], rn[LR_C], ro[LR_C];
    load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, L.base, c0, rz);
    if (BACK) {
      load_steps<T, VW>(p, L, st == ST_FULL, p.dy, p.n, L.hbase, c0, rn);
      if (G == 3) load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, L.base + 2 * p.H, c0, ro);
    } else {
      load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, L.base + p.H, c0, rn);
    }
#pragma unroll
    for (int k = 0; k < LR_C; ++k) {
      const int i = BACK ? LR_C - 1 - k : k;
      const bool live = st == ST_FULL || (c0 + i < c1 && time_of(p, c0 + i) < L.len);
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        float z, c, in;
        sigmoid_pair<T>(rz[i].f(v), z, c);
        if (BACK) in = z * (G == 3 ? rn[i].f(v) * sigmoid_of<T>(ro[i].f(v)) : rn[i].f(v));
        else in = c * tanh_full(rn[i].f(v));
        if (live) { x[v] = fmaf(z, x[v], in); a[v] *= z; }
      }
    }
  }
#pragma unroll
  for (int v = 0; v < VW; ++v) { lds[wave][0][lane * VW + v] = a[v]; lds[wave][1][lane * VW + v] = x[v]; }
  __syncthreads();
  if (wave == 0 && L.valid) {
    float* g = p.agg + (long)seg * 2 * p.n + L.c;
#pragma unroll
    for (int v = 0; v < VW; ++v) {
      float A = 1.f, X = 0.f;
      for (int i = 0; i < nw; ++i) {
        const int w = BACK ? nw - 1 - i : i;
        const float a2 = lds[w][0][lane * VW + v], x2 = lds[w][1][lane * VW + v];
        X = fmaf(a2, X, x2);
        A *= a2;
      }
      g[v] = A;
      g[p.n + v] = X;
    }
  }
}

// Bound by memory, and by its two sigmoids and the tanh beside it: u is read once, y written once.  2000 steps x 32 rows x
// 2048, three gates, bf16, ragged: 236 us with 0.59 GB read and 0.27 written, which is what live steps need and the zeros behind
// them, 3.7 TB/s by the memory counters (a large copy: 4.7; without the tanh's series 215 us, without any exponential 197);
// 110 x 32 x 512 fp32 11 us.  Asking for the next round's rows early cost registers,
// hence blocks on a CU: 292 us.
template <typename T, int VW, int G>
__global__ __launch_bounds__(64 * LR_W) void linrnn_fwd_kernel(LinRnnArgs p) {
  __shared__ float lds[2][LR_W][2][64 * VW];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const Lane<VW> L(p, lane);
  const int seg = blockIdx.y;
  const int s0 = seg * p.seg, s1 = min(p.T, s0 + p.seg);
  T* y = static_cast<T*>(p.y);
  const long ustep = (long)p.B * G * p.H;
  float carry[VW];                                // the state before this block's next 64 steps, in every wave
#pragma unroll
  for (int v = 0; v < VW; ++v) carry[v] = p.h0 ? p.h0[L.c + v] : 0.f;
  if (seg > 0) enter_segment<VW>(p, L, seg, false, wave, nw, lane, lds[0], carry);
  int buf = 0;
  for (int sc = s0; sc < s1; sc += LR_C * nw, buf ^= 1) {
    const int w0 = sc + wave * LR_C, w1 = min(s1, w0 + LR_C);
    const Steps st = steps_of<VW>(p, L, w0, w1);
    float a[LR_C][VW], x[LR_C][VW], A[VW], X[VW];
    Packed<T, VW> ro[LR_C];
#pragma unroll
    for (int v = 0; v < VW; ++v) { A[v] = 1.f; X[v] = 0.f; }
    if (st != ST_DEAD) {
      Packed<T, VW> rz[LR_C], rn[LR_C];
      load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, L.base, w0, rz);
      load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, L.base + p.H, w0, rn);
      if (G == 3) load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, L.base + 2 * p.H, w0, ro);
#pragma unroll
      for (int i = 0; i < LR_C; ++i)
#pragma unroll
        for (int v = 0; v < VW; ++v) {
          float c;
          sigmoid_pair<T>(rz[i].f(v), a[i][v], c);
          x[i][v] = c * tanh_full(rn[i].f(v));
        }
      if (st == ST_MIXED) {
#pragma unroll
        for (int i = 0; i < LR_C; ++i)
          if (!(w0 + i < w1 && time_of(p, w0 + i) < L.len)) {
#pragma unroll
            for (int v = 0; v < VW; ++v) { a[i][v] = 1.f; x[i][v] = 0.f; }
          }
      }
#pragma unroll
      for (int i = 0; i < LR_C; ++i)
#pragma unroll
        for (int v = 0; v < VW; ++v) { X[v] = fmaf(a[i][v], X[v], x[i][v]); A[v] *= a[i][v]; }
    }
    if (p.bounds && wave == 0 && L.valid && sc % (LR_C * LR_W) == 0) {
#pragma unroll
      for (int v = 0; v < VW; ++v) p.bounds[(long)(sc / (LR_C * LR_W)) * p.n + L.c + v] = carry[v];
    }
#pragma unroll
    for (int v = 0; v < VW; ++v) { lds[buf][wave][0][lane * VW + v] = A[v]; lds[buf][wave][1][lane * VW + v] = X[v]; }
    __syncthreads();                              // one barrier a round: the other buffer is written meanwhile
    float h[VW];
    for (int w = 0; w < nw; ++w) {
      if (w == wave) {
#pragma unroll
        for (int v = 0; v < VW; ++v) h[v] = carry[v];
      }
#pragma unroll
      for (int v = 0; v < VW; ++v)
        carry[v] = fmaf(lds[buf][w][0][lane * VW + v], carry[v], lds[buf][w][1][lane * VW + v]);
    }
    if (st == ST_DEAD) {
      for (int s = w0; s < w1; ++s)
        if (L.valid) *reinterpret_cast<Packed<T, VW>*>(y + (long)time_of(p, s) * p.n + (unsigned)L.hbase) = Packed<T, VW>{};
      continue;
    }
#pragma unroll
    for (int i = 0; i < LR_C; ++i) {
      const int s = w0 + i, t = time_of(p, s);
      Packed<T, VW> out;
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        h[v] = fmaf(a[i][v], h[v], x[i][v]);
        out.set(v, G == 3 ? sigmoid_of<T>(ro[i].f(v)) * h[v] : h[v]);
      }
      if (st == ST_MIXED && t >= L.len) out = Packed<T, VW>{};
      if (s < w1 && L.valid) *reinterpret_cast<Packed<T, VW>*>(y + (long)t * p.n + (unsigned)L.hbase) = out;
    }
  }
  if (seg == p.nseg - 1 && wave == 0 && L.valid) {
#pragma unroll
    for (int v = 0; v < VW; ++v) p.h_last[L.c + v] = carry[v];
  }
}

// Two scans from opposite ends in one pass over u and dy: the state again from the one saved every 64 steps, the carry
// downwards.  Four waves on a SIMD (two blocks on a CU): 128 registers.  2000 x 32 x 2048, three gates, bf16, ragged: 377 us with
// 0.80 GB read and 0.79 written, 4.2 TB/s by the memory counters (without that bound on the registers 702 us; with the addresses
// of a round kept through all of them, and 21 values in private memory for it, 422).
template <typename T, int VW, int G>
__global__ __launch_bounds__(64 * LR_W, 4) void linrnn_bwd_kernel(LinRnnArgs p) {
  __shared__ float lds[2][LR_W][3][64 * VW];      // A (both directions), X of the state, X of the carry
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nw = blockDim.x >> 6;
  const Lane<VW> L(p, lane);
  const int seg = blockIdx.y;
  const int s0 = seg * p.seg, s1 = min(p.T, s0 + p.seg);
  T* du = static_cast<T*>(p.du);
  const long ustep = (long)p.B * G * p.H;
  float carry[VW];                                // gradient of the state after this block's steps
#pragma unroll
  for (int v = 0; v < VW; ++v) carry[v] = p.dlast ? p.dlast[L.c + v] : 0.f;
  if (seg < p.nseg - 1)
    enter_segment<VW>(p, L, seg, true, wave, nw, lane, reinterpret_cast<float (*)[2][64 * VW]>(&lds[0][0][0][0]), carry);
  int buf = 0;
  const int R = LR_C * nw;                        // steps of a round: 64, or the whole of a shorter sequence
  for (int sc = s0 + (s1 - s0 + R - 1) / R * R - R; sc >= s0; sc -= R, buf ^= 1) {   // (no steps: no round)
    const int w0 = sc + wave * LR_C, w1 = min(s1, w0 + LR_C);
    const Steps st = steps_of<VW>(p, L, w0, w1);
    // (hides that these are the same every round: the addresses made of them, kept in registers, would push others into memory)
    int ubase = L.base, ybase = L.hbase;
    asm volatile("" : "+v"(ubase), "+v"(ybase));
    float hin[VW];
#pragma unroll
    for (int v = 0; v < VW; ++v) hin[v] = p.bounds[(long)(sc / (LR_C * LR_W)) * p.n + L.c + v];
    float z[LR_C][VW], c[LR_C][VW], n[LR_C][VW], o[LR_C][VW], A[VW], X[VW], Q[VW];
    Packed<T, VW> rd[LR_C];
#pragma unroll
    for (int v = 0; v < VW; ++v) { A[v] = 1.f; X[v] = 0.f; Q[v] = 0.f; }
    if (st != ST_DEAD) {
      Packed<T, VW> rz[LR_C], rn[LR_C], ro[LR_C];
      load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, ubase, w0, rz);
      load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, ubase + p.H, w0, rn);
      if (G == 3) load_steps<T, VW>(p, L, st == ST_FULL, p.u, ustep, ubase + 2 * p.H, w0, ro);
      load_steps<T, VW>(p, L, st == ST_FULL, p.dy, p.n, ybase, w0, rd);
#pragma unroll
      for (int i = 0; i < LR_C; ++i)
#pragma unroll
        for (int v = 0; v < VW; ++v) {
          sigmoid_pair<T>(rz[i].f(v), z[i][v], c[i][v]);
          n[i][v] = tanh_full(rn[i].f(v));
          o[i][v] = G == 3 ? sigmoid_of<T>(ro[i].f(v)) : 1.f;
        }
      if (st == ST_MIXED) {
#pragma unroll
        for (int i = 0; i < LR_C; ++i)
          if (!(w0 + i < w1 && time_of(p, w0 + i) < L.len)) {
#pragma unroll
            for (int v = 0; v < VW; ++v) { z[i][v] = 1.f; c[i][v] = 0.f; n[i][v] = 0.f; o[i][v] = 0.f; }
            rd[i] = Packed<T, VW>{};
          }
      }
#pragma unroll
      for (int i = 0; i < LR_C; ++i)
#pragma unroll
        for (int v = 0; v < VW; ++v) { X[v] = fmaf(z[i][v], X[v], c[i][v] * n[i][v]); A[v] *= z[i][v]; }
#pragma unroll
      for (int i = LR_C - 1; i >= 0; --i)
#pragma unroll
        for (int v = 0; v < VW; ++v) Q[v] = z[i][v] * (G == 3 ? fmaf(rd[i].f(v), o[i][v], Q[v]) : rd[i].f(v) + Q[v]);
    }
#pragma unroll
    for (int v = 0; v < VW; ++v) {
      lds[buf][wave][0][lane * VW + v] = A[v];
      lds[buf][wave][1][lane * VW + v] = X[v];
      lds[buf][wave][2][lane * VW + v] = Q[v];
    }
    __syncthreads();
    for (int w = 0; w < wave; ++w)                // the state this wave starts from
#pragma unroll
      for (int v = 0; v < VW; ++v)
        hin[v] = fmaf(lds[buf][w][0][lane * VW + v], hin[v], lds[buf][w][1][lane * VW + v]);
    float d[VW];
    for (int w = nw - 1; w >= 0; --w) {           // the carry that reaches it, and the one that leaves the round
      if (w == wave) {
#pragma unroll
        for (int v = 0; v < VW; ++v) d[v] = carry[v];
      }
#pragma unroll
      for (int v = 0; v < VW; ++v)
        carry[v] = fmaf(lds[buf][w][0][lane * VW + v], carry[v], lds[buf][w][2][lane * VW + v]);
    }
    if (!du) continue;                            // (not wanted: the carry alone goes on, to dh0)
    if (st == ST_DEAD) {
      for (int s = w0; s < w1; ++s)
        if (L.valid) {
          T* q = du + (long)time_of(p, s) * ustep + (unsigned)ubase;
#pragma unroll
          for (int g = 0; g < G; ++g) *reinterpret_cast<Packed<T, VW>*>(q + g * p.H) = Packed<T, VW>{};
        }
      continue;
    }
    float hp[LR_C + 1][VW];                       // h before each step
#pragma unroll
    for (int v = 0; v < VW; ++v) hp[0][v] = hin[v];
#pragma unroll
    for (int i = 0; i < LR_C; ++i)
#pragma unroll
      for (int v = 0; v < VW; ++v) hp[i + 1][v] = fmaf(z[i][v], hp[i][v], c[i][v] * n[i][v]);
#pragma unroll
    for (int i = LR_C - 1; i >= 0; --i) {
      const int s = w0 + i, t = time_of(p, s);
      Packed<T, VW> gz, gn, go;
#pragma unroll
      for (int v = 0; v < VW; ++v) {
        const float dyo = rd[i].f(v) * o[i][v], zz = z[i][v], cc = c[i][v], nn = n[i][v];
        const float delta = (G == 3 ? dyo : rd[i].f(v)) + d[v];
        const float into = delta * cc;
        gz.set(v, into * (hp[i][v] - nn) * zz);
        gn.set(v, into * fmaf(-nn, nn, 1.f));
        if (G == 3) go.set(v, dyo * hp[i + 1][v] * (1.f - o[i][v]));
        d[v] = zz * delta;
      }
      if (st == ST_MIXED && t >= L.len) gz = gn = go = Packed<T, VW>{};   // exact zeros, whatever the carry holds
      if (s < w1 && L.valid) {
        T* q = du + (long)t * ustep + (unsigned)ubase;
        *reinterpret_cast<Packed<T, VW>*>(q) = gz;
        *reinterpret_cast<Packed<T, VW>*>(q + p.H) = gn;
        if (G == 3) *reinterpret_cast<Packed<T, VW>*>(q + 2 * p.H) = go;
      }
    }
  }
  if (seg == 0 && wave == 0 && L.valid && p.dh0) {
#pragma unroll
    for (int v = 0; v < VW; ++v) p.dh0[L.c + v] = carry[v];
  }
}

// One decoding step: nothing but the element-wise maths, one lane per VW channels.  Launch and one memory latency: 2.3 us for
// 4 rows x 512 fp32, 4.4 for 512 x 2048 bf16 (12 MB, from the caches).
template <typename T, int VW>
__global__ __launch_bounds__(256) void linrnn_step_kernel(LinRnnArgs p) {
  const long c = ((long)blockIdx.x * 256 + threadIdx.x) * VW;
  if (c >= p.n) return;
  const long b = c / p.H, j = c - b * p.H;
  const T* q = static_cast<const T*>(p.u) + b * p.gates * p.H + j;
  const Packed<T, VW> rz = ld<T, VW>(q), rn = ld<T, VW>(q + p.H);
  Packed<T, VW> ro = {}, out;
  if (p.gates == 3) ro = ld<T, VW>(q + 2 * p.H);
  float h[VW];
#pragma unroll
  for (int v = 0; v < VW; ++v) h[v] = p.h0 ? p.h0[c + v] : 0.f;
#pragma unroll
  for (int v = 0; v < VW; ++v) {
    float z, k, o = 1.f, oc;
    sigmoid_pair<T>(rz.f(v), z, k);
    h[v] = fmaf(z, h[v], k * tanh_full(rn.f(v)));
    if (p.gates == 3) sigmoid_pair<T>(ro.f(v), o, oc);
    out.set(v, o * h[v]);
    p.h_last[c + v] = h[v];
  }
  *reinterpret_cast<Packed<T, VW>*>(static_cast<T*>(p.y) + c) = out;
}

// ---------------------------------------------------------------------------------------------- host side
static int lr_channels_per_block(int dtype, int H) { return 64 * ((dtype != DT_F32 && H % 2 == 0) ? 2 : 1); }
// segments of the time axis: enough blocks for two on every CU (8192 x 2000 channels bf16: forward 61 us with 512 blocks,
// 76 with 256, 62 with 1024), of no less than one round (64 steps) each
static void lr_plan(int dtype, int T, int B, int H, int* nseg, int* seg) {
  constexpr int R = LR_C * LR_W;
  const long cb = ((long)B * H + lr_channels_per_block(dtype, H) - 1) / lr_channels_per_block(dtype, H);
  long want = (512 + cb - 1) / (cb > 0 ? cb : 1);
  const long most = ((long)T + R - 1) / R;
  if (want > most) want = most;
  if (cb >= 256 || want < 1) want = 1;
  *seg = (int)((((long)T + want - 1) / want + R - 1) / R * R);
  if (*seg < R) *seg = R;
  *nseg = T > 0 ? cdiv(T, *seg) : 1;
}
long linrnn_bounds_floats(int T, int B, int H) { return (long)cdiv(T, LR_C * LR_W) * B * H; }
long linrnn_workspace_floats(int dtype, int T, int B, int H) {
  int nseg, seg;
  lr_plan(dtype, T, B, H, &nseg, &seg);
  return nseg > 1 ? 2L * nseg * B * H : 0;
}

template <typename T, int VW, int G> static int lr_launch(LinRnnArgs a, bool back, hipStream_t s) {
  const dim3 grid((unsigned)((a.n + 64 * VW - 1) / (64 * VW)), a.nseg);
  const int nw = a.T >= LR_C * LR_W ? LR_W : (a.T > 0 ? cdiv(a.T, LR_C) : 1);
  if (!back && a.T == 1 && !a.bounds && !a.len) {
    hipLaunchKernelGGL((linrnn_step_kernel<T, VW>), dim3((unsigned)((a.n + 256 * VW - 1) / (256 * VW))), dim3(256), 0, s, a);
    CVAE_LAUNCH_CHECK("linrnn_step_kernel");
    return 0;
  }
  if (a.nseg > 1) {
    if (back) hipLaunchKernelGGL((linrnn_maps_kernel<T, VW, G, true>), grid, dim3(64 * nw), 0, s, a);
    else hipLaunchKernelGGL((linrnn_maps_kernel<T, VW, G, false>), grid, dim3(64 * nw), 0, s, a);
    CVAE_LAUNCH_CHECK("linrnn_maps_kernel");
  }
  if (back) hipLaunchKernelGGL((linrnn_bwd_kernel<T, VW, G>), grid, dim3(64 * nw), 0, s, a);
  else hipLaunchKernelGGL((linrnn_fwd_kernel<T, VW, G>), grid, dim3(64 * nw), 0, s, a);
  CVAE_LAUNCH_CHECK("linrnn kernel");
  return 0;
}

template <typename T, int VW> static int lr_gates(const LinRnnArgs& a, bool back, hipStream_t s) {
  return a.gates == 3 ? lr_launch<T, VW, 3>(a, back, s) : lr_launch<T, VW, 2>(a, back, s);
}

static int lr_dispatch(int dtype, const LinRnnArgs& a, bool back, hipStream_t s) {
  // two channels a lane need rows that stay 4-byte aligned: an even H and operands on 4-byte boundaries
  const uintptr_t at = (uintptr_t)a.u | (uintptr_t)a.y | (uintptr_t)a.dy | (uintptr_t)a.du;
  const bool two = a.H % 2 == 0 && (at & 3) == 0;
  if (dtype == DT_F32) return lr_gates<float, 1>(a, back, s);
  if (dtype == DT_BF16) return two ? lr_gates<bf16_t, 2>(a, back, s) : lr_gates<bf16_t, 1>(a, back, s);
  return two ? lr_gates<f16_t, 2>(a, back, s) : lr_gates<f16_t, 1>(a, back, s);
}

static int lr_check(const char* what, int dtype, int gates, int T, int B, int H) {
  CVAE_REQUIRE(dtype >= DT_F32 && dtype <= DT_F16, "%s: dtype %d is none of 0 (fp32), 1 (bf16), 2 (fp16)", what, dtype);
  CVAE_REQUIRE(gates == 2 || gates == 3, "%s: gates must be 2 or 3, not %d", what, gates);
  CVAE_REQUIRE(T >= 0 && B >= 0 && H >= 0 && T < (1 << 30) && (int64_t)B * H <= (1LL << 28), "%s: bad shape T=%d B=%d H=%d",
               what, T, B, H);
  return 0;
}

int launch_linrnn_forward(int dtype, int gates, int reverse, int T, int B, int H, const void* u, const float* h0,
                          const int64_t* len, void* y, float* h_last, float* bounds, float* ws, hipStream_t s) {
  CVAE_TRY(lr_check("linrnn_forward", dtype, gates, T, B, H));
  if ((long)B * H == 0) return 0;
  CVAE_REQUIRE(h_last && (T == 0 || (u && y)), "linrnn_forward: null operand");
  LinRnnArgs a = {};
  a.T = T; a.B = B; a.H = H; a.gates = gates; a.reverse = reverse != 0; a.n = (long)B * H;
  a.u = u; a.h0 = h0; a.len = len; a.y = y; a.h_last = h_last; a.bounds = bounds; a.agg = ws;
  lr_plan(dtype, T, B, H, &a.nseg, &a.seg);
  CVAE_REQUIRE(a.nseg == 1 || ws, "linrnn_forward: null workspace");
  // every segment starts from h0, and the last one may end before another begins
  CVAE_REQUIRE(a.nseg == 1 || h_last != h0, "linrnn_forward: h_last may be h0 only where no workspace is needed");
  return lr_dispatch(dtype, a, false, s);
}

int launch_linrnn_backward(int dtype, int gates, int reverse, int T, int B, int H, const void* u, const int64_t* len,
                           const float* bounds, const void* dy, const float* dlast, void* du, float* dh0, float* ws,
                           hipStream_t s) {
  CVAE_TRY(lr_check("linrnn_backward", dtype, gates, T, B, H));
  if ((long)B * H == 0) return 0;
  if (!du && !dh0) return 0;
  CVAE_REQUIRE(T == 0 || (u && dy && bounds), "linrnn_backward: null operand");
  LinRnnArgs a = {};
  a.T = T; a.B = B; a.H = H; a.gates = gates; a.reverse = reverse != 0; a.n = (long)B * H;
  a.u = u; a.len = len; a.bounds = const_cast<float*>(bounds); a.dy = dy; a.dlast = dlast; a.du = du; a.dh0 = dh0;
  a.agg = ws;
  lr_plan(dtype, T, B, H, &a.nseg, &a.seg);
  CVAE_REQUIRE(a.nseg == 1 || ws, "linrnn_backward: null workspace");
  return lr_dispatch(dtype, a, true, s);
}

}  // namespace cvae
