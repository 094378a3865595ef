// Losses of projected logits S = X W^T + b over a large vocabulary, for fp32, bf16 and fp16 storage and any width E:
//   hard[n] = lse(S[n]) - S[n][target]                                   (softmax cross-entropy)
//   soft[n] = tau^2 sum_k p_k (log p_k - S[n][id_k] / tau + lse(S[n] / tau)),  p = softmax(teacher's top logits / tau)
// and their gradients.  The (rows, V) array is never formed: the forward pass folds 128 x 128 tiles of S into running
// (max, sum) pairs; the backward pass forms d loss / d S again in pieces of the vocabulary that stay in the chip's
// caches, and multiplies each piece with W and X before the next one is made.  Rows whose target is `pad` are dropped
// first (their loss and gradient are zero): everything below works on the compact list of live rows.
//
// Number format.  All four products run on v_mfma_f32_32x32x16_f16 with fp32 accumulation.  X and W are first laid out
// as images: a power-of-two scale brings the tensor's largest element to [2^13, 2^14), 16-bit inputs are then one fp16
// plane (exact: bf16 and fp16 have at most 11 significant bits; elements below 2^-28 of the largest lose bits, an
// absolute 2^-38 of it), fp32 inputs are two planes hi + lo (22 bits), multiplied as hi.lo + lo.hi + hi.hi, which drops
// at most 2^-22 of a product (bf16 planes would drop 2^-16).  The gradient's tile P = dS / s is stored the same way (s: the
// row's power of two above |dS|, carried by the other operand): one plane for bf16, whose own rounding is eight times
// fp16's half step of 2^-11; two planes for fp32, and for fp16, whose outputs' rounding one plane would double.
//
// What bounds it: 8 N E V operations (S twice, dX, dW; fp32 three times that) against reads of X and W and writes of their
// gradients, so from a few hundred rows on the matrix cores do, and beside them two exponentials an element and pass at small
// E.  Measured on live rows, forward and backward: 3650 rows x 1024 x 50000 bf16 1.68 ms (1.49 TFLOP, 0.89 PFLOP/s of
// useful work; a large library product runs at 1.38), 4815 x 200 x 50000 bf16 with 64 teacher entries at tau 2 0.73 ms.
//
// Image layout: rows of 128-byte pieces, one plane: 64 values, two planes: 32 hi values then 32 lo values.  A piece is
// what one row adds to a pipeline stage, so one loop serves both.  Rows are padded to 256 with zeros, columns to 64 (to
// 256 for 129 to 208 columns).
// Both orders that the products need are read from this one layout: rows along K with ds_read_b128, and K down the
// rows with ds_read_b64_tr_b16, which transposes on its way to the registers.
#include "common.hpp"
#include "misc.hpp"
#include "dtype.hpp"
#include "dx_splits.hpp"

namespace cvae {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s4 lds_s4;

constexpr int DT_TILE = 128;               // rows / columns of a tile, both ways
constexpr int DT_STAGE = 16384;            // bytes of one operand's stage: 128 rows x 128 bytes
constexpr int DT_AMAX = 512;               // partial maxima of |X| and |W|, each
constexpr int DT_CROWS = 256;              // rows of one count of the live-row scan
constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
constexpr int P_EXP = 13;                  // |P| <= 1 is stored times 2^13

struct DistillArgs {
  int N, T, R, B, E, V, K;
  int Np, Vp, Kp, Kg;                      // multiples of 256 for N and V, of 64 for E and E + 1
  float tau, itau;
  int two;                                 // tau != 1 and K > 0: a second normaliser
  const void* X; const void* W; const void* bias;
  const int64_t* eos; int64_t pad; int per;   // targets [B,T]; rows per sentence of sentence-major rows, else 0
  const int64_t* ids; const float* top;
  float* hard; float* soft;                // [N], in the workspace
  // kept for the backward pass
  int* counts; int scanned;                // live rows of every DT_CROWS rows, [cdiv(N, DT_CROWS) + 1]; or of all before them
  int* rows; int* inv; int* nlive; int* slive;   // slive[R]: the sentence has a live row
  float* amax; int* sexp;                  // [2][DT_AMAX]; [2] scale exponents of X and W
  _Float16* Ximg; _Float16* Wimg; float* b2;
  float* L1; float* L2; float* some;       // by live row: normalisers (base 2), 1 where the teacher lists anything
  float* pick; float* share;               // picked logits (base 2) and the teacher's share of them, [K + 1]
  float* part; long pplane;                // [3][splits][tiles of live rows][128]; floats of one
  int fvt, least;                          // vocabulary tiles of the forward walk, ranges an XCD takes at least
  // backward
  const float* ghard; const float* gsoft;  // [R]
  _Float16* Gimg; float* coef;             // s X image with a column of s; [3][Np]: a, b, s / gmax
  float* gmax; float* gpart;               // the largest |gradient| of a row; its partials (null: found in every block)
  _Float16* P; int v0, vc;                 // a range of the vocabulary: [vc NP / 64 pieces][Np rows][128 bytes]
  float* slab; int vfull, dwtiles;         // partial tiles of dX; words of a full range, and its tiles of dW
  void* dX; void* dW; void* db;
};

// row n = t R + r reads position (sentence, t): r % B, or r / (R / B) for sentence-major rows
__device__ __forceinline__ long position(const DistillArgs& p, int n) {
  const int t = n / p.R, r = n - t * p.R, b = p.per ? r / p.per : r % p.B;
  return (long)b * p.T + t;
}

// ------------------------------------------------------------------------------------------------- scales and images
// amax * 2^e in [2^13, 2^14), up to the largest float (e = -114); a tensor of less than 2^-97 altogether keeps e = 110, so that the
// powers that undo it stay floats
__device__ __forceinline__ int scale_exp(float amax) {
  if (!(amax > 0.f)) return 0;
  const int e = P_EXP - (int)floorf(log2f(amax));
  return e > 110 ? 110 : e;
}
// from a product of images to a base-2 logit (finite, so that a product of zero stays zero beside tensors of 2^64 and more)
__device__ __forceinline__ float unscale(const int* e) { return fminf(ldexpf(LOG2E, -(e[0] + e[1])), 3.0e38f); }
// largest finite magnitude of a tensor from its partials, by every thread of a block of 256
__device__ __forceinline__ float block_amax(const float* part, float* red) {
  static_assert(DT_AMAX == 512, "two partials a thread");
  float m = wave_max(fmaxf(part[threadIdx.x], part[threadIdx.x + 256]));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  m = 0.f;
  for (int i = 0; i < 4; ++i) m = fmaxf(m, red[i]);
  __syncthreads();
  return m;
}
// four elements at columns k .. k+3 of a row (zero past E), times 2^e, as fp16 planes
template <typename T> __device__ __forceinline__ void load4(const T* row, int k, int E, bool vec, float (&x)[4]) {
  if (vec && k + 3 < E) {
    const Packed<T, 4> r = *reinterpret_cast<const Packed<T, 4>*>(row + k);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = r.f(i);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = k + i < E ? (float)row[k + i] : 0.f;
  }
}
// x as one rounded fp32 value, whose two planes belong together: the compiler may form hi from x's last product or sum in one
// instruction that rounds once, and lo from x itself; where the two hi differ (one x in some 2^14), lo mends nothing
__device__ __forceinline__ void one_value(float& x) { asm("" : "+v"(x)); }
template <int NP> __device__ __forceinline__ long image_at(int k) { return NP == 1 ? k : (long)(k >> 5) * 64 + (k & 31); }
template <int NP> __device__ __forceinline__ void store4(_Float16* row, int k, const float (&x)[4]) {
  Packed<f16_t, 4> hi, lo;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    hi.set(i, x[i]);
    if (NP == 2) {
      const float r = x[i] - hi.f(i);
      lo.set(i, fabsf(x[i]) < 3.0e38f ? r : 0.f);                // an infinity has no remainder
    }
  }
  _Float16* q = row + image_at<NP>(k);
  *reinterpret_cast<Packed<f16_t, 4>*>(q) = hi;
  if (NP == 2) *reinterpret_cast<Packed<f16_t, 4>*>(q + 32) = lo;
}

// Live rows per DT_CROWS rows, zero losses, and (the blocks after those) partial maxima of |X| and |W|: one read of both, at
// the memory's rate (24 us for 110 MB).
template <typename T> __global__ __launch_bounds__(256) void dt_count_kernel(DistillArgs p, int nb) {
  __shared__ float red[4];
  if ((int)blockIdx.x < nb) {
    const int n = blockIdx.x * DT_CROWS + threadIdx.x;
    const bool live = n < p.N && p.eos[position(p, n)] != p.pad;
    if (n < p.N) {
      p.hard[n] = 0.f;
      if (p.K) p.soft[n] = 0.f;
      if (n < p.R) p.slive[n] = 0;
    }
    const int c = __popcll(__ballot(live));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = (float)c;
    __syncthreads();
    if (threadIdx.x == 0) p.counts[blockIdx.x] = (int)(red[0] + red[1] + red[2] + red[3]);
    return;
  }
  // (what stands in dropped rows does not set the scale of the others)
  const int b = blockIdx.x - nb, which = b / DT_AMAX, slot = b % DT_AMAX;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float m = 0.f;
  const auto take = [&](float v) { v = fabsf(v); m = v < INFINITY ? fmaxf(m, v) : m; };
  if (which) {
    const T* x = static_cast<const T*>(p.W);
    constexpr int VN = 16 / sizeof(T);
    const long n = (long)p.V * p.E;
    long head = (long)((16 - ((uintptr_t)x & 15)) & 15) / (long)sizeof(T);      // elements before a 16-byte boundary
    if (head > n) head = n;
    const long nv = (n - head) / VN, tail = head + nv * VN;
    if (slot == 0) {
      for (long i = threadIdx.x; i < head; i += 256) take((float)x[i]);
      for (long i = tail + threadIdx.x; i < n; i += 256) take((float)x[i]);
    }
    const Packed<T, VN>* xv = reinterpret_cast<const Packed<T, VN>*>(x + head);
#pragma unroll 4
    for (long i = (long)slot * 256 + threadIdx.x; i < nv; i += (long)DT_AMAX * 256) {
      const Packed<T, VN> r = xv[i];
#pragma unroll
      for (int j = 0; j < VN; ++j) take(r.f(j));
    }
  } else {
    const T* x = static_cast<const T*>(p.X);
    const bool vec = p.E % 4 == 0 && ((uintptr_t)x % (4 * sizeof(T))) == 0;
#pragma unroll 2
    for (int n = slot * 4 + wave; n < p.N; n += DT_AMAX * 4) {
      if (p.eos[position(p, n)] == p.pad) continue;
      for (int k = lane * 4; k < p.E; k += 256) {
        float v[4];
        load4<T>(x + (long)n * p.E, k, p.E, vec, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) take(v[j]);
      }
    }
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) p.amax[which * DT_AMAX + slot] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// The counts as sums of all before them, in place, by one block.  The kernel behind wants such a sum in every block of 16 rows: up to
// DT_CSCAN counts each block adds up what it needs, more are added up once, here.  E = 8: 2^19 rows 106 us either way, 2^20 234
// (5 + 177 with this), 2^23 6800 (24 + 1580).
constexpr int DT_CSCAN = 2048;
__global__ __launch_bounds__(1024) void dt_scan_kernel(DistillArgs p, int nb) {
  __shared__ int sums[16];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (nb + 1023) / 1024;
  const int i0 = min(nb, (int)threadIdx.x * per), i1 = min(nb, i0 + per);
  int mine = 0;
  for (int i = i0; i < i1; ++i) mine += p.counts[i];
  int upto = mine;                                                // over the lanes of a wave, its own included
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int x = __shfl_up(upto, o, 64);
    if (lane >= o) upto += x;
  }
  if (lane == 63) sums[wave] = upto;
  __syncthreads();
  int at = upto - mine;
  for (int w = 0; w < wave; ++w) at += sums[w];
  for (int i = i0; i < i1; ++i) {
    const int c = p.counts[i];
    p.counts[i] = at;
    at += c;
  }
  if (threadIdx.x == 1023) p.counts[nb] = at;
}

// four rows of an image by a wave, loaded together: row[q] (null: zeros, when `to` is not) -> to[q] (null: none)
template <typename T, int NP>
__device__ __forceinline__ void image_rows(const T* const (&row)[4], _Float16* const (&to)[4], int E, int K4, bool vec,
                                           const int (&e)[4], int lane, float one) {
  for (int k = lane; k < K4; k += 64) {
    float x[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[q][j] = 0.f;
      if (row[q]) load4<T>(row[q], 4 * k, E, vec, x[q]);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (!to[q]) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[q][j] = ldexpf(x[q][j], e[q]);
        if (one != 0.f && 4 * k + j == E && row[q]) x[q][j] = ldexpf(one, e[q]);
      }
      store4<NP>(to[q], 4 * k, x[q]);
    }
  }
}

// The row list and the images, 16 rows a block.  Blocks [0, cdiv(N, 16)): rows of X to their places in the compact
// order; the next Np / 16: zeros of the compact rows past the last live one; the rest: rows of W and its bias.  One read and one
// write of X and W, of which the count before left much in the caches: 36 us for 110 + 110 MB.
template <typename T, int NP> __global__ __launch_bounds__(256) void dt_image_kernel(DistillArgs p, int nx) {
  __shared__ float red[4];
  __shared__ int sred[4], swave[4], slot[DT_CROWS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long ld = (long)p.Kp * NP;
  const int nb = (p.N + DT_CROWS - 1) / DT_CROWS;
  int blk = blockIdx.x;
  const T* row[4];
  _Float16* to[4];
  int ee[4];
  if (blk < nx + p.Np / 16) {
    const bool tail = blk >= nx;
    const int group = tail ? nb : blk * 16 / DT_CROWS;
    int s = 0;
    if (p.scanned) s = threadIdx.x == 0 ? p.counts[group] : 0;
    else for (int i = threadIdx.x; i < group; i += 256) s += p.counts[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) sred[wave] = s;
    if (tail) {
      __syncthreads();
      const int nl = sred[0] + sred[1] + sred[2] + sred[3];
      if (blk == nx && threadIdx.x == 0) *p.nlive = nl;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = (blk - nx) * 16 + wave * 4 + q;
        row[q] = nullptr;
        to[q] = i >= nl ? p.Ximg + i * ld : nullptr;
        ee[q] = 0;
      }
      image_rows<T, NP>(row, to, p.E, p.Kp / 4, false, ee, lane, 0.f);
      return;
    }
    const int n = group * DT_CROWS + threadIdx.x;
    const bool live = n < p.N && p.eos[position(p, n)] != p.pad;
    const unsigned long long b = __ballot(live);
    if (lane == 0) swave[wave] = __popcll(b);
    __syncthreads();
    int off = sred[0] + sred[1] + sred[2] + sred[3];
    for (int i = 0; i < wave; ++i) off += swave[i];
    off += __popcll(b & ((1ull << lane) - 1ull));
    slot[threadIdx.x] = live ? off : -1;
    if (blk * 16 == group * DT_CROWS) {                           // the group's first block writes its lists
      if (n < p.N) p.inv[n] = live ? off : -1;
      if (live) p.rows[off] = n;
    }
    const int e = scale_exp(block_amax(p.amax, red));             // (its barriers also publish slot[])
    if (blk == 0 && threadIdx.x == 0) p.sexp[0] = e;
    const bool vec = p.E % 4 == 0 && ((uintptr_t)p.X % (4 * sizeof(T))) == 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int nn = blk * 16 + wave * 4 + q, at = slot[nn - group * DT_CROWS];
      row[q] = at >= 0 ? static_cast<const T*>(p.X) + (long)nn * p.E : nullptr;
      to[q] = at >= 0 ? p.Ximg + at * ld : nullptr;
      ee[q] = e;
    }
    image_rows<T, NP>(row, to, p.E, p.Kp / 4, vec, ee, lane, 0.f);
    return;
  }
  blk -= nx + p.Np / 16;
  const int e = scale_exp(block_amax(p.amax + DT_AMAX, red));
  if (blk == 0 && threadIdx.x == 0) p.sexp[1] = e;
  const bool vec = p.E % 4 == 0 && ((uintptr_t)p.W % (4 * sizeof(T))) == 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int v = blk * 16 + wave * 4 + q;
    row[q] = v < p.V ? static_cast<const T*>(p.W) + (long)v * p.E : nullptr;
    to[q] = p.Wimg + v * ld;
    ee[q] = e;
  }
  if (threadIdx.x < 16) {
    const int v = blk * 16 + threadIdx.x;
    p.b2[v] = v < p.V ? (float)static_cast<const T*>(p.bias)[v] * LOG2E : -INFINITY;
  }
  image_rows<T, NP>(row, to, p.E, p.Kp / 4, vec, ee, lane, 0.f);
}

// ------------------------------------------------------------------------------------------------- the product loop
// One operand's tile of RT rows / columns, copied to LDS by NW waves.  Memory holds 128-byte pieces: `row` bytes from a
// row's piece to the next row's, `grp` bytes from a piece to the next one of the same row (images: grp = 128, a row is
// contiguous; P: row = 128, the rows of one piece are contiguous).
//   K along the rows (KS = false): RT rows; stage s is piece s of each, KR = 64 / NP values.
//   K down the rows (KS = true): RT columns, that is RT NP / 64 pieces, of KR rows a stage.
// In LDS, 16-byte chunk c of row r sits at chunk c ^ (r / 2 & 7) of its 128 bytes (KS: c ^ 4 (r & 3)): the chunks that
// 16 lanes of a read take lie in different banks of the 64 (c ^ (r & 7) left two rows in each: half of all LDS cycles).
//
// A copy takes its address as a scalar base and 32 bits a lane (64-bit addresses a lane cost the walk at E = 200 two additions a
// copy and the registers for them: 148 -> 135 us).
template <int BYTES> __device__ __forceinline__ void copy_lds(const void* base, unsigned off, void* lds) {
  const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, -1, 0x27000);
  auto* to = (__attribute__((address_space(3))) void*)lds;
  if constexpr (BYTES == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 16, off, 0, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, to, 4, off, 0, 0, 0);
}
template <int NP, bool KS, int RT, int NW, int KR = 64 / NP> struct Operand {
  static constexpr int PLANES = NP, KB = KR / 16;                 // K blocks of 16 in a stage
  static constexpr int PI = RT * 2 * NP * KR / 1024 / NW;         // copies of 1 KiB a wave and stage
  static constexpr int ROW = RT * 2 * NP;                         // bytes of a K row in LDS (KS)
  const char* base;
  long row, grp;
  unsigned off[PI];
  __device__ __forceinline__ void init(const void* p, long row_bytes, long grp_bytes, int lane, int wave) {
    base = static_cast<const char*>(p);
    row = row_bytes;
    grp = grp_bytes;
#pragma unroll
    for (int i = 0; i < PI; ++i) {
      const int piece = wave * PI + i;
      if (!KS) {
        const int r = piece * 8 + (lane >> 3);
        off[i] = (unsigned)(r * row + (((lane & 7) ^ ((r >> 1) & 7)) << 4));
      } else {
        constexpr int LPR = ROW / 16;                             // lanes (chunks) of a row
        const int r = piece * (64 / LPR) + lane / LPR, c = (lane % LPR) ^ ((r & 3) << 2);
        off[i] = (unsigned)(r * row + (c >> 3) * grp + ((c & 7) << 4));
      }
    }
  }
  // copies [i0, i1) of a stage
  __device__ __forceinline__ void issue(int stage, char* lds, int wave, int i0 = 0, int i1 = PI) const {
    const char* b = base + (KS ? (long)stage * KR * row : (long)stage * grp);
#pragma unroll
    for (int i = i0; i < i1; ++i) copy_lds<16>(b, off[i], lds + (wave * PI + i) * 1024);
  }
  // the 32 rows / columns from `c0`, K block `ks` of the stage, plane `pl`, as one MFMA operand
  static __device__ __forceinline__ h8 frag(const char* lds, int c0, int ks, int pl, int lane) {
    if (!KS) {
      const int r = c0 + (lane & 31), c = (NP == 1 ? 0 : pl * 4) + ks * 2 + (lane >> 5);
      return *reinterpret_cast<const h8*>(lds + r * 128 + ((c ^ ((r >> 1) & 7)) << 4));
    }
    const int k = ks * 16 + (lane >> 5) * 8 + ((lane >> 2) & 3);
    const int col = c0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
    const int byte = NP == 1 ? col * 2 : (col >> 5) * 128 + pl * 64 + (col & 31) * 2;
    const char* q = lds + k * ROW + ((((byte >> 4) ^ ((k & 3) << 2)) << 4) | (byte & 15));
    union { s4 s[2]; h8 h; } u;
    u.s[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q));
    u.s[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(q + 4 * ROW));
    return u.h;
  }
};

// acc[i][j] += (rows am + 32 i of A) x (rows bn + 32 j of B) over `blocks` K blocks of the stage in LDS.  The next block's
// operands are read, and more(block) adds its share of the next stage's copies, while the matrix unit works on this one:
// a CU takes a copy of 1 KiB every 16 cycles, so asked for all at once at a stage's start they hold its waves back.
template <typename OA, typename OB, typename More>
__device__ __forceinline__ void stage_product(const char* la, const char* lb, int am, int bn, int blocks, int lane,
                                              f32x16 (&acc)[2][2], const More& more) {
  constexpr int NA = OA::PLANES, NB = OB::PLANES, KB = OA::KB;
  h8 a[2][2][NA], b[2][2][NB];
  const auto read = [&](int ks) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
      for (int q = 0; q < NA; ++q) a[ks & 1][i][q] = OA::frag(la, am + 32 * i, ks, q, lane);
#pragma unroll
      for (int q = 0; q < NB; ++q) b[ks & 1][i][q] = OB::frag(lb, bn + 32 * i, ks, q, lane);
    }
  };
  read(0);
#pragma unroll
  for (int ks = 0; ks < KB; ++ks) {
    if (ks >= blocks) continue;
    if (ks + 1 < KB) read(ks + 1);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) {                               // the small products first
        const int q = ks & 1;
        if (NB == 2) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[q][i][0], b[q][j][NB - 1], acc[i][j], 0, 0, 0);
        if (NA == 2) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[q][i][NA - 1], b[q][j][0], acc[i][j], 0, 0, 0);
        acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[q][i][0], b[q][j][0], acc[i][j], 0, 0, 0);
      }
    more(ks);
    __builtin_amdgcn_sched_barrier(0);
  }
}
__device__ __forceinline__ void clear(f32x16 (&acc)[2][2]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
}
// this wave's copies into LDS have arrived and its reads of the other buffers are over; then those of all waves
__device__ __forceinline__ void stage_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);                             // vmcnt(0) lgkmcnt(0), where the compiler sees it
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
// Two buffers of two operands as four arrays: the compiler then sees that a copy into one is no reason for a read of
// another to wait (it waits for every copy in flight when buffers share an array, and nothing overlaps).
#define DT_LDS \
  __shared__ __attribute__((aligned(16))) char la0[DT_STAGE]; \
  __shared__ __attribute__((aligned(16))) char lb0[DT_STAGE]; \
  __shared__ __attribute__((aligned(16))) char la1[DT_STAGE]; \
  __shared__ __attribute__((aligned(16))) char lb1[DT_STAGE];
// the four together as one area of 64 KiB for an epilogue, in units of 16 KiB
#define DT_AREA(i) ((i) == 0 ? la0 : (i) == 1 ? lb0 : (i) == 2 ? la1 : lb1)

// Stages [0, n), n > 0, of one tile, stage 0 already on its way into (la, lb); `last` K blocks of the last stage are used.
// While a stage is multiplied the next one loads: behind the last one, whatever then(a, b) asks for the free pair.
// (No stage is left out of the loop's middle: a `break` there cost 64 register moves a round.)
template <typename OA, typename OB, typename Then>
__device__ __forceinline__ void stages(const OA& A, const OB& B, int n, int last, char* la,
                                       char* lb, char* na, char* nb, int am, int bn, int lane, int wave,
                                       f32x16 (&acc)[2][2], const Then& then) {
  constexpr int KB = OA::KB, PA = OA::PI, PB = OB::PI;
  const auto copy = [&](int s, char* a, char* b) {
    return [&, s, a, b](int ks) {
      A.issue(s, a, wave, ks * PA / KB, (ks + 1) * PA / KB);
      B.issue(s, b, wave, ks * PB / KB, (ks + 1) * PB / KB);
    };
  };
  const auto none = [](int) {};
  int s = 0;
  for (; s + 3 <= n; s += 2) {
    stage_barrier();
    stage_product<OA, OB>(la, lb, am, bn, KB, lane, acc, copy(s + 1, na, nb));
    stage_barrier();
    stage_product<OA, OB>(na, nb, am, bn, KB, lane, acc, copy(s + 2, la, lb));
  }
  if (s + 2 == n) {
    stage_barrier();
    stage_product<OA, OB>(la, lb, am, bn, KB, lane, acc, copy(s + 1, na, nb));
    stage_barrier();
    then(la, lb);
    stage_product<OA, OB>(na, nb, am, bn, last, lane, acc, none);
  } else {
    stage_barrier();
    then(na, nb);
    stage_product<OA, OB>(la, lb, am, bn, last, lane, acc, none);
  }
}

// The same with three buffers, for tiles of 256 x 128 on 8 waves (one block on a CU): two stages are in flight under the
// one that is multiplied.  A stage's barrier stands before its last K block, whose operands are in registers by then: the
// next stage's first operands are read under that block's products, and the matrix unit does not wait for LDS behind a
// barrier.  Past the end the last stage is copied again, so that the count of copies to wait for is a constant.
template <int C> __device__ __forceinline__ void ring_barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070 | (C & 15) | (C >> 4) << 14);  // vmcnt(C) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
//
// A tile is 8 x 4 fragments of 32 x 32 (columns of E by rows or words; RA = 128: 4 x 8), four to a wave, 2 x 2 of them: where a
// tile of E has at most 224 (96) columns, the waves of its second half (all waves) take 3 x 1 instead, and nothing is
// multiplied for the last 32 columns of padding.  Two waves share a SIMD, w and w + 4: each SIMD then has 7 fragments, not 8
// (both products of 3520 x 200 x 20000 fp32 142 -> 134 us, of 3650 x 1024 x 50000 bf16, whose bias column has a tile, 784 -> 756).
template <int RA> struct Part {
  bool tall;
  int a, b, wave;                                                 // first column of E, first of the other operand
  __device__ __forceinline__ Part(int cols, int w) : wave(w) {
    tall = RA == 256 ? cols <= 224 && w >= 4 : cols <= 96;
    a = RA == 256 ? (tall ? 128 : (w >> 1) * 64) : (tall ? 0 : (w & 1) * 64);
    b = RA == 256 ? (tall ? (w - 4) * 32 : (w & 1) * 64) : (tall ? w * 32 : (w >> 1) * 64);
  }
  __device__ __forceinline__ bool has(int i) const { return !tall || i < 3; }
  __device__ __forceinline__ int col(int i) const { return a + (tall ? i : i >> 1) * 32; }
  __device__ __forceinline__ int row(int i) const { return b + (tall ? 0 : i & 1) * 32; }
};
// FOLD > 0: what FOLD stages added up is put aside and the next ones start from zero, so that a long K is no single chain of
// additions (whose error grows with the root of its length).
template <bool TALL, int FOLD, typename OA, typename OB>
__device__ __forceinline__ void ring_product(const OA& A, const OB& B, int n, char* la0, char* lb0, char* la1, char* lb1,
                                             char* la2, char* lb2, int am, int bn, int lane, int wave, f32x16 (&acc)[4]) {
  constexpr int C = OA::PI + OB::PI, KB = OA::KB, NA = OA::PLANES, NB = OB::PLANES;
  constexpr int SH = KB == 4 ? 3 : 2;                             // a stage's copies in SH shares
  constexpr int FA = TALL ? 3 : 2, FB = TALL ? 1 : 2;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  if (n <= 0) return;
  f32x16 sum[4] = {};
  h8 a[2][FA][NA], b[2][FB][NB];
  const auto read = [&](int q, const char* la, const char* lb, int ks) {
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int pl = 0; pl < NA; ++pl) a[q][i][pl] = OA::frag(la, am + 32 * i, ks, pl, lane);
#pragma unroll
    for (int i = 0; i < FB; ++i)
#pragma unroll
      for (int pl = 0; pl < NB; ++pl) b[q][i][pl] = OB::frag(lb, bn + 32 * i, ks, pl, lane);
  };
  const auto multiply = [&](int q) {
#pragma unroll
    for (int i = 0; i < FA; ++i)
#pragma unroll
      for (int j = 0; j < FB; ++j) {                              // the small products first
        f32x16& x = acc[i * FB + j];
        if (NB == 2) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[q][i][0], b[q][j][NB - 1], x, 0, 0, 0);
        if (NA == 2) x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[q][i][NA - 1], b[q][j][0], x, 0, 0, 0);
        x = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[q][i][0], b[q][j][0], x, 0, 0, 0);
      }
  };
  const auto copy = [&](int s, char* la, char* lb, int share) {
    s = s < n ? s : n - 1;
    A.issue(s, la, wave, share * OA::PI / SH, (share + 1) * OA::PI / SH);
    B.issue(s, lb, wave, share * OB::PI / SH, (share + 1) * OB::PI / SH);
  };
  // stage s from (la, lb); stage s + 1 is in (na, nb); (fa, fb), stage s - 1's, still take stage s + 2's last shares
  const auto step = [&](int s, char* la, char* lb, char* na, char* nb, char* fa, char* fb, bool first) {
#pragma unroll
    for (int ks = 0; ks + 1 < KB; ++ks) {
      read((ks + 1) & 1, la, lb, ks + 1);
      multiply(ks & 1);
      if (!first && ks + 1 < SH) copy(s + 2, fa, fb, ks + 1);
      __builtin_amdgcn_sched_barrier(0);
    }
    ring_barrier<C>();                                            // stage s + 1 is there, and all are done with stage s
    read(0, na, nb, 0);
    multiply((KB - 1) & 1);
    copy(s + 3, la, lb, 0);
    __builtin_amdgcn_sched_barrier(0);
  };
#pragma unroll
  for (int i = 0; i < SH; ++i) copy(0, la0, lb0, i);
#pragma unroll
  for (int i = 0; i < SH; ++i) copy(1, la1, lb1, i);
#pragma unroll
  for (int i = 0; i < SH; ++i) copy(2, la2, lb2, i);
  ring_barrier<2 * C>();
  read(0, la0, lb0, 0);
  step(0, la0, lb0, la1, lb1, la2, lb2, true);
  int s = 1;
  for (; s + 3 <= n; s += 3) {
    step(s, la1, lb1, la2, lb2, la0, lb0, false);
    step(s + 1, la2, lb2, la0, lb0, la1, lb1, false);
    step(s + 2, la0, lb0, la1, lb1, la2, lb2, false);
    static_assert(FOLD % 3 == 0, "whole rounds of the three buffers");
    if (FOLD && s % (FOLD ? FOLD : 1) == 1) {
#pragma unroll
      for (int i = 0; i < FA * FB; ++i) { sum[i] += acc[i]; acc[i] = f32x16{}; }
    }
  }
  if (s < n) step(s, la1, lb1, la2, lb2, la0, lb0, false);
  if (s + 1 < n) step(s + 1, la2, lb2, la0, lb0, la1, lb1, false);
  ring_barrier<0>();                                              // no copy may land in LDS that the next block owns
  if (FOLD) {
#pragma unroll
    for (int i = 0; i < FA * FB; ++i) acc[i] += sum[i];
  }
}
// three buffers for the operand of 256 rows or columns, three for the one of 128
struct Ring { char *x0, *x1, *x2, *y0, *y1, *y2; };
template <int RA, int FOLD, typename OA, typename OB>
__device__ __forceinline__ void tile_product(const OA& A, const OB& B, int n, const Ring& m, const Part<RA>& t, int lane,
                                             f32x16 (&acc)[4]) {
  char *a0 = RA == 256 ? m.x0 : m.y0, *a1 = RA == 256 ? m.x1 : m.y1, *a2 = RA == 256 ? m.x2 : m.y2;
  char *b0 = RA == 256 ? m.y0 : m.x0, *b1 = RA == 256 ? m.y1 : m.x1, *b2 = RA == 256 ? m.y2 : m.x2;
  if (t.tall) ring_product<true, FOLD>(A, B, n, a0, b0, a1, b1, a2, b2, t.a, t.b, lane, t.wave, acc);
  else ring_product<false, FOLD>(A, B, n, a0, b0, a1, b1, a2, b2, t.a, t.b, lane, t.wave, acc);
}

// ------------------------------------------------------------------------------------------------- forward
// Work items of the kernels that walk the vocabulary: (tile of 128 live rows) x (range of its vt tiles).  512 blocks, two
// on a CU; the 64 of an XCD (block % 8) take every eighth range, so that they share W's tiles in its L2.  The number of
// ranges, 8 k with k >= least, is what the live rows (known on the device alone) make cheapest: rounds of 64 items times the
// tiles of an item, and one tile's time for its start.  One wave's lanes try one k each; every kernel that needs it gets the same.
constexpr int DT_WALK_BLOCKS = 512, DT_MOST_ITEMS = 1024;         // the latter: per XCD, for more than one range
__device__ __forceinline__ int dt_splits(int nt, int vt, int least) {
  const int k = (threadIdx.x & 63) + 1;
  const bool ok = k == 1 || (k * 8 <= vt && nt * k <= DT_MOST_ITEMS && k >= least);
  int best = 0x7fffffff;
  if (ok) best = min(((nt * k + 63) / 64) * ((vt + 8 * k - 1) / (8 * k) + 1), 0x1ffffff) * 64 + (k - 1);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
  return __builtin_amdgcn_readfirstlane(((best & 63) + 1) * 8);
}

// An XCD's item q of (row tile, range of W): eight row tiles at a time over all its ranges, so that the rows that are
// walked at once (8 x 128 x K) stay in its L2 beside the tiles of W (E = 1024, V = 50000, with at least 8 ranges: 469 us,
// all 29 row tiles at once: 504).
__device__ __forceinline__ void walk_order(int q, int nt, int ranges, int& tn, int& range) {
  const int group = q / (8 * ranges), rem = q - group * 8 * ranges, size = min(8, nt - 8 * group);
  range = __builtin_amdgcn_readfirstlane(rem / size);             // (scalar, for the copies' addresses)
  tn = __builtin_amdgcn_readfirstlane(group * 8 + rem - range * size);
}

// Fold 64 vocabulary entries of a lane's row into its running (max, sum) pairs, base 2: two accumulator tiles of 32
// entries, of which the lane holds 16 each, and their biases.
template <bool TWO>
__device__ __forceinline__ void fold(f32x16& t0, f32x16& t1, const float4 (&bias)[2][4], float c, float itau, float& m,
                                     float& s1, float& s2) {
  float mx = m;
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float4 &ba = bias[0][r >> 2], &bb = bias[1][r >> 2];
    t0[r] = fmaf(t0[r], c, (r & 3) == 0 ? ba.x : (r & 3) == 1 ? ba.y : (r & 3) == 2 ? ba.z : ba.w);
    t1[r] = fmaf(t1[r], c, (r & 3) == 0 ? bb.x : (r & 3) == 1 ? bb.y : (r & 3) == 2 ? bb.z : bb.w);
    mx = fmaxf(mx, fmaxf(t0[r], t1[r]));
  }
  const float back = m - mx;
  float a = s1 * __builtin_amdgcn_exp2f(back), b = 0.f;
  if (TWO) b = s2 * __builtin_amdgcn_exp2f(back * itau);
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const float d0 = t0[r] - mx, d1 = t1[r] - mx;
    a += __builtin_amdgcn_exp2f(d0) + __builtin_amdgcn_exp2f(d1);
    if (TWO) b += __builtin_amdgcn_exp2f(d0 * itau) + __builtin_amdgcn_exp2f(d1 * itau);
  }
  m = mx; s1 = a; s2 = b;
}
// Join the pairs of the lanes (and of the `waves` waves) that share a row, and store them for the merge:
// part[3][splits][nt * 128].  x: [waves][128][3] floats of LDS.
template <int NJ, bool TWO>
__device__ __forceinline__ void store_pairs(const DistillArgs& p, float* x, const float* m, const float* s1, const float* s2,
                                            int split, int nt, int n0, int bn, int who, int waves, int lane) {
#pragma unroll
  for (int j = 0; j < NJ; ++j) {
    const float m2 = __shfl_xor(m[j], 32, 64), mm = fmaxf(m[j], m2);
    const float f = __builtin_amdgcn_exp2f(m[j] - mm), f2 = __builtin_amdgcn_exp2f(m2 - mm);
    const float a = s1[j] * f + __shfl_xor(s1[j], 32, 64) * f2;
    float b = 0.f;
    if (TWO) b = s2[j] * __builtin_amdgcn_exp2f((m[j] - mm) * p.itau) +
                 __shfl_xor(s2[j], 32, 64) * __builtin_amdgcn_exp2f((m2 - mm) * p.itau);
    if (lane < 32) {
      float* y = x + (who * 128 + bn + 32 * j + lane) * 3;
      y[0] = mm; y[1] = a; y[2] = b;
    }
  }
  __syncthreads();
  if (threadIdx.x < 128) {
    const float* y = x + threadIdx.x * 3;
    float mm = y[0], a = y[1], b = y[2];
    if (waves == 2) {
      const float* z = y + 128 * 3;
      const float m1 = mm;
      mm = fmaxf(m1, z[0]);
      a = a * __builtin_amdgcn_exp2f(m1 - mm) + z[1] * __builtin_amdgcn_exp2f(z[0] - mm);
      if (TWO) b = b * __builtin_amdgcn_exp2f((m1 - mm) * p.itau) + z[2] * __builtin_amdgcn_exp2f((z[0] - mm) * p.itau);
    }
    float* out = p.part + (long)split * nt * 128 + n0 + threadIdx.x;
    out[0] = mm;
    out[p.pplane] = a;
    if (TWO) out[2 * p.pplane] = b;
  }
}

// The forward walk for any E: both operands stream through LDS, a stage of 64 K values (two planes: 32) loading under the
// one that is multiplied, four waves of 64 x 64 each, two blocks on a CU so that one's fold runs under the other's products.
// 3650 rows x 1024 x 50000 bf16: 415 us, 0.90 PFLOP/s, matrix cores busy 53 % of the time at 1.81 GHz; fold and pipeline
// restarts between tiles are the rest.  (256 x 128 tiles of eight waves, one block on a CU: 529 where this took 461, its
// fold stands alone.)
template <int NP, bool TWO>
__global__ __launch_bounds__(256, 2) void dt_forward_kernel(DistillArgs p) {
  DT_LDS
  const int nl = *p.nlive, nt = (nl + DT_TILE - 1) / DT_TILE, vt = p.fvt;
  if (nt == 0) return;
  const int splits = dt_splits(nt, vt, p.least), per = __builtin_amdgcn_readfirstlane((vt + splits - 1) / splits);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int am = (wave >> 1) * 64, bn = (wave & 1) * 64;
  const float c = unscale(p.sexp);
  const long ld = (long)p.Kp * NP * 2;
  const int nst = (p.E + 64 / NP - 1) / (64 / NP), last = ((p.E + 15) / 16) - (nst - 1) * (4 / NP);
  const int xcd = blockIdx.x & 7, per_xcd = nt * (splits / 8);
  for (int q = blockIdx.x >> 3; q < per_xcd; q += DT_WALK_BLOCKS / 8) {
    int tn, range;
    walk_order(q, nt, splits / 8, tn, range);
    const int split = xcd + 8 * range, n0 = tn * DT_TILE;
    const int t0 = split * per, t1 = min(vt, t0 + per);
    using Op = Operand<NP, false, DT_TILE, 4>;
    Op A, B;
    A.init(p.Wimg, ld, 128, lane, wave);
    B.init(reinterpret_cast<const char*>(p.Ximg) + n0 * ld, ld, 128, lane, wave);
    float m[2], s1[2], s2[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) { m[j] = -1e30f; s1[j] = s2[j] = 0.f; }
    f32x16 acc[2][2];
    const char* wbase = A.base;
    A.base = wbase + (long)t0 * DT_TILE * ld;
    __syncthreads();                                              // the last item's reads are over
    if (t0 < t1) { A.issue(0, la0, wave); B.issue(0, lb0, wave); }
    const auto do_tile = [&](int tile, char* la, char* lb, char* na, char* nb) {
      clear(acc);
      stages<Op, Op>(A, B, nst, last, la, lb, na, nb, am, bn, lane, wave, acc, [&](char* fa, char* fb) {
        if (tile + 1 < t1) {                                      // the next tile of W loads under this one's fold
          A.base = wbase + (long)(tile + 1) * DT_TILE * ld;
          A.issue(0, fa, wave);
          B.issue(0, fb, wave);
        }
      });
      const float* b2 = p.b2 + tile * DT_TILE + am;
      float4 bias[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) bias[i][g] = *reinterpret_cast<const float4*>(b2 + 32 * i + 8 * g + 4 * (lane >> 5));
#pragma unroll
      for (int j = 0; j < 2; ++j) fold<TWO>(acc[0][j], acc[1][j], bias, c, p.itau, m[j], s1[j], s2[j]);
    };
    for (int tile = t0; tile < t1; ++tile) {                      // an odd number of stages swaps the pairs
      do_tile(tile, la0, lb0, la1, lb1);
      if ((nst & 1) && tile + 1 < t1) do_tile(++tile, la1, lb1, la0, lb0);
    }
    __syncthreads();
    store_pairs<2, TWO>(p, reinterpret_cast<float*>(la0), m, s1, s2, split, nt, n0, bn, wave >> 1, 2, lane);
  }
}

// The same walk for E <= 208 with the rows of X in registers: a wave holds 64 (two planes: 32) of the 128 rows, all K, as
// MFMA operands, and only W streams through LDS -- half the LDS reads and half the copies of the general kernel, which
// at E = 200 spends its time on them.  Stages of 64 K values x 128 (64) words, four buffers, three in flight; K blocks
// of 16: NK = 4, 8 or 13 (E up to 64, 128, 208; every shipped model has E = 200).  GRAD: instead of folding, the tile
// leaves as P = a 2^(t - L1) + b 2^(t / tau - L2), through 2 KiB of LDS a wave so that rows leave in runs of 64 bytes.
// 4815 rows x 200 x 50000 bf16, two exponentials an element: forward 143 us (0.67 PFLOP/s), gradient 220 in two ranges (527 MB
// written and 214 read by the memory counters, 3.4 TB/s); fp16, whose P has two planes, 360 in four.
// Nothing alone bounds it: left out one at a time when the forward walk took 155, exponentials were worth 35 us, copies 25,
// products 30.  Standing the fold of one tile between the products of the next (two sets of accumulators) gained nothing there
// and cost the gradient 10 %.
template <int NP, int NQ, bool TWO, bool GRAD, int NK>
__global__ __launch_bounds__(256, 2) void dt_rows_kernel(DistillArgs p) {
  constexpr int NST = NK <= 4 ? 1 : NK <= 8 ? 2 : 4, VT = 128 / NP, NJ = 2 / NP, RB = 128 * NP;   // RB: bytes of a row's stage
  __shared__ __attribute__((aligned(16))) char w0[DT_STAGE + 512];
  __shared__ __attribute__((aligned(16))) char w1[DT_STAGE + 512];
  __shared__ __attribute__((aligned(16))) char w2[DT_STAGE + 512];
  __shared__ __attribute__((aligned(16))) char w3[DT_STAGE + 512];
  __shared__ __attribute__((aligned(16))) char turn[GRAD ? 4 * 2048 : 2 * 128 * 3 * sizeof(float)];
  const int nl = *p.nlive, nt = (nl + DT_TILE - 1) / DT_TILE, vt = GRAD ? p.vc / VT : p.fvt;
  if (nt == 0) return;
  const int splits = dt_splits(nt, vt, 1), per = __builtin_amdgcn_readfirstlane((vt + splits - 1) / splits);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int am = NP == 1 ? (wave >> 1) * 64 : 0, bn = NP == 1 ? (wave & 1) * 64 : wave * 32;
  const int l31 = lane & 31, lhi = lane >> 5;
  const float c = unscale(p.sexp);
  const long ld = (long)p.Kp * NP * 2;
  unsigned off[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int piece = wave * 4 + i;
    const int r = NP == 1 ? piece * 8 + (lane >> 3) : piece * 4 + (lane >> 4);
    const int ch = NP == 1 ? (lane & 7) ^ ((r >> 1) & 7) : (lane & 15) ^ (r & 15);
    off[i] = (unsigned)(r * ld + ch * 16);
  }
  const int boff = NP == 1 ? (wave & 1) * 256 : 0;                // each wave copies 64 of the tile's biases
  const int xcd = blockIdx.x & 7, per_xcd = nt * (splits / 8);
  for (int q = blockIdx.x >> 3; q < per_xcd; q += DT_WALK_BLOCKS / 8) {
    const int range = __builtin_amdgcn_readfirstlane(q / nt), split = xcd + 8 * range, n0 = (q - range * nt) * DT_TILE;
    const int t0 = split * per, t1 = min(vt, t0 + per);
    if (GRAD && t0 >= t1) continue;
    float m[NJ], s1[NJ], s2[NJ];                                  // GRAD: L1, a, then L2, b
    float La[NJ], Lb[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      m[j] = -1e30f; s1[j] = s2[j] = 0.f;
      La[j] = Lb[j] = INFINITY;                                   // rows past the last live one: 0 * 2^-inf
      const int i = n0 + bn + 32 * j + l31;
      if (GRAD && i < nl) {
        La[j] = p.L1[i]; Lb[j] = p.L2[i];
        s1[j] = p.coef[i]; s2[j] = p.coef[p.Np + i];
        if (!TWO) s1[j] += s2[j];
      }
    }
    if (t0 < t1) {
      const auto ring = [&](int g) -> char* { return (g & 3) == 0 ? w0 : (g & 3) == 1 ? w1 : (g & 3) == 2 ? w2 : w3; };
      const auto copy = [&](const char* from, char* w) {          // a stage: 16 KiB
#pragma unroll
        for (int i = 0; i < 4; ++i) copy_lds<16>(from, off[i], w + (wave * 4 + i) * 1024);
      };
      // one operand of 32 rows from `r`, K block ks of a stage, plane pl
      const auto frag = [&](const char* w, int r, int ks, int pl) {
        const int ch = NP == 1 ? (ks * 2 + lhi) ^ ((r >> 1) & 7) : ((ks >> 1) * 8 + pl * 4 + (ks & 1) * 2 + lhi) ^ (r & 15);
        return *reinterpret_cast<const h8*>(w + r * RB + ch * 16);
      };
      // the rows pass through the ring once: read from memory straight into operands they would come 32 bytes a row at a time
      // (`row` hides that their places in LDS are the same for every item: kept in registers they would push others into memory)
      h8 xf[NJ][NP][NK];
      int row = l31;
      asm volatile("" : "+v"(row));
#pragma unroll
      for (int half = 0; half < NP; ++half) {
#pragma unroll
        for (int st = 0; st < NST; ++st)
          copy(reinterpret_cast<const char*>(p.Ximg) + (n0 + half * 64) * ld + st * RB, ring(st));
        ring_barrier<0>();
        if (NP == 1 || wave >> 1 == half) {
#pragma unroll
          for (int j = 0; j < NJ; ++j)
#pragma unroll
            for (int pl = 0; pl < NP; ++pl)
#pragma unroll
              for (int kb = 0; kb < NK; ++kb) xf[j][pl][kb] = frag(ring(kb / 4), (NP == 1 ? bn + 32 * j : bn & 32) + row, kb & 3, pl);
        }
        ring_barrier<0>();
      }
      const char* W = reinterpret_cast<const char*>(p.Wimg) + (long)(GRAD ? p.v0 : 0) * ld;
      const float* b2 = p.b2 + (GRAD ? p.v0 : 0);
      const auto issue = [&](int tile, int st, char* w) {         // (past the range: its last tile again)
        tile = tile < t1 ? tile : t1 - 1;
        copy(W + (long)tile * VT * ld + st * RB, w);
        if (st == NST - 1)
          copy_lds<4>(b2 + tile * VT, boff + lane * 4, w + DT_STAGE + boff);
      };
#pragma unroll
      for (int g = 0; g < 3; ++g) issue(t0 + g / NST, g % NST, ring(g));
      for (int tile = t0; tile < t1; tile += 4 / NST) {
#pragma unroll
        for (int u = 0; u < 4 / NST; ++u) {
          const int tl = tile + u;
          if (tl >= t1) continue;
          f32x16 acc[2][NJ];
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < NJ; ++j)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
#pragma unroll
          for (int st = 0; st < NST; ++st) {
            const int g = u * NST + st;
            // Stages g + 1 and g + 2 stay in flight: four copies each, one more for a tile's last stage (its biases);
            // and the stores of every tile that ended within the last three steps (they count like copies, in order;
            // at an item's first three steps there are none to count).
            constexpr int two = 8 + (NST == 1 ? 2 : NST == 2 ? 1 : 0), out = NJ * 2 * NQ * 2;
            if (GRAD && (tl - t0) * NST + st >= 3) {
              if (NST == 4) { if (st == 0) ring_barrier<8 + out>(); else if (st == 3) ring_barrier<8>(); else ring_barrier<9 + out>(); }
              else if (NST == 2) { if (st == 0) ring_barrier<9 + 2 * out>(); else ring_barrier<9 + out>(); }
              else ring_barrier<10 + 3 * out>();
            } else if (NST == 4 && (st == 1 || st == 2)) {
              ring_barrier<9>();
            } else {
              ring_barrier<two>();
            }
            issue(tile + (g + 3) / NST, (g + 3) % NST, ring(g + 3));
            const char* w = ring(g);
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
              if (st * 4 + ks >= NK) continue;
              h8 a[2][NP];
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int pl = 0; pl < NP; ++pl) a[i][pl] = frag(w, am + 32 * i + l31, ks, pl);
#pragma unroll
              for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                  const int kb = st * 4 + ks;
                  if (NP == 2) {
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][0], xf[j][NP - 1][kb], acc[i][j], 0, 0, 0);
                    acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][NP - 1], xf[j][0][kb], acc[i][j], 0, 0, 0);
                  }
                  acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a[i][0], xf[j][0][kb], acc[i][j], 0, 0, 0);
                }
            }
          }
          const float* bl = reinterpret_cast<const float*>(ring(u * NST + NST - 1) + DT_STAGE) + am;
          if (!GRAD) {
            float4 bias[2][4];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int g = 0; g < 4; ++g) bias[i][g] = *reinterpret_cast<const float4*>(bl + 32 * i + 8 * g + 4 * lhi);
#pragma unroll
            for (int j = 0; j < NJ; ++j) fold<TWO>(acc[0][j], acc[1][j], bias, c, p.itau, m[j], s1[j], s2[j]);
            continue;
          }
          char* tr = turn + wave * 2048;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int v = tl * VT + am + 32 * i;                  // in the range
            float4 bias[4];
#pragma unroll
            for (int g = 0; g < 4; ++g) bias[g] = *reinterpret_cast<const float4*>(bl + 32 * i + 8 * g + 4 * lhi);
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
              char* out = reinterpret_cast<char*>(p.P) + ((long)(v * NQ >> 6) * p.Np + n0 + bn + 32 * j + (lane >> 2)) * 128 +
                          (NQ == 1 ? (v & 32) * 2 : 0) + (lane & 3) * 16;
              Packed<f16_t, 4> hi[4], lo[4];
#pragma unroll
              for (int g = 0; g < 4; ++g) {
                const float bv[4] = {bias[g].x, bias[g].y, bias[g].z, bias[g].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  const float t = fmaf(acc[i][j][4 * g + k], c, bv[k]);
                  float x = s1[j] * __builtin_amdgcn_exp2f(t - La[j]);
                  if (TWO) x = fmaf(s2[j], __builtin_amdgcn_exp2f(fmaf(t, p.itau, -Lb[j])), x);
                  if (NQ == 2) one_value(x);
                  hi[g].set(k, x);
                  if (NQ == 2) lo[g].set(k, x - hi[g].f(k));
                }
              }
#pragma unroll
              for (int pl = 0; pl < NQ; ++pl) {
#pragma unroll
                for (int g = 0; g < 4; ++g)
                  *reinterpret_cast<Packed<f16_t, 4>*>(tr + l31 * 64 + ((g ^ ((l31 >> 1) & 3)) << 4) + lhi * 8) = pl ? lo[g] : hi[g];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const int r = h * 16 + (lane >> 2);
                  const uint4 x = *reinterpret_cast<const uint4*>(tr + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4));
                  *reinterpret_cast<uint4*>(out + h * 16 * 128 + pl * 64) = x;
                }
              }
            }
          }
        }
      }
      ring_barrier<0>();                                          // the next item's copies go where the last ones landed
    }
    if (!GRAD) store_pairs<NJ, TWO>(p, reinterpret_cast<float*>(turn), m, s1, s2, split, nt, n0, bn, NP == 1 ? wave >> 1 : 0, 2 / NP, lane);
    if (!GRAD) __syncthreads();                                   // turn is read before the next item writes it
  }
}

// log2 of a picked word's softmax, its logit (a product of its own) less the normaliser (the walk's): at most 0, also where they are
// large enough that their roundings say otherwise; a NaN stays one
__device__ __forceinline__ float log_share(float d) { return d > 0.f ? 0.f : d; }

// sum over the 32 lanes of a half-wave: four steps inside rows of 16 lanes on the vector ALU, one through LDS
__device__ __forceinline__ float half_sum(float v) {
  const auto step = [](float x, int y) { return x + __builtin_bit_cast(float, y); };
  v = step(v, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));    // lane ^ 1
  v = step(v, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));    // lane ^ 2
  v = step(v, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));   // mirrored within 8
  v = step(v, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));   // mirrored within 16
  return v + __shfl_xor(v, 16, 64);
}

// One block per live row: the picked logits, the merge of the walk's pairs, the teacher's distribution, the two losses,
// and the teacher's shares as the backward pass wants them.  A row is one chain of dependent loads, so everything that
// does not wait for another load is asked for at once: the ids and teacher logits first.  (Two picked rows of W in flight
// a group of lanes: with 64 entries a row 41 us for 4815 rows, by the memory counters 159 MB at 4.0 TB/s; four took a seventh more,
// eight a half.)
constexpr int DT_MOST_K = 1024;
// Ids listed more than once are found through a table of first places, at most half full (comparing all pairs took, for 3520 rows x
// 200 bf16, 34 us with 64 entries, 178 with 256 and 1950 with 1024; this 26, 66 and 248).
constexpr int DT_FREE = 0x7fffffff;
__host__ __device__ __forceinline__ int dt_table_bits(int K) {
  int bits = 5;
  while ((1 << bits) < 2 * K) ++bits;
  return bits;
}
__host__ __device__ __forceinline__ int dt_combine_words(int K) {  // of LDS: ids, picked logits, teacher logits, table, repeats
  return 3 * K + 2 + (1 << dt_table_bits(K)) + (K + 31) / 32;
}
__device__ __forceinline__ unsigned table_slot(int id, int bits) { return (unsigned)id * 2654435769u >> (32 - bits); }
template <typename T, bool TWO>
__global__ __launch_bounds__(256) void dt_combine_kernel(DistillArgs p) {
  __shared__ float red[4][3];
  extern __shared__ __attribute__((aligned(16))) char words[];
  int* sid = reinterpret_cast<int*>(words);                       // ids inside the vocabulary, else -1; [K]: the target
  float* spick = reinterpret_cast<float*>(sid + p.K + 1);
  float* slog = spick + p.K + 1;
  int* table = reinterpret_cast<int*>(slog + p.K);                // first place of an id, at its slot or the next free one
  const int bits = dt_table_bits(p.K), size = 1 << bits;
  unsigned* multi = reinterpret_cast<unsigned*>(table + size);    // a bit per entry: its id is listed again
  const int i = blockIdx.x;
  const int nl = *p.nlive;
  if (i >= nl) return;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, K = p.K;
  const int n = p.rows[i];
  const long at = position(p, n);
  for (int k = threadIdx.x; k <= K; k += 256) {
    const int64_t id = k < K ? p.ids[at * K + k] : p.eos[at];
    sid[k] = id >= 0 && id < p.V ? (int)id : -1;
    if (k < K) slog[k] = p.top[at * K + k];
  }
  for (int i = threadIdx.x; i < size; i += 256) table[i] = DT_FREE;
  for (int i = threadIdx.x; i < (K + 31) / 32; i += 256) multi[i] = 0;
  // normalisers: every thread a share of the walk's ranges
  const int nt = (nl + DT_TILE - 1) / DT_TILE, splits = dt_splits(nt, p.fvt, p.least);
  float m = -1e30f, a = 0.f, b = 0.f;
  for (int s = threadIdx.x; s < splits; s += 256) {
    const float* q = p.part + (long)s * nt * 128 + i;
    const float m2 = q[0], mm = fmaxf(m, m2);
    a = a * __builtin_amdgcn_exp2f(m - mm) + q[p.pplane] * __builtin_amdgcn_exp2f(m2 - mm);
    if (TWO) b = b * __builtin_amdgcn_exp2f((m - mm) * p.itau) + q[2 * p.pplane] * __builtin_amdgcn_exp2f((m2 - mm) * p.itau);
    m = mm;
  }
  __syncthreads();
  for (int k = threadIdx.x; k < K; k += 256) {                    // (a slot holds places of one id for good; the least of them stays)
    const int id = sid[k];
    if (id < 0) continue;
    for (unsigned h = table_slot(id, bits);; h = (h + 1) & (size - 1)) {
      const int old = atomicCAS(&table[h], DT_FREE, k);
      if (old == DT_FREE) break;
      if (sid[old] == id) { atomicMin(&table[h], k); break; }
    }
  }
  // Picked logits, base 2: 32 lanes a dot product, 16 bytes a lane where rows allow it (a row of E = 200 in 16 bits is
  // then one access), else single elements.
  const T* x = static_cast<const T*>(p.X) + (long)n * p.E;
  const T* W = static_cast<const T*>(p.W);
  constexpr int VN = 16 / sizeof(T), FLY = 2;
  const bool vec = p.E % VN == 0 && (((uintptr_t)p.X | (uintptr_t)p.W) & 15) == 0;
  const int l32 = threadIdx.x & 31;
  for (int k0 = threadIdx.x >> 5; k0 <= K; k0 += 8 * FLY) {
    int id[FLY];
    float dot[FLY];
#pragma unroll
    for (int q = 0; q < FLY; ++q) {
      id[q] = k0 + 8 * q <= K ? sid[k0 + 8 * q] : -1;
      dot[q] = 0.f;
    }
    if (vec) {
      for (int e = l32 * VN; e < p.E; e += 32 * VN) {
        const Packed<T, VN> r = *reinterpret_cast<const Packed<T, VN>*>(x + e);
        Packed<T, VN> w[FLY];
#pragma unroll
        for (int q = 0; q < FLY; ++q)
          w[q] = *reinterpret_cast<const Packed<T, VN>*>(W + (long)max(id[q], 0) * p.E + e);
#pragma unroll
        for (int q = 0; q < FLY; ++q)
#pragma unroll
            for (int j = 0; j < VN; ++j) dot[q] = fmaf(r.f(j), w[q].f(j), dot[q]);
      }
    } else {
      for (int e = l32; e < p.E; e += 32) {
        const float r = (float)x[e];
#pragma unroll
        for (int q = 0; q < FLY; ++q)
          dot[q] = fmaf(r, (float)W[(long)max(id[q], 0) * p.E + e], dot[q]);
      }
    }
#pragma unroll
    for (int q = 0; q < FLY; ++q) {
      dot[q] = half_sum(dot[q]);
      if (l32 == 0 && k0 + 8 * q <= K) {
        const float v = id[q] >= 0 ? (dot[q] + (float)static_cast<const T*>(p.bias)[id[q]]) * LOG2E : 0.f;
        spick[k0 + 8 * q] = v;
        p.pick[(long)i * (K + 1) + k0 + 8 * q] = v;
      }
    }
  }
  {
    const float mm = wave_max(m);
    a = wave_sum(a * __builtin_amdgcn_exp2f(m - mm));
    if (TWO) b = wave_sum(b * __builtin_amdgcn_exp2f((m - mm) * p.itau));
    if (lane == 0) { red[wave][0] = mm; red[wave][1] = a; red[wave][2] = b; }
  }
  __syncthreads();
  if (wave != 0) return;
  m = fmaxf(fmaxf(red[0][0], red[1][0]), fmaxf(red[2][0], red[3][0]));
  a = b = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float d = red[w][0] - m;
    a += red[w][1] * __builtin_amdgcn_exp2f(d);
    if (TWO) b += red[w][2] * __builtin_amdgcn_exp2f(d * p.itau);
  }
  // (a, b >= 1, so L1 >= m; where rounding leaves L2 below m / tau, the next float: no share of the gradient walk passes 1)
  const float L1 = m + log2f(a);
  float L2 = TWO ? fmaf(m, p.itau, log2f(b)) : L1;
  if (TWO && fmaf(m, p.itau, -L2) > 0.f) L2 = fmaf(fabsf(L2), 0x1p-23f, L2);
  float tm = -INFINITY;
  bool bad = false;                                               // a NaN among the teacher's logits
  for (int k = lane; k < K; k += 64)
    if (sid[k] >= 0) { tm = fmaxf(tm, slog[k]); bad |= slog[k] != slog[k]; }
  tm = wave_max(tm);
  if (__any(bad)) tm = NAN;
  const bool some = tm != -INFINITY;
  if (lane == 0) {
    p.L1[i] = L1;
    p.L2[i] = L2;
    p.slive[n % p.R] = 1;
    p.hard[n] = (sid[K] >= 0 ? -log_share(spick[K] - L1) : L1) * LN2;   // (outside the vocabulary: a logit of 0)
    p.some[i] = K == 0 || !some ? 0.f : tm != tm ? NAN : 1.f;
  }
  float* share = p.share + (long)i * (K + 1);
  float sum = 0.f;
  for (int k = lane; k < K; k += 64)
    if (some && sid[k] >= 0) sum += __builtin_amdgcn_exp2f((slog[k] - tm) * p.itau * LOG2E);
  sum = wave_sum(sum);
  const float lsum = log2f(sum), inv = 1.0f / sum;
  float loss = 0.f;
  bool listed = false;
  for (int k = lane; k < K; k += 64) {
    const float lp = (slog[k] - tm) * p.itau * LOG2E, pk = some && sid[k] >= 0 ? __builtin_amdgcn_exp2f(lp) * inv : 0.f;
    if (pk != 0.f) loss += pk * (lp - lsum - log_share(fmaf(spick[k], p.itau, -L2)));
    listed |= sid[k] >= 0 && sid[k] == sid[K];
    slog[k] = pk;                                                 // (its own lane's entry) from here on: p_k
  }
  loss = wave_sum(loss);
  if (lane == 0 && K) p.soft[n] = p.tau * p.tau * LN2 * loss;
  const bool tgt_listed = __any(listed);
  if (lane == 0) share[K] = tgt_listed ? -1.f : 0.f;
  // an id listed several times is one entry of the gradient: its first place holds the sum of the shares, the others -1
  // (as does the target's own place, K, if the teacher lists it)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int k = lane; k < K; k += 64) {
    const int id = sid[k];
    int f = -1;
    if (id >= 0) {
      unsigned h = table_slot(id, bits);
      while (sid[f = table[h]] != id) h = (h + 1) & (size - 1);
      if (f != k) atomicOr(&multi[f >> 5], 1u << (f & 31));
    }
    spick[k] = __int_as_float(f);                                 // (its own lane's entry, no longer needed)
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  for (int k = lane; k < K; k += 64) {
    const bool first = __float_as_int(spick[k]) == k;
    float all = slog[k];
    if (first && (multi[k >> 5] >> (k & 31) & 1))
      for (int q = k + 1; q < K; ++q)
        if (sid[q] == sid[k]) all += slog[q];
    share[k] = first ? all : -1.f;
  }
}

// a wave per sentence: out[r] = sum over t, of the hard rows and (blockIdx.y = 1) the soft ones (5 us: launch and latency)
__global__ __launch_bounds__(256) void dt_sum_kernel(int T, int R, const float* __restrict__ h, const float* __restrict__ f,
                                                     float* __restrict__ hard, float* __restrict__ soft) {
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (r >= R) return;
  const float* x = blockIdx.y ? f : h;
  float s = 0.f;
  for (int t = lane; t < T; t += 64) s += x[(long)t * R + r];
  s = wave_sum(s);
  if (lane == 0) (blockIdx.y ? soft : hard)[r] = s;
}

// ------------------------------------------------------------------------------------------------- backward
// |upstream gradient| of a sentence's rows (0: no live row, or no number)
__device__ __forceinline__ float sentence_grad(const DistillArgs& p, int r) {
  if (!p.slive[r]) return 0.f;
  const float x = fabsf(p.ghard[r]) + (p.K ? fabsf(p.gsoft[r]) * p.tau : 0.f);
  return x < 3.4e38f ? x : 0.f;
}
// Partial maxima of it.  The kernel behind needs the largest in every block of 16 rows: up to DT_GSCAN sentences each block looks at
// them all, more are looked at once, here.  65536 rows of E = 64: 1024 sentences 24 us in every block, 2048 28; with partials 2 here
// and 19 there.  A flat batch (T = 1) has as many sentences as rows: 240 us without them, and four times that for twice the rows.
constexpr int DT_GPART = 256, DT_GSCAN = 1024;
__global__ __launch_bounds__(256) void dt_gmax_kernel(DistillArgs p) {
  __shared__ float red[4];
  float g = 0.f;
  for (int r = blockIdx.x * 256 + threadIdx.x; r < p.R; r += DT_GPART * 256) g = fmaxf(g, sentence_grad(p, r));
  g = wave_max(g);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = g;
  __syncthreads();
  if (threadIdx.x == 0) p.gpart[blockIdx.x] = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
}

// Per live row: the two coefficients of its gradient over the row's power of two s, and the image of s X (with a column
// of s itself: the product with P gives the bias gradient beside the weights').  Zeros: dX of dead rows, image rows past
// the last live one.  16 rows a block: blocks [0, nx) original rows, the next Np / 16 the image's tail.  9 us for 7680 rows of
// 200, 15 for 4096 of 1024: latency.
template <typename T, int NP> __global__ __launch_bounds__(256) void dt_gimage_kernel(DistillArgs p, int nx) {
  __shared__ float red[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long ld = (long)p.Kg * NP;
  const int nl = *p.nlive;
  const T* row[4];
  _Float16* to[4];
  int ee[4];
  if ((int)blockIdx.x >= nx) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int i = (blockIdx.x - nx) * 16 + wave * 4 + q;
      row[q] = nullptr;
      to[q] = i >= nl ? p.Gimg + i * ld : nullptr;
      ee[q] = 0;
    }
    image_rows<T, NP>(row, to, p.E, p.Kg / 4, false, ee, lane, 0.f);
    return;
  }
  float g = 0.f;
  static_assert(DT_GPART == 256, "one partial a thread");
  if (p.gpart) g = p.gpart[threadIdx.x];
  else for (int r = threadIdx.x; r < p.R; r += 256) g = fmaxf(g, sentence_grad(p, r));
  g = wave_max(g);
  if (lane == 0) red[wave] = g;
  __syncthreads();
  g = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  const int eg = g > 0.f ? (int)ceilf(log2f(g)) : 0;              // gmax = 2^eg
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.gmax = ldexpf(1.f, eg);
  const int ex = p.sexp[0];
  const bool vec = p.E % 4 == 0 && ((uintptr_t)p.X % (4 * sizeof(T))) == 0;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int n = blockIdx.x * 16 + wave * 4 + q;
    const int i = n < p.N ? p.inv[n] : -1;
    row[q] = nullptr;
    to[q] = nullptr;
    ee[q] = 0;
    if (i < 0) {
      T* z = static_cast<T*>(p.dX) + (long)n * p.E;
      if (n < p.N && p.dX)
        for (int k = lane; k < p.E; k += 64) z[k] = (T)0.f;
      continue;
    }
    const int r = n % p.R;
    const float gh = p.ghard[r], some = p.some[i];                // no soft part where the teacher lists nothing
    const float gs = !p.K || some == 0.f ? 0.f : some != some ? some : p.gsoft[r] * p.tau;
    const float mag = fabsf(gh) + fabsf(gs);
    int es = (mag > 0.f && mag < 3.4e38f) ? (int)ceilf(log2f(mag)) : eg;
    es = es > eg ? eg : (es < eg - 40 ? eg - 40 : es);
    if (lane == 0) {
      p.coef[i] = ldexpf(gh, P_EXP - es);
      p.coef[p.Np + i] = ldexpf(gs, P_EXP - es);
      p.coef[2 * (long)p.Np + i] = ldexpf(1.f, es);
    }
    row[q] = static_cast<const T*>(p.X) + (long)n * p.E;
    to[q] = p.Gimg + i * ld;
    ee[q] = ex + es - eg;
  }
  image_rows<T, NP>(row, to, p.E, p.Kg / 4, vec, ee, lane, ldexpf(1.f, P_EXP - ex));
}

// P[n][v] of a piece of the vocabulary without the picked entries: a 2^(t - L1) + b 2^(t / tau - L2), for any E: the forward
// walk's product, once a 128 x 128 tile.  The tile goes through LDS so that rows leave whole.  3650 rows x 1024 x 50000 bf16:
// 474 us, 0.79 PFLOP/s and 365 MB written.  (As a walk like the forward one 560: a stage's wait would count the stores.)
template <int NP, int NQ, bool TWO>
__global__ __launch_bounds__(256, 2) void dt_grad_kernel(DistillArgs p) {
  DT_LDS
  const int nl = *p.nlive, nt = (nl + DT_TILE - 1) / DT_TILE, vt = (p.vc + DT_TILE - 1) / DT_TILE;
  // block -> (vocabulary tile, row tile): an XCD walks its own range of W, all row tiles of one tile of W in turn
  const int pv = (vt + 7) / 8, j0 = blockIdx.x >> 3;
  if (j0 >= nt * pv) return;
  int tn, tv;
  walk_order(j0, nt, pv, tn, tv);
  tv += (blockIdx.x & 7) * pv;
  if (tv >= vt) return;
  const int n0 = tn * DT_TILE, w0 = p.v0 + tv * DT_TILE;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int am = (wave >> 1) * 64, bn = (wave & 1) * 64;
  const long ld = (long)p.Kp * NP * 2;
  using Op = Operand<NP, false, DT_TILE, 4>;
  Op A, B;
  A.init(reinterpret_cast<const char*>(p.Wimg) + w0 * ld, ld, 128, lane, wave);
  B.init(reinterpret_cast<const char*>(p.Ximg) + n0 * ld, ld, 128, lane, wave);
  const int nst = (p.E + 64 / NP - 1) / (64 / NP), last = ((p.E + 15) / 16) - (nst - 1) * (4 / NP);
  const float c = unscale(p.sexp);
  f32x16 acc[2][2];
  clear(acc);
  A.issue(0, la0, wave);
  B.issue(0, lb0, wave);
  stages<Op, Op>(A, B, nst, last, la0, lb0, la1, lb1, am, bn, lane, wave, acc, [](char*, char*) {});
  __syncthreads();
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int nn = bn + 32 * j + (lane & 31), i = n0 + nn;
    const bool in = i < nl;
    const float L1 = in ? p.L1[i] : 0.f, L2 = (TWO && in) ? p.L2[i] : 0.f;
    const float ca = in ? p.coef[i] + (TWO ? 0.f : p.coef[p.Np + i]) : 0.f, cb = (TWO && in) ? p.coef[p.Np + i] : 0.f;
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int v = am + 32 * q + 8 * g + 4 * (lane >> 5);
        const float4 bb = *reinterpret_cast<const float4*>(p.b2 + w0 + v);
        const float bv[4] = {bb.x, bb.y, bb.z, bb.w};
        Packed<f16_t, 4> hi, lo;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float t = fmaf(acc[q][j][4 * g + k], c, bv[k]);
          float x = ca * __builtin_amdgcn_exp2f(t - L1);
          if (TWO) x = fmaf(cb, __builtin_amdgcn_exp2f(fmaf(t, p.itau, -L2)), x);
          x = in ? x : 0.f;
          if (NQ == 2) one_value(x);
          hi.set(k, x);
          if (NQ == 2) lo.set(k, x - hi.f(k));
        }
        const int byte = NQ == 1 ? v * 2 : (v >> 5) * 128 + (v & 31) * 2;
        char* row = DT_AREA(nn * NQ >> 6) + (nn * 256 * NQ & (DT_STAGE - 1));
        *reinterpret_cast<Packed<f16_t, 4>*>(row + ((((byte >> 4) ^ (nn & 15)) << 4) | (byte & 15))) = hi;
        if (NQ == 2) {
          const int bl = byte + 64;
          *reinterpret_cast<Packed<f16_t, 4>*>(row + ((((bl >> 4) ^ (nn & 15)) << 4) | (bl & 15))) = lo;
        }
      }
  }
  __syncthreads();
  char* P = reinterpret_cast<char*>(p.P) + ((long)tv * 2 * NQ * p.Np + n0) * 128;
  for (int k = threadIdx.x; k < DT_TILE * 16 * NQ; k += 256) {    // piece by piece, its 128 rows in one run of memory
    const int g = k >> 10, nn = (k >> 3) & 127, ch = g * 8 + (k & 7);
    const uint4 x = *reinterpret_cast<const uint4*>(DT_AREA(nn * NQ >> 6) + (nn * 256 * NQ & (DT_STAGE - 1)) + ((ch ^ (nn & 15)) << 4));
    *reinterpret_cast<uint4*>(P + (long)g * p.Np * 128 + (k & 1023) * 16) = x;
  }
}

// The picked entries of a row, from their own fp32 logits: softmax minus the target / the teacher's share (an id that
// was listed before, or a target that the teacher lists, has share -1 here: its first place writes it).  A wave a row, one
// scattered store an entry: 9 us for 4815 rows of 65.
template <int NQ, bool TWO>
__global__ __launch_bounds__(256) void dt_pick_kernel(DistillArgs p) {
  const int i = blockIdx.x * 4 + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  if (i >= *p.nlive) return;
  const long at = position(p, p.rows[i]);
  const int64_t* ids = p.K ? p.ids + at * p.K : nullptr;
  const int64_t tg = p.eos[at];
  const float a = p.coef[i], b = p.coef[p.Np + i], L1 = p.L1[i], L2 = p.L2[i];
  for (int k = lane; k <= p.K; k += 64) {
    const int64_t id = k < p.K ? ids[k] : tg;
    const float share = p.share[(long)i * (p.K + 1) + k], pick = p.pick[(long)i * (p.K + 1) + k];
    if (id < p.v0 || id >= (int64_t)p.v0 + p.vc || id >= p.V || share == -1.f) continue;
    float x = a * (__builtin_amdgcn_exp2f(log_share(pick - L1)) - (id == tg ? 1.f : 0.f));
    if (p.K) x = fmaf(b, __builtin_amdgcn_exp2f(log_share(fmaf(pick, TWO ? p.itau : 1.f, -L2))) - share, x);
    const int v = (int)(id - p.v0);
    _Float16* q = p.P + ((long)(v * NQ >> 6) * p.Np + i) * 64 + (v & (64 / NQ - 1));
    if (NQ == 2) one_value(x);
    const _Float16 hi = (_Float16)x;
    q[0] = hi;
    if (NQ == 2) q[32] = (_Float16)(x - (float)hi);
  }
}

// Splits of the vocabulary for the dX product's tiles (known on the device alone): a block a CU, items in rounds of 256; an
// item costs its stages and about 14 more for its partial tile's way out and back.  dW's tiles follow on the same CUs and need
// not come out even (157 of them for a vocabulary of 20000).  With two planes of W, where a stage is matrix work, as many splits
// as there are CUs spared in dW's last round are therefore longer by a tile of dW, if dX's items are one round (also where only
// dX is wanted: its bits do not depend on that): 3520 x 200 x 20000 fp32 131 -> 116 us for both products.  With one plane a
// stage is memory work, twice as long in dX as in dW, and even splits are better (4815 x 200 x 50000 bf16: 140 us a range, 173).
template <int NP> __device__ __forceinline__ Splits dt_dx_splits(const DistillArgs& p, int tiles, int stages, int nl, int bk) {
  const DxSplit mine = dx_split((threadIdx.x & 63) + 1, tiles, stages, (nl + bk - 1) / bk + 6, p.dwtiles, NP == 2);
  int best = mine.cost;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) best = min(best, __shfl_xor(best, o, 64));
  const int lane = best & 63;
  return dx_splits_of(__builtin_amdgcn_readfirstlane(lane + 1), __builtin_amdgcn_readfirstlane(__shfl(mine.size, lane, 64)),
                      __builtin_amdgcn_readfirstlane(__shfl(mine.longer, lane, 64)), stages);
}

// dX: (W down its rows: K = vocabulary) x (P along its rows), tiles of RA columns of E x RB rows.  Items (tile, split of
// the range): partial tiles in accumulator order, added to what an earlier range left there.
template <int NP, int NQ, int RA>
__device__ __forceinline__ void dx_items(const DistillArgs& p, const Ring& m, int first, int et, int add) {
  constexpr int RB = 384 - RA, BK = 64 / NQ;
  const int nl = *p.nlive, tiles = (nl + RB - 1) / RB * et;
  const Splits splits = dt_dx_splits<NP>(p, tiles, p.vfull / BK, nl, BK);
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int stages = p.vc / BK;
  const long ldw = (long)p.Kp * NP * 2;
  using OA = Operand<NP, true, RA, 8, BK>;
  using OB = Operand<NQ, false, RB, 8>;
  OA A;
  OB B;
  A.init(nullptr, ldw, 128, lane, wave);
  B.init(nullptr, 128, (long)p.Np * 128, lane, wave);
  for (int item = first; item < tiles * splits.n; item += DT_DX_BLOCKS) {
    const int split = item / tiles, tile = item - split * tiles, te = tile % et, tn = tile / et;
    const int s0 = min(stages, splits.begin(split)), s1 = min(stages, splits.begin(split + 1));   // (the last range may be shorter)
    A.base = reinterpret_cast<const char*>(p.Wimg) + (p.v0 + (long)s0 * BK) * ldw + (long)te * RA * 2 * NP;
    B.base = reinterpret_cast<const char*>(p.P) + ((long)s0 * p.Np + tn * RB) * 128;
    f32x16 acc[4];
    const Part<RA> t(__builtin_amdgcn_readfirstlane(p.E - te * RA), wave);
    tile_product<RA, 0>(A, B, s1 - s0, m, t, lane, acc);
    float4* out = reinterpret_cast<float4*>(p.slab) + ((long)split * tiles + tile) * (RA * RB / 4) + wave * 1024 + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!t.has(i)) continue;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        float4* q = out + (i * 4 + g) * 64;
        float4 x = make_float4(acc[i][4 * g], acc[i][4 * g + 1], acc[i][4 * g + 2], acc[i][4 * g + 3]);
        if (add) { const float4 y = *q; x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w; }
        *q = x;
      }
    }
  }
}
// dX from the splits' partial tiles, always in the same order: the result does not depend on which block came first.  11 us for
// 4815 x 200, 19 for 3650 x 1024 (the partial tiles are still in the caches).
template <typename T, int NQ, int RA>
__global__ __launch_bounds__(256) void dt_dx_sum_kernel(DistillArgs p, int et) {
  constexpr int RB = 384 - RA;
  const int nl = *p.nlive, tiles = (nl + RB - 1) / RB * et;
  const int tile = blockIdx.x >> 5;                               // 32 blocks a tile
  if (tile >= tiles) return;
  const int splits = dt_dx_splits<sizeof(T) == 4 ? 2 : 1>(p, tiles, p.vfull / (64 / NQ), nl, 64 / NQ).n;
  const float w = ldexpf(1.f, -p.sexp[1] - P_EXP);
  const int slot = (blockIdx.x & 31) * 256 + threadIdx.x;
  const long step = (long)tiles * (RA * RB / 4);
  const float4* q = reinterpret_cast<const float4*>(p.slab) + (long)tile * (RA * RB / 4) + slot;
  const int lane = slot & 63, frag = (slot >> 6) & 15, wave = slot >> 10;
  const int te = tile % et;
  const Part<RA> t(p.E - te * RA, wave);
  const int i = (tile / et) * RB + t.row(frag >> 2) + (lane & 31);
  const int e = te * RA + t.col(frag >> 2) + (frag & 3) * 8 + (lane >> 5) * 4;
  if (i >= nl || e >= p.E || !t.has(frag >> 2)) return;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int k = 0; k < splits; ++k) { const float4 y = q[k * step]; s.x += y.x; s.y += y.y; s.z += y.z; s.w += y.w; }
  const float f = w * p.coef[2 * (long)p.Np + i];
  T* out = static_cast<T*>(p.dX) + (long)p.rows[i] * p.E + e;
  const float v[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (e + k < p.E) out[k] = (T)(v[k] * f);
}

// dW and db: (s X down its rows: K = live rows) x (P down its rows), tiles of RA columns of E x RB words, whole K in one
// block.  fp32: chains of 24 stages (768 rows), joined: relative error of dW and db at 131072 x 200 x 512 3.6e-7 and 1.9e-7 (one chain
// 5.5e-6 and 5.9e-7; at 8192 rows 3.1e-7 and 6e-8 against 9.9e-7 and 4.2e-7), no time measured for it.  16-bit gradients round by more.
template <typename T, int NP, int NQ, int RA>
__device__ __forceinline__ void dw_tile(const DistillArgs& p, const Ring& m, int block, int et) {
  constexpr int RB = 384 - RA, BK = 64 / NQ;
  const int nl = *p.nlive, vt = p.vc / RB;
  const int pv = (vt + 7) / 8, j0 = block >> 3, tv = (block & 7) * pv + j0 / et, te = j0 % et;
  if (j0 / et >= pv || tv >= vt) return;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  using OA = Operand<NP, true, RA, 8, BK>;
  using OB = Operand<NQ, true, RB, 8>;
  OA A;
  OB B;
  A.init(reinterpret_cast<const char*>(p.Gimg) + (long)te * RA * 2 * NP, (long)p.Kg * NP * 2, 128, lane, wave);
  B.init(reinterpret_cast<const char*>(p.P) + (long)(tv * RB / BK) * p.Np * 128, 128, (long)p.Np * 128, lane, wave);
  const float fw = *p.gmax * ldexpf(1.f, -P_EXP - p.sexp[0]), fb = *p.gmax * ldexpf(1.f, -2 * P_EXP);
  f32x16 acc[4];
  const Part<RA> t(__builtin_amdgcn_readfirstlane(p.E + 1 - te * RA), wave);   // (the bias' column too)
  tile_product<RA, sizeof(T) == 4 ? 24 : 0>(A, B, (nl + BK - 1) / BK, m, t, lane, acc);
  // a lane holds four neighbouring columns of a word's row at a time
  const bool vec = p.E % 4 == 0 && ((uintptr_t)p.dW % (4 * sizeof(T))) == 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int v = p.v0 + tv * RB + t.row(i) + (lane & 31);
    if (v >= p.V || !t.has(i)) continue;
    T* out = static_cast<T*>(p.dW) + (long)v * p.E;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int e = te * RA + t.col(i) + 8 * g + 4 * (lane >> 5);
      if (vec && e + 3 < p.E) {
        Packed<T, 4> x;
#pragma unroll
        for (int k = 0; k < 4; ++k) x.set(k, acc[i][4 * g + k] * fw);
        *reinterpret_cast<Packed<T, 4>*>(out + e) = x;
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
          if (e + k < p.E) out[e + k] = (T)(acc[i][4 * g + k] * fw);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (e + k == p.E) static_cast<T*>(p.db)[v] = (T)(acc[i][4 * g + k] * fb);
    }
  }
}

// Both products of a range in one launch, dX's items in the first DT_DX_BLOCKS blocks (one a CU), dW's tiles behind them:
// the CUs that one of them leaves idle at its end work on the other.  256 x 128 tiles of eight waves, three buffers, P read once
// by each product from the caches that the range was sized for.  3650 x 1024 x 50000 bf16: 755 us for both, 0.99 PFLOP/s;
// matrix cores busy 61 % of the time at the 1.71 GHz that their power leaves.  By the memory counters 3.5 GB read
// and 0.14 written, 4.9 TB/s.  4815 x 200 x 50000: 290 us in two ranges, 0.66 PFLOP/s, matrix cores busy 33 %, bound by P: a range of
// 240 MB is read by each product, with W and the partial tiles 652 MB read and 36 written, 4.7 TB/s.
template <typename T, int NP, int NQ, int RAX, int RAW>
__global__ __launch_bounds__(512, 2) void dt_products_kernel(DistillArgs p, int etx, int etw, int add) {
  __shared__ __attribute__((aligned(16))) char x0[32768];
  __shared__ __attribute__((aligned(16))) char x1[32768];
  __shared__ __attribute__((aligned(16))) char x2[32768];
  __shared__ __attribute__((aligned(16))) char y0[16384];
  __shared__ __attribute__((aligned(16))) char y1[16384];
  __shared__ __attribute__((aligned(16))) char y2[16384];
  const Ring m = {x0, x1, x2, y0, y1, y2};
  const int behind = p.dX ? DT_DX_BLOCKS : 0;                     // either product may not be wanted
  if ((int)blockIdx.x < behind) dx_items<NP, NQ, RAX>(p, m, blockIdx.x, etx, add);
  else dw_tile<T, NP, NQ, RAW>(p, m, blockIdx.x - behind, etw);
}

// ------------------------------------------------------------------------------------------------- host side
constexpr long DT_PIECE_BYTES = 400L << 20;        // of P: it is written, then read twice (4815 x 200 x 50000 bf16, both passes: 110 MiB
                                                   // 1045 us, 200 868, 300 798, 400 773, 900 777 and twice the workspace)

struct DistillPlan {
  long bytes, back_bytes;
  long hard, soft, counts, rows, inv, nlive, slive, amax, sexp, Ximg, Wimg, b2, L1, L2, some, pick, share, part;   // offsets in bytes
  long Gimg, coef, gmax, gpart, P, slab;
  int np, nq, Np, Vp, Kp, Kg, nb, nk, fvt, rax, raw, et, etw;
  long vc, pplane;
};
static DistillPlan dt_plan(int dtype, long N, int E, int V, int K) {
  DistillPlan d = {};
  d.np = dtype == DT_F32 ? 2 : 1;
  d.nq = dtype == DT_BF16 ? 1 : 2;                  // planes of P
  d.Np = (int)((N + 255) / 256 * 256); d.Vp = (V + 255) / 256 * 256; d.nk = E <= 64 ? 4 : E <= 128 ? 8 : E <= 208 ? 13 : 0;
  d.Kp = d.nk == 13 ? 256 : (E + 63) / 64 * 64; d.Kg = (E + 64) / 64 * 64;
  d.nb = cdiv(N, DT_CROWS);
  // the gradient products' tiles, 256 columns of E x 128 rows or words or 128 x 256: what pads E less
  d.rax = (E + 255) / 256 * 256 == (E + 127) / 128 * 128 ? 256 : 128;
  d.raw = (E + 256) / 256 * 256 == (E + 128) / 128 * 128 ? 256 : 128;
  d.et = cdiv(E, d.rax); d.etw = cdiv(E + 1, d.raw);
  const int nt = d.Np / DT_TILE;
  d.fvt = d.Vp / (d.nk ? DT_TILE / d.np : DT_TILE);
  const int ranges = d.fvt / 8 < 1 ? 1 : (d.fvt / 8 > 64 ? 64 : d.fvt / 8);        // of an XCD at most (dt_splits)
  const long items = (long)nt * ranges < DT_MOST_ITEMS ? (long)nt * ranges : DT_MOST_ITEMS;
  d.pplane = 8L * (nt > items ? nt : items) * 128;
  auto take = [](long& at, long bytes) { const long o = at; at += (bytes + 255) / 256 * 256; return o; };
  long at = 0;
  d.hard = take(at, 4 * N); d.soft = take(at, K ? 4 * N : 0);
  d.counts = take(at, 4L * (d.nb + 1)); d.rows = take(at, 4 * N); d.inv = take(at, 4 * N); d.nlive = take(at, 4);
  d.slive = take(at, 4 * N);
  d.amax = take(at, 8L * DT_AMAX); d.sexp = take(at, 8);
  const long slack = 2048;                          // a column tile of the last row may be read past the row's end
  d.Ximg = take(at, 2L * d.Np * d.Kp * d.np); d.Wimg = take(at, 2L * d.Vp * d.Kp * d.np + slack);
  d.b2 = take(at, 4L * d.Vp);
  d.L1 = take(at, 4L * d.Np); d.L2 = take(at, 4L * d.Np);
  d.some = take(at, 4L * d.Np);
  d.pick = take(at, 4L * N * (K + 1)); d.share = take(at, 4L * N * (K + 1));
  d.part = take(at, 12L * d.pplane);
  d.bytes = at;
  long vc = DT_PIECE_BYTES / (2L * d.nq * d.Np) / 256 * 256;
  if (vc < 1024) vc = 1024;
  const int pieces = cdiv(d.Vp, vc);
  d.vc = ((long)d.Vp / 256 + pieces - 1) / pieces * 256;          // ranges of equal size
  const int tiles = d.Np / (384 - d.rax) * d.et;
  at = 0;
  d.Gimg = take(at, 2L * d.Np * d.Kg * d.np + slack); d.coef = take(at, 12L * d.Np); d.gmax = take(at, 4); d.gpart = take(at, 4L * DT_GPART);
  d.P = take(at, 2L * d.Np * d.vc * d.nq);
  d.slab = take(at, 4L * 32768 * dx_partial_tiles(tiles, (int)(d.vc * d.nq / 64)));
  d.back_bytes = at;
  return d;
}
// (a launch has fewer than 2^32 threads: 256 a row in the merge, 16 a word in the images)
static bool dt_sizes_ok(long N, long E, long V, long K) {
  return N <= (1L << 23) && E > 0 && E <= 65536 && V > 0 && V <= (1L << 26) && K >= 0 && K <= V && K <= DT_MOST_K;
}
// 0 where there are no rows, or for sizes that the calls refuse
long distill_workspace_floats(int dtype, long N, long E, long V, long K) {
  return N > 0 && dt_sizes_ok(N, E, V, K) ? dt_plan(dtype, N, (int)E, (int)V, (int)K).bytes / 4 : 0;
}
long distill_backward_workspace_floats(int dtype, long N, long E, long V, long K) {
  return N > 0 && dt_sizes_ok(N, E, V, K) ? dt_plan(dtype, N, (int)E, (int)V, (int)K).back_bytes / 4 : 0;
}

static int dt_check(const char* what, const DistillCall& c) {
  CVAE_REQUIRE(c.dtype >= DT_F32 && c.dtype <= DT_F16, "%s: dtype %d is none of 0 (fp32), 1 (bf16), 2 (fp16)", what, c.dtype);
  CVAE_REQUIRE(c.B > 0 && c.T >= 0 && c.R >= 0 && c.R % c.B == 0, "%s: R = %d must be a multiple of B = %d", what, c.R, c.B);
  CVAE_REQUIRE(dt_sizes_ok((int64_t)c.T * c.R, c.E, c.V, c.K), "%s: bad shape T=%d R=%d E=%d V=%lld K=%d", what, c.T, c.R,
               c.E, (long long)c.V, c.K);
  // (below, S / tau has no bits left in fp32, and its exponentials overflow in the gradient)
  CVAE_REQUIRE(c.K == 0 || (c.tau >= 1e-6f && c.tau < 1e6f), "%s: tau must be in [1e-6, 1e6)", what);
  return 0;
}
static void dt_fill(DistillArgs& a, const DistillPlan& d, const DistillCall& c, void* ws) {
  a.N = c.T * c.R; a.T = c.T; a.R = c.R; a.B = c.B; a.E = c.E; a.V = (int)c.V; a.K = c.K;
  a.Np = d.Np; a.Vp = d.Vp; a.Kp = d.Kp; a.Kg = d.Kg;
  a.tau = c.K ? c.tau : 1.f; a.itau = 1.f / a.tau;
  a.two = c.K > 0 && a.tau != 1.f;
  a.X = c.X; a.W = c.W; a.bias = c.b; a.eos = c.eos; a.pad = c.pad; a.per = c.sentence_major ? c.R / c.B : 0; a.ids = c.ids; a.top = c.top;
  char* w = static_cast<char*>(ws);
  a.hard = (float*)(w + d.hard); a.soft = (float*)(w + d.soft);
  a.counts = (int*)(w + d.counts); a.scanned = d.nb > DT_CSCAN; a.rows = (int*)(w + d.rows); a.inv = (int*)(w + d.inv); a.nlive = (int*)(w + d.nlive); a.slive = (int*)(w + d.slive);
  a.amax = (float*)(w + d.amax); a.sexp = (int*)(w + d.sexp); a.Ximg = (_Float16*)(w + d.Ximg); a.Wimg = (_Float16*)(w + d.Wimg); a.b2 = (float*)(w + d.b2);
  a.L1 = (float*)(w + d.L1); a.L2 = (float*)(w + d.L2); a.some = (float*)(w + d.some);
  a.pick = (float*)(w + d.pick); a.share = (float*)(w + d.share);
  a.part = (float*)(w + d.part); a.pplane = d.pplane; a.fvt = d.fvt; a.least = d.nk ? 1 : 8;
}

template <int NP, int NQ, bool TWO, bool GRAD> static void dt_rows(int nk, const DistillArgs& a, hipStream_t s) {
  const dim3 grid(DT_WALK_BLOCKS);
  if (nk == 4) hipLaunchKernelGGL((dt_rows_kernel<NP, NQ, TWO, GRAD, 4>), grid, dim3(256), 0, s, a);
  else if (nk == 8) hipLaunchKernelGGL((dt_rows_kernel<NP, NQ, TWO, GRAD, 8>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((dt_rows_kernel<NP, NQ, TWO, GRAD, 13>), grid, dim3(256), 0, s, a);
}
template <typename T, int NP, bool TWO> static int dt_forward(const DistillPlan& d, const DistillArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((dt_count_kernel<T>), dim3(d.nb + 2 * DT_AMAX), dim3(256), 0, s, a, d.nb);
  CVAE_LAUNCH_CHECK("dt_count_kernel");
  if (a.scanned) {
    hipLaunchKernelGGL(dt_scan_kernel, dim3(1), dim3(1024), 0, s, a, d.nb);
    CVAE_LAUNCH_CHECK("dt_scan_kernel");
  }
  hipLaunchKernelGGL((dt_image_kernel<T, NP>), dim3(cdiv(a.N, 16) + d.Np / 16 + d.Vp / 16), dim3(256), 0, s, a, cdiv(a.N, 16));
  CVAE_LAUNCH_CHECK("dt_image_kernel");
  if (d.nk) dt_rows<NP, 1, TWO, false>(d.nk, a, s);
  else hipLaunchKernelGGL((dt_forward_kernel<NP, TWO>), dim3(DT_WALK_BLOCKS), dim3(256), 0, s, a);
  CVAE_LAUNCH_CHECK("dt_forward_kernel");
  hipLaunchKernelGGL((dt_combine_kernel<T, TWO>), dim3(a.N), dim3(256), 4 * dt_combine_words(a.K), s, a);
  CVAE_LAUNCH_CHECK("dt_combine_kernel");
  return 0;
}
template <typename T, int NP, int NQ, bool TWO> static int dt_backward(const DistillPlan& d, DistillArgs a, hipStream_t s) {
  const int nx = cdiv(a.N, 16), nt = d.Np / DT_TILE;
  if (a.gpart) {
    hipLaunchKernelGGL(dt_gmax_kernel, dim3(DT_GPART), dim3(256), 0, s, a);
    CVAE_LAUNCH_CHECK("dt_gmax_kernel");
  }
  hipLaunchKernelGGL((dt_gimage_kernel<T, NP>), dim3(nx + d.Np / 16), dim3(256), 0, s, a, nx);
  CVAE_LAUNCH_CHECK("dt_gimage_kernel");
  for (long v0 = 0; v0 < d.Vp; v0 += d.vc) {
    a.v0 = (int)v0;
    a.vc = (int)(d.Vp - v0 < d.vc ? d.Vp - v0 : d.vc);
    const int vt = cdiv(a.vc, DT_TILE);
    if (d.nk) dt_rows<NP, NQ, TWO, true>(d.nk, a, s);
    else hipLaunchKernelGGL((dt_grad_kernel<NP, NQ, TWO>), dim3((unsigned)((long)cdiv(vt, 8) * 8 * nt)), dim3(256), 0, s, a);
    CVAE_LAUNCH_CHECK("dt_grad_kernel");
    hipLaunchKernelGGL((dt_pick_kernel<NQ, TWO>), dim3(cdiv(a.N, 4)), dim3(256), 0, s, a);
    CVAE_LAUNCH_CHECK("dt_pick_kernel");
    const dim3 grid((unsigned)((a.dX ? DT_DX_BLOCKS : 0) + (a.dW ? (long)cdiv(a.vc / (384 - d.raw), 8) * 8 * d.etw : 0)));
    const int add = v0 > 0 ? 1 : 0;
    if (d.rax == 256 && d.raw == 256) hipLaunchKernelGGL((dt_products_kernel<T, NP, NQ, 256, 256>), grid, dim3(512), 0, s, a, d.et, d.etw, add);
    else if (d.rax == 256) hipLaunchKernelGGL((dt_products_kernel<T, NP, NQ, 256, 128>), grid, dim3(512), 0, s, a, d.et, d.etw, add);
    else if (d.raw == 256) hipLaunchKernelGGL((dt_products_kernel<T, NP, NQ, 128, 256>), grid, dim3(512), 0, s, a, d.et, d.etw, add);
    else hipLaunchKernelGGL((dt_products_kernel<T, NP, NQ, 128, 128>), grid, dim3(512), 0, s, a, d.et, d.etw, add);
    CVAE_LAUNCH_CHECK("dt_products_kernel");
  }
  if (!a.dX) return 0;
  const dim3 gs((unsigned)((long)(d.Np / (384 - d.rax)) * d.et * 32));
  if (d.rax == 256) hipLaunchKernelGGL((dt_dx_sum_kernel<T, NQ, 256>), gs, dim3(256), 0, s, a, d.et);
  else hipLaunchKernelGGL((dt_dx_sum_kernel<T, NQ, 128>), gs, dim3(256), 0, s, a, d.et);
  CVAE_LAUNCH_CHECK("dt_dx_sum_kernel");
  return 0;
}
template <typename T, int NP, int NQ> static int dt_run(const DistillPlan& d, const DistillArgs& a, bool back, hipStream_t s) {
  if (back) return a.two ? dt_backward<T, NP, NQ, true>(d, a, s) : dt_backward<T, NP, NQ, false>(d, a, s);
  return a.two ? dt_forward<T, NP, true>(d, a, s) : dt_forward<T, NP, false>(d, a, s);
}
static int dt_dispatch(int dtype, const DistillPlan& d, const DistillArgs& a, bool back, hipStream_t s) {
  if (dtype == DT_F32) return dt_run<float, 2, 2>(d, a, back, s);
  return dtype == DT_BF16 ? dt_run<bf16_t, 1, 1>(d, a, back, s) : dt_run<f16_t, 1, 2>(d, a, back, s);
}

int launch_distill_forward(const DistillCall& c, float* hard, float* soft, void* ws, hipStream_t s) {
  CVAE_TRY(dt_check("distill_forward", c));
  if (c.R == 0) return 0;
  CVAE_REQUIRE(hard && (c.K == 0 || soft), "distill_forward: null operand");
  DistillArgs a = {};
  if (c.T > 0) {
    CVAE_REQUIRE(c.X && c.W && c.b && c.eos && ws && (c.K == 0 || (c.ids && c.top)), "distill_forward: null operand");
    CVAE_REQUIRE(((uintptr_t)ws & 15) == 0, "distill_forward: the workspace must be 16-byte aligned");
    const DistillPlan d = dt_plan(c.dtype, (long)c.T * c.R, c.E, (int)c.V, c.K);
    dt_fill(a, d, c, ws);
    CVAE_TRY(dt_dispatch(c.dtype, d, a, false, s));
  }
  hipLaunchKernelGGL(dt_sum_kernel, dim3(cdiv(c.R, 4), c.K ? 2 : 1), dim3(256), 0, s, c.T, c.R, a.hard, a.soft, hard, soft);
  CVAE_LAUNCH_CHECK("dt_sum_kernel");
  return 0;
}

int launch_distill_backward(const DistillCall& c, const float* ghard, const float* gsoft, const void* saved, void* dX,
                            void* dW, void* db, void* ws, hipStream_t s) {
  CVAE_TRY(dt_check("distill_backward", c));
  CVAE_REQUIRE((int64_t)c.T * c.R > 0, "distill_backward: no rows");
  CVAE_REQUIRE((int64_t)c.T * c.R <= (1 << 22), "distill_backward: more than %d rows", 1 << 22);   // 32-bit lane offsets in P
  CVAE_REQUIRE(c.X && c.W && c.b && c.eos && ghard && saved && ws && (c.K == 0 || (c.ids && c.top && gsoft)),
               "distill_backward: null operand");
  CVAE_REQUIRE((dW == nullptr) == (db == nullptr), "distill_backward: dW and db go together");
  if (!dX && !dW) return 0;
  CVAE_REQUIRE((((uintptr_t)ws | (uintptr_t)saved) & 15) == 0, "distill_backward: the workspaces must be 16-byte aligned");
  const DistillPlan d = dt_plan(c.dtype, (long)c.T * c.R, c.E, (int)c.V, c.K);
  CVAE_REQUIRE((long)(d.Np / (384 - d.rax)) * d.et < (1 << 19), "distill_backward: too many rows of E = %d", c.E);   // 2^13 threads a tile
  DistillArgs a = {};
  dt_fill(a, d, c, const_cast<void*>(saved));
  a.ghard = ghard; a.gsoft = gsoft; a.dX = dX; a.dW = dW; a.db = db;
  char* w = static_cast<char*>(ws);
  a.Gimg = (_Float16*)(w + d.Gimg); a.coef = (float*)(w + d.coef); a.gmax = (float*)(w + d.gmax);
  a.gpart = c.R > DT_GSCAN ? (float*)(w + d.gpart) : nullptr;
  a.P = (_Float16*)(w + d.P); a.slab = (float*)(w + d.slab); a.vfull = (int)d.vc;
  a.dwtiles = a.vfull / (384 - d.raw) * d.etw;
  return dt_dispatch(c.dtype, d, a, true, s);
}

}  // namespace cvae
