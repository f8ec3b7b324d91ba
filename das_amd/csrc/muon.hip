// Newton-Schulz orthogonalisation of a ragged set of matrices, and the Muon step around it (include/das_hip.h).
//
// For U (rows x cols; m = min, n = max; transposed if rows > cols, so X is m x n):  X = U / (|U|_F + eps), then `steps` times
// X = (a I + b X X^T + c (X X^T)^2) X: in singular values s -> s (a + b s^2 + c s^4). All matrices of a set go through the same launches:
// a table (built once on the host, das_ns_plan) lists every tile of every matrix, one workgroup per tile.
//
// Every operand is a pair of f16, high + low part, 22 bits, and a product is three (high high + high low + low high), whatever the
// result's type: an error of X outside its row and column space grows by |a| a step, 485-fold in five default ones. Single f16 operands,
// 11 bits, would do for gradients of full rank (2e-3 off 64-bit arithmetic in bf16 with its own rounding, and 1.4 to 2.1 times faster),
// but lose gradients out of few pixels: rank 128 1e-2, rank 16 4e-2, rank one 0.2 off. Pairs, f32 result: full rank 2e-6 ... 5e-6, rank
// 16 2e-5 ... 6e-5, rank one 9e-5 (256 x 2304) ... 3e-4 (4096 x 4096). More steps, or steeper ones, cost the product of the polynomial's
// slopes. To pay for three products the m x n matrix is touched as seldom as possible: Z(G) commutes with G, so several steps can be
// taken on m x m matrices alone,
//   G = X X^T;  each step  Z = a I + b G + c G G,  Q = Z Q,  G = X' X'^T = Z G Z;  X' = Q X at the end of such a phase
// 18 m m n + 42 m^3 flops for five steps (plain steps with three products: 45 m m n + 15 m^3; a symmetric product is computed on and
// below its diagonal). A phase ends before an error of G, which grows by (a + b s^2 + c s^4)^2 a step in the direction of small singular
// values s while G's true entries there grow alike but start smaller, has grown 256-fold: with the default polynomial three steps, then
// two.
//
// Scales keep entries, and the low parts of pairs, among f16's normal numbers. X is kept times S, 2^15 over the bound of its norm: an
// entry of a rank-one X is about (m n)^-1/2, and with S = sqrt(n) its low part was subnormal, 2^-25 off (4096 x 4096, f32 result: 8e-4
// off instead of 3e-4). G is kept times gscale, about m (its trace starts at one). Row lengths are padded with zeros (ldx, lda) to whole
// stages of the inner axis.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <functional>
#include <mutex>
#include <new>
#include <queue>
#include <type_traits>
#include <vector>

#include "common.h"
#include "prof.h"

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));

constexpr int TPB = 256;
constexpr int N_AREAS = 5;   // m x m work matrices: G, R, Z, two of Q
constexpr int CHUNK = 64;   // side of the blocks that ingest_kernel / normalise_kernel work on

struct NsMatrix {           // one matrix, as the kernels see it
  long long src;            // element offset in the flat buffers / in the result
  long long x, a;           // element offsets in the work areas X (m x ldx) and A, B (m x lda)
  int rows, cols, m, n, ldx, lda;
  int group, index;         // source tensor and matrix in it (das_orthogonalize)
  int chunk0, chunks;       // its blocks in the partial-sum table
  float scale, gscale;      // S; what G is kept times
  int tall;                 // rows > cols: X holds the transpose
  int thin;                 // m <= 64, too long for one workgroup: X and Q are in areas of their own
};
struct NsItem {             // a workgroup's share: output tile (ti, tj) of a matrix, inner elements 64 k0 ... 64 (k0 + kn)
  int matrix, ti, tj, k0, kn;
  int slot;                 // >= 0: the sums go to this slot of the partial tiles; JOIN items: the first of `slots`
  int slots;
  int m, ldx, lda;          // of the matrix (copied here: a launch starts one load latency earlier than through its index)
  float scale, gscale;
  long long x, a;
};
struct Partial {            // of one 64 x 64 block: sum of squares of (u 2^-e), and e
  float ss;
  int e;
};

// v as a pair of f16: v rounded, and what that leaves. Both parts come from one f32 value: the empty asm (no instruction; what comes here is a
// sum or a product formed by the vector unit, or was loaded) keeps hipcc from fusing the multiplication that v comes from into one of two
// conversions of it. v_fma_mixlo_f16 rounds the product once, v_mul_f32 and v_cvt_pk_f16_f32 round it twice: next to a tie they differ, and
// a high part with the low part of its neighbour is 2^-11 of v off (one element in 2^15; rank one, 256 x 2304: 7.4e-4 off instead of 1.3e-4).
struct Pair {
  _Float16 high, low;
};
__device__ __forceinline__ Pair pair_of(float v) {
  asm("" : "+v"(v));
  const _Float16 h = (_Float16)v;
  return {h, (_Float16)(v - (float)h)};
}

// N (4 or 8) neighbouring values of a row of a work matrix: 32 high parts, then their 32 low parts, and so on along the row
__device__ __forceinline__ long long at(int ld, int r, int c) {
  return (long long)r * (2 * ld) + (c >> 5) * 64 + (c & 31);
}
template <int N>
__device__ __forceinline__ void put(_Float16* base, int ld, int r, int c, const float (&v)[N]) {
  typedef _Float16 vec_t __attribute__((ext_vector_type(N)));
  _Float16* p = base + at(ld, r, c);
  vec_t h, l;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const Pair q = pair_of(v[e]);
    h[e] = q.high;
    l[e] = q.low;
  }
  *reinterpret_cast<vec_t*>(p) = h;
  *reinterpret_cast<vec_t*>(p + 32) = l;
}
template <int N>
__device__ __forceinline__ void get(const _Float16* base, int ld, int r, int c, float (&v)[N]) {
  typedef _Float16 vec_t __attribute__((ext_vector_type(N)));
  const _Float16* p = base + at(ld, r, c);
  const vec_t h = *reinterpret_cast<const vec_t*>(p), l = *reinterpret_cast<const vec_t*>(p + 32);
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = (float)h[e] + (float)l[e];
}

// ------------------------------------------------------------------ U -> X
struct Sources {            // das_orthogonalize's tensors, by value (no pointer table to upload)
  static constexpr int MAX = 64;
  DasNsSource s[MAX];
  int first, count;         // group of s[0], groups in this launch
};
struct MuonIn {
  const float* g;
  float* buf;
  float momentum, rest;     // mu, 1 - mu (each rounded once: 1 - f32(0.98) is 9e-7 off 0.02)
  float grad_scale, max_norm;
  int nesterov;
  const float* sumsq;
};

__device__ __forceinline__ float block_reduce(float v, bool is_max, float* red) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const float w = __shfl_xor(v, o, 64);
    v = is_max ? fmaxf(v, w) : v + w;
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  return is_max ? fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])) : (red[0] + red[1]) + (red[2] + red[3]);
}

// g's factor: the scale times min(1, max_norm / (norm + 1e-6)); a NaN norm stays NaN
__device__ __forceinline__ float grad_factor(const MuonIn& mu) {
  float f = mu.grad_scale;
  if (mu.max_norm > 0.f) {
    const float k = mu.max_norm / (sqrtf(*mu.sumsq) * mu.grad_scale + 1e-6f);
    f *= k > 1.f ? 1.f : k;
  }
  return f;
}
// the momentum's new value in b, returns U
__device__ __forceinline__ float muon_in(const MuonIn& mu, float f, float g, float& b) {
  g *= f;
  b = mu.momentum * b + mu.rest * g;
  return mu.nesterov ? mu.rest * g + mu.momentum * b : b;
}

template <typename T>
__device__ __forceinline__ float load_as_f32(const void* base, long long i) {
  const T v = reinterpret_cast<const T*>(base)[i];
  if constexpr (std::is_same<T, bf16_t>::value) return bf16_to_f32(v);
  else return (float)v;
}

// One 64 x 64 block of U: update the momentum (Muon), find the block's exponent e (largest entry in [1/2, 1) 2^(e + 10)) and sum of
// squares, store u 2^-e in X's layout (transposed through LDS for tall matrices), zeros in the padding. The exponent keeps gradients
// of any magnitude inside f16's range until the norm is known; normalise_kernel rounds a second time.
template <typename T, bool MUON>
__global__ __launch_bounds__(TPB) void ingest_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ chunks, Sources src,
                                                     MuonIn mu, _Float16* __restrict__ X, _Float16* __restrict__ XT, Partial* __restrict__ part) {
  __shared__ float tile[CHUNK][CHUNK + 1];
  __shared__ float red[4];
  const int4 ch = chunks[blockIdx.x];
  const NsMatrix M = mats[ch.x];
  if (!MUON && (unsigned)(M.group - src.first) >= (unsigned)src.count) return;   // (whole workgroups)
  const int r0 = ch.y * CHUNK, c0 = ch.z * CHUNK;
  const int c4 = (threadIdx.x & 15) * 4, rr = threadIdx.x >> 4;
  float u[4][4] = {}, big = 0.f;
  // Four values a load where the matrix allows it: every row of four starts on 16 bytes (8 for two-byte types) of the source
  const int c = c0 + c4, left = M.cols - c;
  if constexpr (MUON) {
    const float coef = grad_factor(mu);
    const float* g = mu.g + M.src + c;
    float* m = mu.buf + M.src + c;
    float b[4][4];
    if (!((M.cols | M.src) & 3) && !(((uintptr_t)mu.g | (uintptr_t)mu.buf) & 15)) {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long o = (long long)(r0 + rr + k * 16) * M.cols;
        if (r0 + rr + k * 16 < M.rows && left > 0) {
          *reinterpret_cast<float4*>(u[k]) = *reinterpret_cast<const float4*>(g + o);
          *reinterpret_cast<float4*>(b[k]) = *reinterpret_cast<const float4*>(m + o);
        }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long o = (long long)(r0 + rr + k * 16) * M.cols;
        if (r0 + rr + k * 16 < M.rows && left > 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) u[k][j] = muon_in(mu, coef, u[k][j], b[k][j]);
          *reinterpret_cast<float4*>(m + o) = *reinterpret_cast<const float4*>(b[k]);
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long o = (long long)(r0 + rr + k * 16) * M.cols;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r0 + rr + k * 16 < M.rows && j < left) {
            u[k][j] = g[o + j];
            b[k][j] = m[o + j];
          }
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const long long o = (long long)(r0 + rr + k * 16) * M.cols;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (r0 + rr + k * 16 < M.rows && j < left) {
            u[k][j] = muon_in(mu, coef, u[k][j], b[k][j]);
            m[o + j] = b[k][j];
          }
      }
    }
  } else {
    const DasNsSource& s = src.s[M.group - src.first];
    const T* from = reinterpret_cast<const T*>(s.base) + M.index * s.batch_stride + c;
    const bool vec = !((s.row_stride | s.batch_stride) & 3) && !((uintptr_t)s.base & (4 * sizeof(T) - 1));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const long long o = (r0 + rr + k * 16) * s.row_stride;
      if (r0 + rr + k * 16 >= M.rows) continue;
      if (vec && left >= 4) {
        struct alignas(4 * sizeof(T)) Four { T v[4]; };
        const Four f = *reinterpret_cast<const Four*>(from + o);
#pragma unroll
        for (int j = 0; j < 4; ++j) u[k][j] = load_as_f32<T>(f.v, j);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < left) u[k][j] = load_as_f32<T>(from, o + j);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) big = fmaxf(big, fabsf(u[k][j]));   // (NaN is passed over here and stays NaN in u)
  big = block_reduce(big, true, red);
  int e = 0;
  if (big > 0.f && big <= 3.4028235e38f) {
    (void)frexpf(big, &e);
    e -= 10;
  }
  float ss = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      u[k][j] = ldexpf(u[k][j], -e);
      ss += u[k][j] * u[k][j];
    }
  ss = block_reduce(ss, false, red);
  if (threadIdx.x == 0) part[M.chunk0 + ch.w] = Partial{ss, e};
  if (M.tall) {
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) tile[c4 + j][rr + k * 16] = u[k][j];
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int j = 0; j < 4; ++j) u[k][j] = tile[rr + k * 16][c4 + j];
  }
  const int x_r0 = M.tall ? c0 : r0, x_c0 = M.tall ? r0 : c0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = x_r0 + rr + k * 16;
    if (r >= M.m) continue;
    put((M.thin ? XT : X) + 2 * M.x, M.ldx, r, x_c0 + c4, u[k]);
  }
}

// X <- X 2^e S / (|U|_F + eps), block by block. Every workgroup sums its matrix's partials itself, in one fixed order, in f64.
__global__ __launch_bounds__(TPB) void normalise_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ chunks, float eps,
                                                        _Float16* __restrict__ X, const Partial* __restrict__ part) {
  __shared__ double red[4];
  const int4 ch = chunks[blockIdx.x];
  const NsMatrix M = mats[ch.x];
  double s = 0.0;
  for (int i = threadIdx.x; i < M.chunks; i += TPB) {
    const Partial q = part[M.chunk0 + i];
    s += ldexp((double)q.ss, 2 * q.e);
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  const double norm = sqrt((red[0] + red[1]) + (red[2] + red[3]));
  const float f = (float)ldexp((double)M.scale / (norm + (double)eps), part[M.chunk0 + ch.w].e);
  const int x_r0 = (M.tall ? ch.z : ch.y) * CHUNK, x_c0 = (M.tall ? ch.y : ch.z) * CHUNK;
  const int c4 = (threadIdx.x & 15) * 4, rr = threadIdx.x >> 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = x_r0 + rr + k * 16;
    if (r >= M.m) continue;
    _Float16* x = X + 2 * M.x;
    float v[4];
    get(x, M.ldx, r, x_c0 + c4, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= f;
    put(x, M.ldx, r, x_c0 + c4, v);
  }
}

// ------------------------------------------------------------------ products
// T x T tile (T = 128 or 64) of one matrix by four waves of T/2 x T/2, v_mfma_f32_16x16x32_f16: lane l holds row l % 16 of A (column of
// B), inner elements (l / 16) * 8 ... + 8, and gets column l % 16, rows (l / 16) * 4 ... + 4 of the result.
//
// A stage is 128 bytes of every row of both operands, a whole line: 32 inner elements' high parts and their low parts, which lie next to
// each other in memory. It is copied global -> LDS without passing registers into one of two buffers.
//   acc += Al Bh + Ah Bl + Ah Bh   (the low x low part is 2^-22 of the product)
// KG groups of four waves divide the inner axis between them (KG = 4 or 2 where a launch has few tiles and latency is all: every
// group has its own buffers and copies in flight) and join their sums through LDS, in order.
// LDS images. Rows by rows (gram, product, and B of the update): two panels of T rows x 64 bytes, 16-byte slot s of row r holds source
// slot s ^ (r / 2 % 4): eight neighbouring rows cover all banks. Columns of X (update): inner rows as they are in memory, 32-byte units
// swizzled by row, read with ds_read_tr16_b64 (four inner rows x 16 columns a 16-lane group, one column a lane).
typedef short i16x4_t __attribute__((ext_vector_type(4)));

// 16 bytes a lane, global -> LDS (lane 0's destination + 16 l). Issued from asm: for the builtin hipcc waits for every copy in flight in
// front of the next LDS read. The waits are multiply()'s. M0 (the destination) is put back.
__device__ __forceinline__ void copy16(const void* src, const char* lds_wave_base) {
  unsigned keep;
  const unsigned dst = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(const __attribute__((address_space(3))) char*)lds_wave_base);
  asm volatile("s_mov_b32 %0, m0\n\ts_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n\ts_mov_b32 m0, %0"
               : "=&s"(keep)
               : "v"(src), "s"(dst)
               : "memory");
}
// every copy of this wave has landed and every LDS read of it is done, then the same of every wave
// (the wait is the builtin's: after one in asm hipcc takes the reads for unfinished and waits again, for the next stage's too, before
// the first matrix instruction)
__device__ __forceinline__ void landed() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int T>
struct RowsOperand {        // T rows of a matrix whose rows run along the inner axis
  const char* src[T / 32];
  __device__ __forceinline__ void init(const _Float16* base, int pitch, int row0, int rows, int stage0) {
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      const int q = wave * (T / 32) + i, r = (q >> 1) * 16 + (lane >> 2), kg = (lane & 3) ^ ((r >> 1) & 3);
      src[i] = (const char*)(base + (long long)min(row0 + r, rows - 1) * pitch + stage0 * 64 + (q & 1) * 32 + kg * 8);   // (rows past the end: stand-ins)
    }
  }
  __device__ __forceinline__ void issue(char* lds) {
    const int wave = (threadIdx.x >> 6) & 3;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      const int q = wave * (T / 32) + i;
      copy16(src[i], lds + (q & 1) * (T * 64) + (q >> 1) * 1024);
      src[i] += 128;
    }
  }
  // fragment t of part p (half of the inner axis / high or low part)
  static __device__ __forceinline__ f16x8_t frag(const char* lds, int row0, int t, int p) {
    const int lane = threadIdx.x & 63, r = row0 + t * 16 + (lane & 15);
    return *reinterpret_cast<const f16x8_t*>(lds + p * (T * 64) + r * 64 + (((lane >> 4) ^ ((r >> 1) & 3)) << 4));
  }
};

template <int T>
struct ColsOperand {        // T columns of a matrix whose rows run across the inner axis
  static constexpr int ROWB = T * 4, LPR = ROWB / 16, ROWS = 32;   // bytes and lanes of a row, rows of a stage
  const char* base;
  int pitch, rows, row;     // bytes; rows of the matrix; the stage's first row
  static __device__ __forceinline__ int swz(int r) {
    return (r & 3) | ((r >> 1) & 4);
  }
  __device__ __forceinline__ void init(const _Float16* x, int pitch_elems, int col0, int rows_, int stage0) {
    base = (const char*)(x + col0 * 2);
    pitch = pitch_elems * 2;
    rows = rows_;
    row = stage0 * ROWS;
  }
  __device__ __forceinline__ void issue(char* lds) {
    const int lane = threadIdx.x & 63, wave = (threadIdx.x >> 6) & 3;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      const int q = wave * (T / 32) + i, r = q * (64 / LPR) + lane / LPR, s = lane % LPR;
      // (rows past the end meet zeros of the other operand; a row of the same matrix stands in, so that only its own NaN can enter)
      copy16(base + (long long)min(row + r, rows - 1) * pitch + (((s >> 1) ^ swz(r)) * 32 + (s & 1) * 16), lds + q * 1024);
    }
    row += ROWS;
  }
  static __device__ __forceinline__ f16x8_t frag(const char* lds, int col0, int t, int p) {
    const int lane = threadIdx.x & 63, q = lane & 15, c = col0 + t * 16;
    const int unit = (c >> 5) * 4 + p * 2 + ((c >> 4) & 1);
    i16x4_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (lane >> 4) * 8 + h * 4 + (q >> 2);
      v[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) i16x4_t*)(lds + r * ROWB + ((unit ^ swz(r)) * 32) + (q & 3) * 8));
    }
    f16x8_t f;
    const f16x4_t a = __builtin_bit_cast(f16x4_t, v[0]), b = __builtin_bit_cast(f16x4_t, v[1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      f[e] = a[e];
      f[e + 4] = b[e];
    }
    return f;
  }
};

template <int T>
using Acc = f32x4_t[T / 32][T / 32];

template <int T, int KG>
constexpr int lds_bytes() { return KG * 4 * T * 128; }

// `stages`: of the workgroup's part of the inner axis; the group's first one is group * ceil(stages / KG)
template <int T, int KG, typename OB>
__device__ __forceinline__ void multiply(RowsOperand<T>& a, OB& b, int stages, char* smem, Acc<T>& acc) {
  constexpr int HALF = T * 128, N = T / 32;   // bytes of one operand's stage; fragments a wave has of each operand
  const int wave = (threadIdx.x >> 6) & 3, wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
  const int group = KG == 1 ? 0 : threadIdx.x >> 8, per = (stages + KG - 1) / KG, mine = KG == 1 ? stages : min(per, stages - group * per);
  char* base = smem + group * 4 * HALF;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  f16x8_t fa[2][2][N], fb[2][2][N];   // [parity of the stage][part][fragment]
  auto read = [&](int k, auto parity) {
    constexpr int Z = decltype(parity)::value;
    const char* cur = base + (k & 1) * 2 * HALF;
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int t = 0; t < N; ++t) {
        fa[Z][p][t] = RowsOperand<T>::frag(cur, wr, t, p);
        fb[Z][p][t] = OB::frag(cur + HALF, wc, t, p);
      }
  };
  auto issue = [&](int k) {
    if (k < mine) {
      char* dst = base + (k & 1) * 2 * HALF;
      a.issue(dst);
      b.issue(dst + HALF);
    }
  };
  // Stage k is multiplied from registers while stage k + 1 is read from LDS and stage k + 2 is copied into the buffer that k has left.
  auto step = [&](int k, auto parity) {
    constexpr int Z = decltype(parity)::value;
    landed();                          // stage k + 1 is in LDS, stage k in registers, in every wave
    issue(k + 2);
    if (k + 1 < mine) read(k + 1, std::integral_constant<int, Z ^ 1>{});
    if (k < mine) {
#pragma unroll
      for (int q = 0; q < 3; ++q)   // low parts first
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) {
            acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[Z][q == 0][i], fb[Z][q == 1][j], acc[i][j], 0, 0, 0);
          }
    }
  };
  issue(0);
  landed();
  issue(1);
  if (mine > 0) read(0, std::integral_constant<int, 0>{});
  for (int k = 0; k < per; k += 2) {
    step(k, std::integral_constant<int, 0>{});
    if (k + 1 < per) step(k + 1, std::integral_constant<int, 1>{});
  }
  __syncthreads();
  if constexpr (KG > 1) {
    f32x4_t* sums = reinterpret_cast<f32x4_t*>(smem);   // [group - 1][fragment][thread of the group]
    const int t = threadIdx.x & 255;
    if (group > 0) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) sums[((group - 1) * N * N + i * N + j) * 256 + t] = acc[i][j];
    }
    __syncthreads();
    if (group == 0) {
#pragma unroll
      for (int g = 0; g < KG - 1; ++g)
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
          for (int j = 0; j < N; ++j) acc[i][j] += sums[(g * N * N + i * N + j) * 256 + t];
    }
  }
}
template <int KG>
__device__ __forceinline__ int first_stage(int stages) { return KG == 1 ? 0 : (int)(threadIdx.x >> 8) * ((stages + KG - 1) / KG); }

// The tile (of the first group) through LDS, row by row: f(row, col, eight values of the row). TRANSPOSED: rows and columns exchanged.
template <int T, int KG, bool TRANSPOSED, typename F>
__device__ __forceinline__ void store_tile(const Acc<T>& acc, char* smem, F f) {
  constexpr int P = T + 4;   // floats of a row: the four row groups of a fragment start 16 banks apart
  float* buf = reinterpret_cast<float*>(smem);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int major = (TRANSPOSED ? wave & 1 : (wave >> 1) & 1) * (T / 2), minor = (TRANSPOSED ? (wave >> 1) & 1 : wave & 1) * (T / 2);
  for (int r0 = 0; r0 < T; r0 += 64) {
    __syncthreads();
    if ((KG == 1 || wave < 4) && (T == 64 || major == r0)) {
#pragma unroll
      for (int i = 0; i < T / 32; ++i)
#pragma unroll
        for (int j = 0; j < T / 32; ++j) {
          if constexpr (TRANSPOSED) {
            *reinterpret_cast<f32x4_t*>(buf + (major - r0 + j * 16 + (lane & 15)) * P + minor + i * 16 + (lane >> 4) * 4) = acc[i][j];
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) buf[(major - r0 + i * 16 + (lane >> 4) * 4 + e) * P + minor + j * 16 + (lane & 15)] = acc[i][j][e];
          }
        }
    }
    __syncthreads();
    constexpr int TPR = T / 8, RPS = KG * TPB / TPR;
#pragma unroll
    for (int s = 0; s < (64 + RPS - 1) / RPS; ++s) {
      const int r = s * RPS + threadIdx.x / TPR, c = (threadIdx.x % TPR) * 8;
      if (RPS > 64 && r >= 64) continue;
      float v[8];
      *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(buf + r * P + c);
      *reinterpret_cast<float4*>(v + 4) = *reinterpret_cast<const float4*>(buf + r * P + c + 4);
      f(r0 + r, c, v);
    }
  }
}

enum SymKind { GRAM, POLY, PRODUCT };
struct SymArgs {            // two independent products a launch (blockIdx.y)
  const _Float16 *p[2], *q[2];
  _Float16* out[2];
  float a, b, c;
  long long slots;          // partial tiles of one product
};

// Symmetric m x m results, tiles on and below the diagonal, each stored as it is and transposed.
//   GRAM:     G = X X^T times (gscale / S^2)      POLY: Z = a I + b G + c G G      PRODUCT: P Q of symmetric P, Q that commute
// Columns m ... lda are stored as zeros: the inner axis of the next product.
template <int T, int KG, SymKind KIND>
__device__ __forceinline__ void sym_store(const NsItem& M, const SymArgs& s, int z, int i0, int j0, const Acc<T>& acc, char* smem) {
  const _Float16* P = s.p[z] + 2 * M.a;
  _Float16* out = s.out[z] + 2 * M.a;
  const float f = KIND == GRAM ? M.gscale / (M.scale * M.scale) : 1.f, cb = s.b / M.gscale, cc = s.c / (M.gscale * M.gscale);
  auto store = [&](int r, int c, float (&v)[8]) {
    if (r >= M.m || c >= M.lda) return;
    if constexpr (KIND == POLY) {
      float g[8];
      get(P, M.lda, r, c, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = cc * v[e] + cb * g[e] + (r == c + e ? s.a : 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e >= M.m) v[e] = 0.f;
    put(out, M.lda, r, c, v);
  };
  store_tile<T, KG, false>(acc, smem, [&](int r, int c, float (&v)[8]) { store(i0 + r, j0 + c, v); });
  if (i0 != j0) store_tile<T, KG, true>(acc, smem, [&](int r, int c, float (&v)[8]) { store(j0 + r, i0 + c, v); });
}

template <int T, int KG, SymKind KIND>
__global__ __launch_bounds__(KG * TPB, KG == 1 ? 2 : KG) void sym_kernel(const NsItem* __restrict__ items, SymArgs s, f32x4_t* __restrict__ partial) {
  extern __shared__ __align__(16) char smem[];
  const NsItem t = items[blockIdx.x];
  if (t.matrix < 0) return;   // (filling: an XCD's queue is shorter than the longest)
  const int z = blockIdx.y, i0 = t.ti * T, j0 = t.tj * T;
  const int ld = KIND == GRAM ? t.ldx : t.lda, pitch = 2 * ld;
  const _Float16* P = s.p[z] + 2 * (KIND == GRAM ? t.x : t.a);
  const _Float16* Q = s.q[z] + 2 * (KIND == GRAM ? t.x : t.a);
  RowsOperand<T> a, b;
  const int stages = 2 * t.kn, first = 2 * t.k0 + first_stage<KG>(stages);
  a.init(P, pitch, i0, t.m, first);
  b.init(Q, pitch, j0, t.m, first);
  Acc<T> acc;
  multiply<T, KG>(a, b, stages, smem, acc);
  if (t.slot >= 0) {   // (a part of the inner axis: join_kernel goes on)
    if (KG == 1 || threadIdx.x < TPB) {
#pragma unroll
      for (int i = 0; i < T / 32; ++i)
#pragma unroll
        for (int j = 0; j < T / 32; ++j) partial[(((long long)z * s.slots + t.slot) * (T / 32) * (T / 32) + i * (T / 32) + j) * TPB + threadIdx.x] = acc[i][j];
    }
    return;
  }
  sym_store<T, KG, KIND>(t, s, z, i0, j0, acc, smem);
}

// The parts of a tile whose inner axis was split, added in order, and stored as sym_store does; 16 workgroups a tile, four rows of one
// column a thread (one workgroup a tile: 12 us, most of them waiting for one load after the other).
template <int T, SymKind KIND>
__global__ __launch_bounds__(TPB) void join_kernel(const NsItem* __restrict__ items, SymArgs s,
                                                   const f32x4_t* __restrict__ partial) {
  constexpr int N = T / 32;
  const NsItem t = items[blockIdx.x / (N * N)];
  const int frag = blockIdx.x % (N * N), z = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const f32x4_t* from = partial + (((long long)z * s.slots + t.slot) * N * N + frag) * TPB + threadIdx.x;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  for (int k0 = 0; k0 < t.slots; k0 += 4) {
    f32x4_t v[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = k0 + k < t.slots ? from[(long long)(k0 + k) * N * N * TPB] : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) sum += v[k];
  }
  const int r = t.ti * T + (wave >> 1) * (T / 2) + (frag / N) * 16 + (lane >> 4) * 4;   // four rows of one column
  const int c = t.tj * T + (wave & 1) * (T / 2) + (frag % N) * 16 + (lane & 15);
  if (r >= t.lda) return;
  _Float16* out = s.out[z] + 2 * t.a;
  float v[4] = {sum[0], sum[1], sum[2], sum[3]};
  if constexpr (KIND == GRAM) {
    const float f = t.gscale / (t.scale * t.scale);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] *= f;
  }
  if constexpr (KIND == POLY) {
    const float cb = s.b / t.gscale, cc = s.c / (t.gscale * t.gscale);
    float g[4] = {0.f, 0.f, 0.f, 0.f};
    if (c < t.m) get(s.p[0] + 2 * t.a, t.lda, c, r, g);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = cc * v[e] + cb * g[e] + (r + e == c ? s.a : 0.f);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (r + e >= t.m || c >= t.m) v[e] = 0.f;
  if (c < t.m) put(out, t.lda, c, r, v);
  if (t.ti == t.tj) return;   // (a diagonal tile holds both halves)
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (r + e < t.m && c < t.lda) {
      _Float16* p = out + at(t.lda, r + e, c);
      const Pair q = pair_of(v[e]);
      p[0] = q.high;
      p[32] = q.low;
    }
}

struct Result {             // where the last product goes
  void* out;                // das_orthogonalize
  int out_dtype;
  float* p;                 // das_muon_step: p = keep p - lr f X
  float keep, lr;
  int lr_scale;
};
__device__ __forceinline__ float result_factor(const NsMatrix& M, const Result& res) {
  float f = 1.f / M.scale;
  if (res.p) {
    const float r = (float)M.rows, c = (float)M.cols;
    f *= res.lr * (res.lr_scale ? 0.2f * sqrtf(fmaxf(r, c)) : sqrtf(fmaxf(1.f, r / c)));
  }
  return f;
}

// X' = Q X: Q's rows by X's columns. LAST: the result leaves the work area (and its scale S), transposed back where needed.
template <int T, int KG, bool LAST>
__global__ __launch_bounds__(KG * TPB, KG == 1 ? 2 : KG) void update_kernel(const NsMatrix* __restrict__ mats, const NsItem* __restrict__ items,
                                                        const _Float16* __restrict__ Q, const _Float16* __restrict__ X,
                                                        _Float16* __restrict__ Y, Result res) {
  extern __shared__ __align__(16) char smem[];
  const NsItem t = items[blockIdx.x];
  if (t.matrix < 0) return;
  const int i0 = t.ti * T, j0 = t.tj * T;
  RowsOperand<T> a;
  ColsOperand<T> b;
  const int stages = 2 * t.kn, first = first_stage<KG>(stages);
  a.init(Q + 2 * t.a, 2 * t.lda, i0, t.m, first);
  b.init(X + 2 * t.x, 2 * t.ldx, j0, t.m, first);
  Acc<T> acc;
  multiply<T, KG>(a, b, stages, smem, acc);
  if constexpr (!LAST) {
    store_tile<T, KG, false>(acc, smem, [&](int r, int c, float (&v)[8]) {
      if (i0 + r < t.m) put(Y + 2 * t.x, t.ldx, i0 + r, j0 + c, v);   // (columns n ... ldx: zero, as X's are)
    });
  } else {
    const NsMatrix M = mats[t.matrix];
    const float f = result_factor(M, res);
    const bool vec = M.cols % 8 == 0 && M.src % 8 == 0 && !((uintptr_t)(res.p ? (const void*)res.p : res.out) & 15);
    auto emit = [&](int r, int c, float (&v)[8]) {   // in the caller's rows and columns
      if (r >= M.rows || c >= M.cols) return;
      const long long o = M.src + (long long)r * M.cols + c;
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
      const int n = vec ? 8 : min(8, M.cols - c);
      if (res.p) {
        float* p = res.p + o;
        if (vec) {
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            float4 w = *reinterpret_cast<float4*>(p + e);
            w.x = res.keep * w.x - v[e]; w.y = res.keep * w.y - v[e + 1]; w.z = res.keep * w.z - v[e + 2]; w.w = res.keep * w.w - v[e + 3];
            *reinterpret_cast<float4*>(p + e) = w;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = res.keep * p[e] - v[e];
        }
      } else if (res.out_dtype == DAS_F32) {
        float* p = reinterpret_cast<float*>(res.out) + o;
        if (vec) {
          *reinterpret_cast<float4*>(p) = *reinterpret_cast<const float4*>(v);
          *reinterpret_cast<float4*>(p + 4) = *reinterpret_cast<const float4*>(v + 4);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = v[e];
        }
      } else {
        uint16_t h[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
          h[e] = res.out_dtype == DAS_BF16 ? f32_to_bf16(v[e]) : __builtin_bit_cast(uint16_t, (_Float16)v[e]);
        uint16_t* p = reinterpret_cast<uint16_t*>(res.out) + o;
        if (vec) {
          *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (e < n) p[e] = h[e];
        }
      }
    };
    if (M.tall) store_tile<T, KG, true>(acc, smem, [&](int r, int c, float (&v)[8]) { emit(j0 + r, i0 + c, v); });
    else store_tile<T, KG, false>(acc, smem, [&](int r, int c, float (&v)[8]) { emit(i0 + r, j0 + c, v); });
  }
}

// ------------------------------------------------------------------ small and thin matrices
// small_kernel: the whole of a matrix in one workgroup, everything between the caller's reads and writes in LDS, where it fits (64 x 256,
// 16 x 1856). A launch for every product would cost 4 us each; 64 x 64: 67 us as 17 launches.
// thin_kernel / chain_kernel: longer ones, by slices of their columns. X X^T is summed over the slices' parts by chain_kernel, which takes
// all steps of a phase on the m x m matrices in LDS and leaves Q; the pass over the slices that forms Q X also forms the parts of the next
// X X^T: five launches after the first pass (16 x 1056 by tiles: 85 us).
//
// 16 waves, one 16 x 16 fragment of an m x m product a wave (2 x 2 fragments each on four waves: 20.4 us for 64 x 64 instead of 19.8, the
// flows' and predictors' set, up to 64 x 256, 31.7 us instead of 25.0: one wave a SIMD hides no latency). m <= 32 leaves waves over: they
// divide the long inner axis of X X^T, and Z Q and Z G are formed by different ones. LDS matrices: rows of pairs (32 high parts, 32 low
// parts, ...), row pitch 16 bytes past a multiple of 256; 32 columns of X take 128 bytes as pairs and as floats: U, X and the result use
// the same place. Rows and columns up to the next multiple of 16 are zero.
constexpr int SMALL_M = 64, SMALL_TPB = 1024, SMALL_LDS = 155 * 1024;
constexpr int PA = 2 * SMALL_M + 8;   // row pitch of the m x m matrices, f16 elements
constexpr int SMALL_QUADS = 8;        // float4 of U, and 16 x 16 fragments of X, a thread / wave can have: m n <= 32 Ki (fewer where a set allows it: no spills)
struct Steps {
  float coef[3 * DAS_NS_MAX_STEPS];
  int end[DAS_NS_MAX_STEPS];          // of the phase that starts at this step
  int steps;
  float eps;
};
__host__ __device__ inline int up16(int m) { return (m + 15) & ~15; }
__host__ __device__ inline int up64(int n) { return (n + 63) & ~63; }
// X, the m x m matrices, and behind them room for the shares of a sum (not over the m x m matrices: m <= 16 reads 32 columns of them,
// 16 of them zero)
inline long long small_lds(int m, int n) { return 2LL * up16(m) * (2 * up64(n) + 8 + N_AREAS * PA) + (m <= 32 ? SMALL_TPB * 16 : 0); }

__device__ __forceinline__ f16x8_t row_frag(const _Float16* p, int pitch, int row0, int k, int part) {
  const int lane = threadIdx.x & 63;
  return *reinterpret_cast<const f16x8_t*>(p + (row0 + (lane & 15)) * pitch + k * 64 + part * 32 + (lane >> 4) * 8);
}
__device__ __forceinline__ f16x8_t col_frag(const _Float16* x, int pitch, int rows, int col0, int k, int part) {
  const int lane = threadIdx.x & 63, q = lane & 15, c = col0 + (q & 3) * 4;
  f16x8_t f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int r = min(k * 32 + (lane >> 4) * 8 + h * 4 + (q >> 2), rows - 1);   // (rows past the end meet zeros of the other operand)
    const f16x4_t v = __builtin_bit_cast(
        f16x4_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4_t*)(x + r * pitch + (c >> 5) * 64 + part * 32 + (c & 31))));
#pragma unroll
    for (int e = 0; e < 4; ++e) f[h * 4 + e] = v[e];
  }
  return f;
}
// One fragment: P's rows from row0 by (Q's rows from q0, or its columns from q0), an inner step of 32. Two chains of sums
template <bool COLS>
__device__ __forceinline__ void frag_step(const _Float16* p, int pp, int row0, const _Float16* q, int qp, int q_rows, int q0, int k, f32x4_t& high,
                                          f32x4_t& low) {
  f16x8_t a[2], b[2];
#pragma unroll
  for (int u = 0; u < 2; ++u) {
    a[u] = row_frag(p, pp, row0, k, u);
    b[u] = COLS ? col_frag(q, qp, q_rows, q0, k, u) : row_frag(q, qp, q0, k, u);
  }
  high = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[0], high, 0, 0, 0);
  low = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[1], b[0], low, 0, 0, 0);
  low = __builtin_amdgcn_mfma_f32_16x16x32_f16(a[0], b[1], low, 0, 0, 0);
}
template <int K>   // m x m matrices, K inner steps
__device__ __forceinline__ f32x4_t square_product(const _Float16* p, int row0, const _Float16* q, int q0) {
  f32x4_t acc = {}, low = {};
#pragma unroll
  for (int k = 0; k < K; ++k) frag_step<false>(p, PA, row0, q, PA, 0, q0, k, acc, low);
  return acc + low;
}
// X X^T, inner steps k0, k0 + stride, ... < k1
__device__ __forceinline__ f32x4_t long_product(const _Float16* x, int pitch, int row0, int col0, int k0, int k1, int stride) {
  f32x4_t acc = {}, low = {};
  for (int k = k0; k < k1; k += stride) frag_step<false>(x, pitch, row0, x, pitch, 0, col0, k, acc, low);
  return acc + low;
}
// Q's rows from row0 (m x m) by X's columns from col0
template <int K>
__device__ __forceinline__ f32x4_t update_fragment(const _Float16* q, int row0, const _Float16* x, int pitch, int rows, int col0) {
  f32x4_t acc = {}, low = {};
#pragma unroll
  for (int k = 0; k < K; ++k) frag_step<true>(q, PA, row0, x, pitch, rows, col0, k, acc, low);
  return acc + low;
}
__device__ __forceinline__ void put4(_Float16* p, const float (&v)[4]) {
  f16x4_t h, l;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const Pair q = pair_of(v[e]);
    h[e] = q.high;
    l[e] = q.low;
  }
  *reinterpret_cast<f16x4_t*>(p) = h;
  *reinterpret_cast<f16x4_t*>(p + 32) = l;
}
__device__ __forceinline__ int pair_at(int pitch, int r, int c) { return r * pitch + (c >> 5) * 64 + (c & 31); }

// Which fragment of an m16 x m16 matrix a wave has (first row and column), and which share of a long inner axis
struct Share {
  int r0, c0, part, parts;     // part >= parts: a wave without work
  __device__ explicit Share(int m16) {
    const int w = threadIdx.x >> 6, n = m16 >> 4, frags = n * n, f = w % frags;
    parts = (SMALL_TPB / 64) / frags;
    part = w / frags;
    r0 = (f / n) * 16;
    c0 = (f % n) * 16;
  }
};
// P Q^T's fragment stored transposed (four values of a lane are neighbours then), so that Q P^T is what lies there: f(row, col, four
// values) may change them
template <typename F>
__device__ __forceinline__ void frag_store(const Share& w, const f32x4_t& acc, _Float16* out, F f) {
  const int lane = threadIdx.x & 63, r = w.c0 + (lane & 15), c = w.r0 + (lane >> 4) * 4;
  float v[4] = {acc[0], acc[1], acc[2], acc[3]};
  f(r, c, v);
  put4(out + pair_at(PA, r, c), v);
}
// The shares of a sum over a long inner axis, added in order and stored as G. scratch: 16 KiB of LDS of its own where there are several
__device__ __forceinline__ void store_gram(const Share& w, f32x4_t acc, f32x4_t* scratch, _Float16* G, float scale) {
  if (w.parts > 1) {
    scratch[threadIdx.x] = acc;
    __syncthreads();
    if (w.part == 0)
      for (int s = 1; s < w.parts; ++s) acc += scratch[s * (SMALL_TPB / w.parts) + threadIdx.x];
  }
  if (w.part == 0)
    frag_store(w, acc, G, [&](int, int, float (&v)[4]) {
#pragma unroll
      for (int t = 0; t < 4; ++t) v[t] *= scale;
    });
  __syncthreads();
}
// Steps k ... end - 1 on the m x m matrices (the same products as iterate), G in A[0]; -> Q.
// The factors' order matters to rounding errors alone. Between the null space of X X^T, where Z is near 3.4, and the rest, where it is
// near 1, those of Z G Z and of Z Q (Q's columns in the rest) grow by the product of both a step, those of Z Z G or Q Z by the larger one
// squared (64 x 64 of rank one: 4e-4 off instead of 2e-5). The tiles' form has no order: it computes one half and mirrors it.
template <int K>   // K inner steps of 32: m <= 32 K
__device__ __forceinline__ _Float16* phase_chain(const Share& w, _Float16* const (&A)[N_AREAS], const Steps& st, int k, int end, float gscale) {
  const bool on = w.part == 0, second = w.part == (w.parts > 1 ? 1 : 0);
  _Float16 *G = A[0], *R = A[1], *Z = A[2], *q = nullptr, *spare = A[3], *other = A[4];
  auto plain = [](int, int, float (&)[4]) {};
  const float inv = 1.f / gscale;    // (a power of two)
  for (int j = k; j < end; ++j) {
    const float ca = st.coef[3 * j], cb = st.coef[3 * j + 1] * inv, cc = st.coef[3 * j + 2] * inv * inv;
    _Float16* z = q ? Z : spare;
    if (on)
      frag_store(w, square_product<K>(G, w.r0, G, w.c0), z, [&](int r, int c, float (&v)[4]) {
        const _Float16* g = G + pair_at(PA, r, c);
        const f16x4_t h = *reinterpret_cast<const f16x4_t*>(g), l = *reinterpret_cast<const f16x4_t*>(g + 32);
#pragma unroll
        for (int t = 0; t < 4; ++t) v[t] = cc * v[t] + cb * ((float)h[t] + (float)l[t]) + (r == c + t ? ca : 0.f);
      });
    __syncthreads();
    // Q between the steps is kept transposed, Q^T Z; the last product is Z (Q^T)^T, the rows that meet X
    if (on && q) frag_store(w, j + 1 < end ? square_product<K>(z, w.r0, q, w.c0) : square_product<K>(q, w.r0, z, w.c0), other, plain);
    if (second && j + 1 < end) frag_store(w, square_product<K>(G, w.r0, z, w.c0), R, plain);   // Z G
    __syncthreads();
    if (q) {
      _Float16* t = q;
      q = other;
      other = t;
    } else {
      q = z;
    }
    if (j + 1 < end) {
      // Z (Z G)^T (nobody reads G any more)
      if (on) frag_store(w, square_product<K>(R, w.r0, z, w.c0), G, plain);
      __syncthreads();
    }
  }
  return q;
}
__device__ __forceinline__ void zero_lds(void* p, int bytes, int threads) {
  for (int i = threadIdx.x; i < bytes / 16; i += threads) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
}
// result element o = old value of a parameter, x = f X
template <bool MUON>
__device__ __forceinline__ void emit_one(const Result& res, long long o, float x, float old) {
  if constexpr (MUON) res.p[o] = res.keep * old - x;
  else if (res.out_dtype == DAS_F32) reinterpret_cast<float*>(res.out)[o] = x;
  else reinterpret_cast<uint16_t*>(res.out)[o] = res.out_dtype == DAS_BF16 ? f32_to_bf16(x) : __builtin_bit_cast(uint16_t, (_Float16)x);
}

template <typename T, bool MUON, int QUADS, int K>
__device__ __forceinline__ void small_matrix(const NsMatrix& M, const DasNsSource& s, const MuonIn& mu, const Steps& st, const Result& res, char* smem,
                                             double* redd) {
  const int m16 = up16(M.m), n64 = up64(M.n), PX = 2 * n64 + 8, PF = n64 + 4;   // X's row pitch in f16 elements and in floats
  _Float16* X = reinterpret_cast<_Float16*>(smem);
  float* U = reinterpret_cast<float*>(smem);
  _Float16* A[N_AREAS];
#pragma unroll
  for (int i = 0; i < N_AREAS; ++i) A[i] = X + m16 * (PX + i * PA);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;

  // U, zeros around it and in the m x m matrices. The first loads go out before.
  const int count = M.rows * M.cols;
  const float per_row = 1.f / (float)M.cols;   // (index + 1/2) / cols is exact enough to truncate for indices under 2^20
  constexpr int BATCH = QUADS <= 2 ? 4 : 8;    // loads in flight per thread: a load a time is a memory latency each
  float coef = 1.f;
  double sum = 0.0;                            // (f64 holds the square of any f32: no scaling before the norm is known)
  if constexpr (MUON) coef = grad_factor(mu);
  for (int i0 = threadIdx.x; i0 < max(count, SMALL_TPB); i0 += BATCH * SMALL_TPB) {
    float v[BATCH], b[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * SMALL_TPB, r = (int)((i + 0.5f) * per_row), c = i - r * M.cols;
      v[k] = 0.f;
      if (i < count) {
        if constexpr (MUON) {
          v[k] = mu.g[M.src + i];
          b[k] = mu.buf[M.src + i];
        } else {
          v[k] = load_as_f32<T>(s.base, M.index * s.batch_stride + r * s.row_stride + c);
        }
      }
    }
    if (i0 < SMALL_TPB) {
      zero_lds(smem, 2 * m16 * (PX + N_AREAS * PA), SMALL_TPB);
      __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * SMALL_TPB, r = (int)((i + 0.5f) * per_row), c = i - r * M.cols;
      if (i >= count) continue;
      if constexpr (MUON) {
        v[k] = muon_in(mu, coef, v[k], b[k]);
        mu.buf[M.src + i] = b[k];
      }
      U[M.tall ? c * PF + r : r * PF + c] = v[k];
      sum += (double)v[k] * (double)v[k];
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
  if (lane == 0) redd[wave] = sum;
  __syncthreads();                             // (U is whole, too)
  sum = 0.0;
#pragma unroll
  for (int i = 0; i < SMALL_TPB / 64; ++i) sum += redd[i];
  const double f = (double)M.scale / (sqrt(sum) + (double)st.eps);
  float v[QUADS][4];
  const int quads = m16 * n64 / 4, per = n64 / 4;
#pragma unroll
  for (int b = 0; b < QUADS; ++b) {
    const int i = threadIdx.x + b * SMALL_TPB, r = i / per;
    if (i >= quads) continue;
    const float4 w = *reinterpret_cast<const float4*>(U + r * PF + (i - r * per) * 4);
    v[b][0] = (float)(w.x * f); v[b][1] = (float)(w.y * f); v[b][2] = (float)(w.z * f); v[b][3] = (float)(w.w * f);
  }
  __syncthreads();                             // (every read of U is done)
#pragma unroll
  for (int b = 0; b < QUADS; ++b) {
    const int i = threadIdx.x + b * SMALL_TPB, r = i / per;
    if (i < quads) put4(X + pair_at(PX, r, (i - r * per) * 4), v[b]);
  }
  __syncthreads();

  const Share w(m16);
  const int n = m16 >> 4, cols = n64 >> 4;
  const float gs = M.gscale / (M.scale * M.scale);
  for (int k = 0; k < st.steps;) {
    const int end = st.end[k];
    f32x4_t g = {};
    if (w.part < w.parts) g = long_product(X, PX, w.r0, w.c0, w.part, n64 >> 5, w.parts);
    store_gram(w, g, reinterpret_cast<f32x4_t*>(X + m16 * (PX + N_AREAS * PA)), A[0], gs);
    const _Float16* q = phase_chain<K>(w, A, st, k, end, M.gscale);
    const bool last = end == st.steps;
    f32x4_t acc[QUADS];
#pragma unroll
    for (int t = 0; t < QUADS; ++t) {
      const int x = t * 16 + wave, j = x / n;
      if (j < cols) acc[t] = update_fragment<K>(q, (x - j * n) * 16, X, PX, m16, j * 16);
    }
    __syncthreads();                    // (X has been read)
#pragma unroll
    for (int t = 0; t < QUADS; ++t) {
      const int x = t * 16 + wave, j = x / n;
      if (j >= cols) continue;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = (x - j * n) * 16 + (lane >> 4) * 4 + i, c = j * 16 + (lane & 15);
        const float y = acc[t][i];
        if (last) {
          U[r * PF + c] = y;
        } else {
          _Float16* p = X + pair_at(PX, r, c);
          const Pair h = pair_of(y);
          p[0] = h.high;
          p[32] = h.low;
        }
      }
    }
    __syncthreads();
    k = end;
  }

  const float factor = result_factor(M, res);
  for (int i0 = threadIdx.x; i0 < count; i0 += BATCH * SMALL_TPB) {
    float old[BATCH];
#pragma unroll
    for (int k = 0; k < BATCH; ++k) old[k] = MUON && i0 + k * SMALL_TPB < count ? res.p[M.src + i0 + k * SMALL_TPB] : 0.f;
#pragma unroll
    for (int k = 0; k < BATCH; ++k) {
      const int i = i0 + k * SMALL_TPB, r = (int)((i + 0.5f) * per_row), c = i - r * M.cols;
      if (i < count) emit_one<MUON>(res, M.src + i, factor * U[M.tall ? c * PF + r : r * PF + c], old[k]);
    }
  }
}

template <typename T, bool MUON, int QUADS>
__global__ __launch_bounds__(SMALL_TPB) void small_kernel(const NsMatrix* __restrict__ mats, Sources src, MuonIn mu, Steps st, Result res) {
  extern __shared__ __align__(16) char smem[];
  __shared__ double redd[SMALL_TPB / 64];
  const NsMatrix M = mats[blockIdx.x];
  if (!MUON && (unsigned)(M.group - src.first) >= (unsigned)src.count) return;   // (whole workgroups)
  const DasNsSource& s = src.s[MUON ? 0 : M.group - src.first];
  if (M.m <= 32) small_matrix<T, MUON, QUADS, 1>(M, s, mu, st, res, smem, redd);
  else small_matrix<T, MUON, QUADS, 2>(M, s, mu, st, res, smem, redd);
}

// A slice of a thin matrix: t.kn pieces of 128 columns from piece t.k0 on. FIRST: X = U's blocks times their exponents and 1 / norm (as
// normalise_kernel), and the slice's part of X X^T. MIDDLE: X = Q X, and the part. LAST: Q X goes to the result.
enum ThinKind { FIRST, MIDDLE, LAST };
constexpr int THIN_COLS = 128, PT = 2 * THIN_COLS + 8, PTF = THIN_COLS + 4;
template <ThinKind KIND, bool MUON>
__global__ __launch_bounds__(TPB) void thin_kernel(const NsMatrix* __restrict__ mats, const NsItem* __restrict__ items, float eps,
                                                   const Partial* __restrict__ norm_part, _Float16* __restrict__ X, const _Float16* __restrict__ Q,
                                                   f32x4_t* __restrict__ part, Result res) {
  __shared__ __align__(16) _Float16 xs[SMALL_M * PT], qs[SMALL_M * PA];
  __shared__ double red[4];
  const NsItem t = items[blockIdx.x];
  const NsMatrix M = mats[t.matrix];
  const int m16 = up16(M.m), n = m16 >> 4, lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k32 = (m16 + 31) >> 5;
  float* us = reinterpret_cast<float*>(xs);
  float factor = 1.f;
  double scale = 1.0;
  if constexpr (KIND == FIRST) {
    double s = 0.0;
    for (int i = threadIdx.x; i < M.chunks; i += TPB) {
      const Partial p = norm_part[M.chunk0 + i];
      s += ldexp((double)p.ss, 2 * p.e);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) red[wave] = s;
    __syncthreads();
    scale = (double)M.scale / (sqrt((red[0] + red[1]) + (red[2] + red[3])) + (double)eps);
  } else {
    if constexpr (KIND == LAST) factor = result_factor(M, res);
    for (int i = threadIdx.x; i < m16 * 16; i += TPB) {   // Q: rows of 256 bytes
      const int r = i >> 4, c = i & 15;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < M.m) v = *reinterpret_cast<const uint4*>(Q + 2 * M.a + r * 128 + c * 8);
      *reinterpret_cast<uint4*>(qs + r * PA + c * 8) = v;
    }
  }
  f32x4_t gram[4] = {};
  for (int piece = t.k0; piece < t.k0 + t.kn; ++piece) {
    __syncthreads();
    for (int i = threadIdx.x; i < m16 * 16; i += TPB) {   // 8 columns of a row a thread
      const int r = i >> 4, c = (i & 15) * 8;
      float v[8] = {};
      uint4 h = make_uint4(0, 0, 0, 0), l = h;
      _Float16* p = X + 2 * M.x + at(M.ldx, r, piece * THIN_COLS + c);
      if (r < M.m) {
        if constexpr (KIND == FIRST) {
          // (m <= 64: one row of blocks along the columns of X, whichever way the source lies)
          const int blk = piece * 2 + (c >> 6);
          const float f = (float)ldexp(scale, norm_part[M.chunk0 + blk].e);
          get(X + 2 * M.x, M.ldx, r, piece * THIN_COLS + c, v);
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] *= f;
          put(X + 2 * M.x, M.ldx, r, piece * THIN_COLS + c, v);
        } else {
          h = *reinterpret_cast<const uint4*>(p);
          l = *reinterpret_cast<const uint4*>(p + 32);
        }
      }
      if constexpr (KIND == FIRST) {
        f16x8_t a, b;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const Pair q = pair_of(v[e]);
          a[e] = q.high;
          b[e] = q.low;
        }
        h = __builtin_bit_cast(uint4, a);
        l = __builtin_bit_cast(uint4, b);
      }
      _Float16* d = xs + pair_at(PT, r, c);
      *reinterpret_cast<uint4*>(d) = h;
      *reinterpret_cast<uint4*>(d + 32) = l;
    }
    __syncthreads();
    if constexpr (KIND != FIRST) {
      f32x4_t acc[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int x = u * 4 + wave, j = x / n;
        if (j < 8)
          acc[u] = k32 == 1 ? update_fragment<1>(qs, (x - j * n) * 16, xs, PT, m16, j * 16) : update_fragment<2>(qs, (x - j * n) * 16, xs, PT, m16, j * 16);
      }
      __syncthreads();
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int x = u * 4 + wave, j = x / n;
        if (j >= 8) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = (x - j * n) * 16 + (lane >> 4) * 4 + i, c = j * 16 + (lane & 15);
          const float y = acc[u][i];
          if constexpr (KIND == LAST) {
            us[r * PTF + c] = y;
          } else {
            _Float16* p = xs + pair_at(PT, r, c);
            const Pair h = pair_of(y);
            p[0] = h.high;
            p[32] = h.low;
          }
        }
      }
      __syncthreads();
      if constexpr (KIND == MIDDLE) {
        for (int i = threadIdx.x; i < M.m * 32; i += TPB) {
          const int r = i >> 5, c = (i & 31) * 8;    // 16 bytes of a row of 512
          *reinterpret_cast<uint4*>(X + 2 * M.x + (long long)r * (2 * M.ldx) + piece * (2 * THIN_COLS) + c) =
              *reinterpret_cast<const uint4*>(xs + r * PT + c);
        }
      }
    }
    if constexpr (KIND == LAST) {
      const int c0 = piece * THIN_COLS, width = min(THIN_COLS, M.n - c0);
      const long long base = M.tall ? M.src + (long long)c0 * M.cols : M.src + c0;
      constexpr int BATCH = 8;
      for (int i0 = threadIdx.x; i0 < M.m * THIN_COLS; i0 += BATCH * TPB) {
        // tall: the piece is `width` whole rows of the source, one after the other; else THIN_COLS of each of its m rows
        long long o[BATCH];
        float x[BATCH], old[BATCH];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const int i = i0 + k * TPB, r = M.tall ? i % M.m : i / THIN_COLS, c = M.tall ? i / M.m : i % THIN_COLS;
          o[k] = i < M.m * THIN_COLS && c < width ? (M.tall ? base + i : base + (long long)r * M.cols + c) : -1;
          x[k] = o[k] >= 0 ? factor * us[r * PTF + c] : 0.f;
          old[k] = MUON && o[k] >= 0 ? res.p[o[k]] : 0.f;
        }
#pragma unroll
        for (int k = 0; k < BATCH; ++k)
          if (o[k] >= 0) emit_one<MUON>(res, o[k], x[k], old[k]);
      }
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int x = u * 4 + wave, i = x / n;
        if (i < n) {
          gram[u] += long_product(xs, PT, i * 16, (x - i * n) * 16, 0, THIN_COLS / 32, 1);
        }
      }
    }
  }
  if constexpr (KIND != LAST) {
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int x = u * 4 + wave;
      if (x < n * n) part[((long long)t.slot + x) * 64 + lane] = gram[u];
    }
  }
}

// One workgroup a thin matrix: X X^T from its slices' parts, the phase's steps, Q out
template <int K>
__device__ __forceinline__ void chain_matrix(const NsMatrix& M, const f32x4_t* part, int slices, _Float16* Q, const Steps& st, int k0, char* smem) {
  const int m16 = up16(M.m), n = m16 >> 4, lane = threadIdx.x & 63;
  _Float16* A[N_AREAS];
#pragma unroll
  for (int i = 0; i < N_AREAS; ++i) A[i] = reinterpret_cast<_Float16*>(smem) + i * m16 * PA;
  zero_lds(smem, 2 * N_AREAS * m16 * PA, SMALL_TPB);
  // thread = four values of a fragment; every one adds the slices' parts, eight loads in flight
  const int frags = n * n;
  f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
  if ((int)threadIdx.x < frags * 64) {
    for (int s0 = 0; s0 < slices; s0 += 8) {
      f32x4_t v[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) v[u] = s0 + u < slices ? part[(long long)(s0 + u) * frags * 64 + threadIdx.x] : f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int u = 0; u < 8; ++u) sum += v[u];
    }
  }
  __syncthreads();
  if ((int)threadIdx.x < frags * 64) {
    const int f = threadIdx.x >> 6, r = (f % n) * 16 + (lane & 15), c = (f / n) * 16 + (lane >> 4) * 4;   // (stored transposed, as frag_store)
    const float gs = M.gscale / (M.scale * M.scale), v[4] = {sum[0] * gs, sum[1] * gs, sum[2] * gs, sum[3] * gs};
    put4(A[0] + pair_at(PA, r, c), v);
  }
  __syncthreads();
  const Share w(m16);
  const _Float16* q = phase_chain<K>(w, A, st, k0, st.end[k0], M.gscale);
  for (int i = threadIdx.x; i < M.m * 16; i += SMALL_TPB) {
    const int r = i >> 4, c = i & 15;
    *reinterpret_cast<uint4*>(Q + 2 * M.a + r * 128 + c * 8) = *reinterpret_cast<const uint4*>(q + r * PA + c * 8);
  }
}
__global__ __launch_bounds__(SMALL_TPB) void chain_kernel(const NsMatrix* __restrict__ mats, const NsItem* __restrict__ slices, const int2* __restrict__ thin,
                                                          const f32x4_t* __restrict__ part, _Float16* __restrict__ Q, Steps st, int k) {
  extern __shared__ __align__(16) char smem[];
  const int2 range = thin[blockIdx.x];    // its slices
  const NsItem first = slices[range.x];
  const NsMatrix M = mats[first.matrix];
  if (M.m <= 32) chain_matrix<1>(M, part + (long long)first.slot * 64, range.y, Q, st, k, smem);
  else chain_matrix<2>(M, part + (long long)first.slot * 64, range.y, Q, st, k, smem);
}

// ------------------------------------------------------------------ host side
inline long long up256(long long v) { return (v + 255) / 256 * 256; }

struct Work {
  _Float16 *x[2], *a[N_AREAS];
  _Float16 *xt, *qt;         // thin matrices: X, Q
  f32x4_t* thin_part;        // parts of X X^T
  Partial* part;
  f32x4_t* slots;            // partial tiles
  long long bytes;
};
Work carve(const DasNsPlan* p, void* ws) {
  const long long xb = up256(4 * p->x_elems), ab = up256(4 * p->a_elems);
  char* c = (char*)ws;
  Work w = {};
  auto take = [&](long long n) { char* r = c; if (c) c += n; w.bytes += n; return r; };
  for (int i = 0; i < 2; ++i) w.x[i] = (_Float16*)take(xb);
  for (int i = 0; i < N_AREAS; ++i) w.a[i] = (_Float16*)take(ab);
  w.xt = (_Float16*)take(up256(4 * p->thin_x_elems));
  w.qt = (_Float16*)take(up256(4 * p->thin_a_elems));
  w.thin_part = (f32x4_t*)take(1024 * p->thin_slots);
  w.part = (Partial*)take(up256((long long)sizeof(Partial) * p->n_chunks));
  w.slots = (f32x4_t*)take(4 * std::max(p->gram_slots * p->gram_tile * p->gram_tile, 2 * p->product_slots * p->product_tile * p->product_tile));
  return w;
}

// Lets a kernel have a whole CU's dynamic LDS: asked of the runtime once a thread, device and kernel (in front of every launch: 0.4 us of
// host time each)
void allow_lds(const void* kernel) {
  constexpr int KERNELS = 64;
  thread_local const void* seen[KERNELS];
  thread_local int n = 0, of_dev = -1;
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess) return;
  if (dev != of_dev) n = 0;
  of_dev = dev;
  for (int i = 0; i < n; ++i)
    if (seen[i] == kernel) return;
  if (hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, SMALL_LDS) == hipSuccess && n < KERNELS) seen[n++] = kernel;
}

bool phases_valid(const DasNsPlan* p) {
  for (int k = 0; k < p->steps; ++k)
    if (p->phase_end[k] <= k || p->phase_end[k] > p->steps) return false;
  return true;
}
bool plan_valid(const DasNsPlan* p, const void* tables, const void* ws) {
  return p && tables && ws && p->n_matrices > 0 && p->n_small >= 0 && p->n_small <= p->n_matrices && p->steps > 0 &&
         p->steps <= DAS_NS_MAX_STEPS && phases_valid(p) && (p->product_tile == 64 || p->product_tile == 128) && (p->update_tile == 64 || p->update_tile == 128) &&
         !(((uintptr_t)tables | (uintptr_t)ws) & 15);
}

struct Bounds {              // of step k over the singular values that can reach it
  double top;                // |X| before the step
  double factor;             // max |a + b s^2 + c s^4|
};
// What f16 and the phases have to hold: X's norm, Z's norm step by step. false: outside f16's range.
bool polynomial_bounds(const float* coef, int steps, Bounds* out) {
  double top = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    double next = 0.0, factor = 0.0;
    for (int i = 0; i <= 4096; ++i) {
      const double x = top * i / 4096, y = x * x, z = std::fabs(a + b * y + c * y * y);
      factor = std::max(factor, z);
      next = std::max(next, x * z);
    }
    out[k] = Bounds{top, factor};
    top = next;
    if (!(top <= 16.0) || !(factor <= 64.0)) return false;
  }
  return true;
}

// where the phase that starts at step k ends
int phase_end(const Bounds* bound, int steps, int k) {
  double growth = bound[k].factor * bound[k].factor;
  int end = k + 1;
  while (end < steps && growth <= 256.0) {
    growth *= bound[end].factor * bound[end].factor;
    ++end;
  }
  return end;
}

// A second stream for the small and thin matrices of a set that holds others too: a chain of short launches that leaves the GPU nearly
// empty, beside the tiles' launches instead of before them, from their own part of the first pass on (fork and join by events; the
// caller's stream waits for the end). Streams of default priority, from a pool: one call has one for itself. A call that is being
// captured stays on its stream.
struct Side {
  int dev = 0;
  hipStream_t stream = nullptr;
  hipEvent_t fork = nullptr, join = nullptr;
};
class Fork {
 public:
  Fork(hipStream_t main, bool wanted) : main_(main) {
    if (!wanted) return;
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing(main, &st) != hipSuccess) {
      (void)hipGetLastError();
      return;
    }
    if (st != hipStreamCaptureStatusNone) return;
    side_ = take();
    if (side_ && (hipEventRecord(side_->fork, main) != hipSuccess || hipStreamWaitEvent(side_->stream, side_->fork, 0) != hipSuccess)) {
      (void)hipGetLastError();
      give(side_);
      side_ = nullptr;
    }
  }
  ~Fork() { (void)finish(); }
  hipStream_t stream() const { return side_ ? side_->stream : main_; }
  bool apart() const { return side_ != nullptr; }
  int finish() {
    if (!side_) return DAS_OK;
    const bool ok = hipEventRecord(side_->join, side_->stream) == hipSuccess && hipStreamWaitEvent(main_, side_->join, 0) == hipSuccess;
    if (!ok) (void)hipStreamSynchronize(side_->stream);   // (nothing of this call may run on after it is reported done)
    give(side_);
    side_ = nullptr;
    return ok ? DAS_OK : DAS_ERR_LAUNCH;
  }

 private:
  static std::mutex& mutex() {
    static std::mutex m;
    return m;
  }
  static std::vector<Side*>& pool() {
    static std::vector<Side*>* p = new std::vector<Side*>;   // (lives as long as the process: streams outlast static destructors)
    return *p;
  }
  static size_t& made() {
    static size_t n = 0;
    return n;
  }
  static Side* take() {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return nullptr;
    {
      std::lock_guard<std::mutex> lock(mutex());
      auto& p = pool();
      for (size_t i = 0; i < p.size(); ++i)
        if (p[i]->dev == dev) {
          Side* s = p[i];
          p.erase(p.begin() + i);
          return s;
        }
    }
    Side* s = new (std::nothrow) Side;
    if (!s) return nullptr;
    s->dev = dev;
    try {                // (room for it: giving it back never allocates)
      std::lock_guard<std::mutex> lock(mutex());
      pool().reserve(++made());
    } catch (...) {
      delete s;
      return nullptr;
    }
    if (hipStreamCreateWithFlags(&s->stream, hipStreamNonBlocking) != hipSuccess ||
        hipEventCreateWithFlags(&s->fork, hipEventDisableTiming) != hipSuccess ||
        hipEventCreateWithFlags(&s->join, hipEventDisableTiming) != hipSuccess) {
      (void)hipGetLastError();
      delete s;          // (a device that gives no stream: the call goes on without)
      return nullptr;
    }
    return s;
  }
  static void give(Side* s) {
    std::lock_guard<std::mutex> lock(mutex());
    pool().push_back(s);
  }
  hipStream_t main_;
  Side* side_ = nullptr;
};
// It pays beside launches of tens of microseconds (the detector's set 2276 -> 2216 us), that is with 128 x 128 tiles of the products;
// beside 64 x 64 ones where there is a whole chain of eight launches to hide, of small and of thin matrices, and tiles to hide it under:
// 700 x 513 (45 tiles) with one 64 x 64 and one 64 x 5000 254 -> 190 us in a queue of calls, 281 -> 248 alone; but 256 x 2304 (10 tiles)
// with one 16 x 16 and one 8 x 5000 161 -> 158 and 187 -> 200, 128 x 256 with five 64 x 64 114 -> 118, 700 x 513 with two 1 x 256 185 ->
// 194: its events cost the host 50 ... 80 us a call. Without tiles there is nothing to be beside (60 -> 85 us for five small and thin
// ones).
bool worth_a_fork(const DasNsPlan* p) {
  if (p->n_tile_chunks == 0 || p->n_small + p->n_thin == 0) return false;
  return p->product_tile == 128 || (p->n_small > 0 && p->n_thin > 0 && p->n_product >= 32);
}

Steps steps_of(const DasNsPlan* p) {
  Steps st;
  memcpy(st.coef, p->coef, sizeof(st.coef));
  memcpy(st.end, p->phase_end, sizeof(st.end));
  st.steps = p->steps;
  st.eps = p->eps;
  return st;
}

template <typename T, bool MUON>
int launch_small(const DasNsPlan* p, const char* tab, const Sources& src, const MuonIn& mu, const Result& res, hipStream_t s) {
  if (p->n_small == 0) return DAS_OK;
  auto launch = [&](auto kernel) {
    allow_lds((const void*)kernel);
    hipLaunchKernelGGL(kernel, dim3(p->n_small), dim3(SMALL_TPB), p->small_lds, s, (const NsMatrix*)(tab + p->mat_at), src, mu, steps_of(p), res);
  };
  if (p->small_quads <= 2) launch(small_kernel<T, MUON, 2>);
  else if (p->small_quads <= 4) launch(small_kernel<T, MUON, 4>);
  else launch(small_kernel<T, MUON, SMALL_QUADS>);
  DAS_CHECK_LAUNCH();
  return DAS_OK;
}

// thin matrices, after ingest_kernel
template <bool MUON>
int launch_thin(const DasNsPlan* p, const char* tab, const Work& w, const Result& res, hipStream_t s) {
  if (p->n_thin == 0) return DAS_OK;
  const NsMatrix* mats = (const NsMatrix*)(tab + p->mat_at);
  const NsItem* slices = (const NsItem*)(tab + p->slice_at);
  const int2* thin = (const int2*)(tab + p->thin_at);
  const Steps st = steps_of(p);
  constexpr int LDS = 2 * N_AREAS * SMALL_M * PA;
  allow_lds((const void*)chain_kernel);
  auto pass = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(p->n_slices), dim3(TPB), 0, s, mats, slices, p->eps, w.part, w.xt, w.qt, w.thin_part, res);
  };
  pass(thin_kernel<FIRST, false>);
  DAS_CHECK_LAUNCH();
  for (int k = 0; k < p->steps; k = p->phase_end[k]) {
    hipLaunchKernelGGL(chain_kernel, dim3(p->n_thin), dim3(SMALL_TPB), LDS, s, mats, slices, thin, w.thin_part, w.qt, st, k);
    DAS_CHECK_LAUNCH();
    if (p->phase_end[k] < p->steps) pass(thin_kernel<MIDDLE, false>);
    else pass(thin_kernel<LAST, MUON>);
    DAS_CHECK_LAUNCH();
  }
  return DAS_OK;
}

int iterate(const DasNsPlan* p, const char* tab, Work w, const Result& res, hipStream_t s) {
  const NsMatrix* mats = (const NsMatrix*)(tab + p->mat_at);
  const int4* chunks = (const int4*)(tab + p->chunk_at);
  const NsItem *gram = (const NsItem*)(tab + p->gram_at), *prod = (const NsItem*)(tab + p->product_at),
               *upd = (const NsItem*)(tab + p->update_at), *gram_join = (const NsItem*)(tab + p->gram_join_at),
               *prod_join = (const NsItem*)(tab + p->product_join_at);
  auto launch_sym = [&](auto kernel, int tile, int kg, const NsItem* items, int n, int products, const SymArgs& a) {
    const int lds = kg * 4 * tile * 128;
    allow_lds((const void*)kernel);
    hipLaunchKernelGGL(kernel, dim3(n, products), dim3(kg * TPB), lds, s, items, a, w.slots);
  };
  auto gram_of = [&](const _Float16* x, _Float16* g) {
    const SymArgs a = {{x}, {x}, {g}, 0.f, 0.f, 0.f, p->gram_slots};
    if (p->gram_kg == 4) launch_sym(sym_kernel<64, 4, GRAM>, 64, 4, gram, p->n_gram, 1, a);
    else if (p->gram_kg == 2) launch_sym(sym_kernel<128, 2, GRAM>, 128, 2, gram, p->n_gram, 1, a);
    else launch_sym(sym_kernel<128, 1, GRAM>, 128, 1, gram, p->n_gram, 1, a);
    if (p->n_gram_join && p->gram_kg == 4)
      hipLaunchKernelGGL((join_kernel<64, GRAM>), dim3(p->n_gram_join * 4), dim3(TPB), 0, s, gram_join, a, w.slots);
    else if (p->n_gram_join)
      hipLaunchKernelGGL((join_kernel<128, GRAM>), dim3(p->n_gram_join * 16), dim3(TPB), 0, s, gram_join, a, w.slots);
  };
  auto sym = [&](auto kind, int products, SymArgs a) {
    constexpr SymKind K = decltype(kind)::value;
    a.slots = p->product_slots;
    if (p->product_tile == 128 && p->product_kg == 2) launch_sym(sym_kernel<128, 2, K>, 128, 2, prod, p->n_product, products, a);
    else if (p->product_tile == 128) launch_sym(sym_kernel<128, 1, K>, 128, 1, prod, p->n_product, products, a);
    else launch_sym(sym_kernel<64, 4, K>, 64, 4, prod, p->n_product, products, a);
    if (p->n_product_join)
      hipLaunchKernelGGL((join_kernel<128, K>), dim3(p->n_product_join * 16, products), dim3(TPB), 0, s, prod_join, a, w.slots);
  };
  auto update = [&](auto last, const _Float16* q, const _Float16* x, _Float16* y) {
    constexpr bool L = decltype(last)::value;
    auto launch = [&](auto kernel, int tile, int kg) {
      const int lds = kg * 4 * tile * 128;
      allow_lds((const void*)kernel);
      hipLaunchKernelGGL(kernel, dim3(p->n_update), dim3(kg * TPB), lds, s, mats, upd, q, x, y, res);
    };
    if (p->update_tile == 128 && p->update_kg == 2) launch(update_kernel<128, 2, L>, 128, 2);
    else if (p->update_tile == 128) launch(update_kernel<128, 1, L>, 128, 1);
    else launch(update_kernel<64, 4, L>, 64, 4);
  };
  const std::integral_constant<SymKind, POLY> poly_k;
  const std::integral_constant<SymKind, PRODUCT> product_k;
  hipLaunchKernelGGL(normalise_kernel, dim3(p->n_tile_chunks), dim3(TPB), 0, s, mats, chunks, p->eps, w.x[0], w.part);
  DAS_CHECK_LAUNCH();
  _Float16 *X = w.x[0], *Y = w.x[1], *G = w.a[0], *R = w.a[1], *Z = w.a[2];
  for (int k = 0; k < p->steps;) {
    // steps k ... end - 1 are one phase
    const int end = p->phase_end[k];
    gram_of(X, G);
    _Float16 *q = nullptr, *spare = w.a[3], *other = w.a[4];   // (q: the phase's product so far)
    for (int j = k; j < end; ++j) {
      const float* c = p->coef + 3 * j;
      _Float16* z = q ? Z : spare;
      sym(poly_k, 1, SymArgs{{G}, {G}, {z}, c[0], c[1], c[2]});
      if (!q) {
        q = z;
        if (j + 1 < end) sym(product_k, 1, SymArgs{{z}, {G}, {R}, 0.f, 0.f, 0.f});
      } else if (j + 1 < end) {
        sym(product_k, 2, SymArgs{{z, z}, {q, G}, {other, R}, 0.f, 0.f, 0.f});
        std::swap(q, other);
      } else {
        sym(product_k, 1, SymArgs{{z}, {q}, {other}, 0.f, 0.f, 0.f});
        std::swap(q, other);
      }
      if (j + 1 < end) sym(product_k, 1, SymArgs{{R}, {z}, {G}, 0.f, 0.f, 0.f});
    }
    if (end < p->steps) update(std::false_type{}, q, X, Y);
    else update(std::true_type{}, q, X, Y);
    DAS_CHECK_LAUNCH();
    std::swap(X, Y);
    k = end;
  }
  return DAS_OK;
}

// the blocks of the first pass: those of thin matrices (behind the tiled ones' in the table) on the stream that goes on with them
template <typename F>
void launch_ingest(const DasNsPlan* p, const char* tab, const Fork& fork, hipStream_t s, F launch) {
  const int4* chunks = (const int4*)(tab + p->chunk_at);
  const int here = fork.apart() ? p->n_tile_chunks : p->n_chunks;
  if (here) launch(chunks, here, s);
  if (p->n_chunks > here) launch(chunks + here, p->n_chunks - here, fork.stream());
}

// thin and tiled matrices after ingest_kernel, and the join with the small ones
template <bool MUON>
int the_rest(const DasNsPlan* p, const char* tab, const Work& w, const Result& res, hipStream_t s, Fork& fork) {
  int st = launch_thin<MUON>(p, tab, w, res, fork.stream());
  if (st == DAS_OK && p->n_tile_chunks) st = iterate(p, tab, w, res, s);
  const int joined = fork.finish();
  return st != DAS_OK ? st : joined;
}

// Items of one launch. The hardware deals workgroups to the 8 XCDs in turn, and every XCD has its own 4 MiB L2: tiles that share rows
// or columns are kept together in a group, the XCDs' queues are filled evenly, longest inner axis first, and then
// interleaved (item i runs on XCD i % 8). (Tiles in table order: each XCD read nearly every panel itself, 512 x 4608: 47 us
// for X X^T at the Infinity Cache's rate.)
struct Launch {
  struct Group {
    std::vector<NsItem> items;
    long long cost = 0;
    int longest = 0;
  };
  std::vector<Group> groups;
  std::vector<NsItem> order;

  void add(bool fresh, const NsItem& t) {
    if (fresh || groups.empty()) groups.emplace_back();
    Group& g = groups.back();
    g.items.push_back(t);
    g.cost += t.kn + 2;        // (a tile's start and end cost about two steps of its inner axis)
    g.longest = std::max(g.longest, t.kn);
  }
  void place() {
    std::stable_sort(groups.begin(), groups.end(), [](const Group& u, const Group& v) {
      return u.longest != v.longest ? u.longest > v.longest : u.cost > v.cost;
    });
    std::vector<NsItem> queue[8];
    long long load[8] = {};
    for (size_t i = 0; i < groups.size();) {
      // groups of one length: the least loaded queues are filled up to the level that the whole class brings them to
      size_t end = i;
      long long cost = 0;
      for (; end < groups.size() && groups[end].longest == groups[i].longest; ++end) cost += groups[end].cost;
      int by_load[8] = {0, 1, 2, 3, 4, 5, 6, 7};
      std::stable_sort(by_load, by_load + 8, [&](int u, int v) { return load[u] < load[v]; });
      long long level = 0, sum = cost;
      for (int k = 0; k < 8; ++k) {
        sum += load[by_load[k]];
        level = (sum + k) / (k + 1);
        if (k == 7 || level <= load[by_load[k + 1]]) break;
      }
      int k = 0;
      for (; i < end; ++i)
        for (const NsItem& t : groups[i].items) {
          while (k < 7 && load[by_load[k]] + (t.kn + 2) / 2 > level) ++k;
          queue[by_load[k]].push_back(t);
          load[by_load[k]] += t.kn + 2;
        }
    }
    size_t depth = 0;
    for (const auto& q : queue) depth = std::max(depth, q.size());
    NsItem none = {};
    none.matrix = -1;
    for (size_t i = 0; i < depth; ++i)
      for (const auto& q : queue) order.push_back(i < q.size() ? q[i] : none);
    while (!order.empty() && order.back().matrix < 0) order.pop_back();
  }
};

struct Tables {
  std::vector<NsMatrix> mats;
  std::vector<int4> chunks;
  Launch gram, product, update;
  std::vector<NsItem> gram_join, product_join, slices;
  std::vector<int2> thin;    // first slice and slices of each thin matrix
  NsItem item(int q, int ti, int tj, int k0, int kn, int slot, int slots) const {
    const NsMatrix& M = mats[q];
    return NsItem{q, ti, tj, k0, kn, slot, slots, M.m, M.ldx, M.lda, M.scale, M.gscale, M.x, M.a};
  }
};

struct Tile {
  bool fresh;                // first of its group
  int matrix, ti, tj, steps;
};

// when the last of `slots` workers is done, longest pieces first; late (if given): the pieces that end after `limit`
long long makespan(const std::vector<int>& pieces, int slots, long long limit, std::vector<int>* late) {
  std::priority_queue<long long, std::vector<long long>, std::greater<long long>> free_at;
  for (int i = 0; i < slots; ++i) free_at.push(0);
  long long last = 0;
  for (size_t i = 0; i < pieces.size(); ++i) {
    const long long end = free_at.top() + pieces[i] + 2;
    free_at.pop();
    free_at.push(end);
    last = std::max(last, end);
    if (late && end > limit) late->push_back((int)i);
  }
  return last;
}

// Symmetric tiles of a launch for `slots` workgroups at a time. Tiles that would end after the others are split along the inner axis
// where that pays: 1056 equal tiles in 512 slots are two rounds and a sixteenth, and took the time of nearly three. A part costs 128 KiB
// of traffic, the join a launch: 0.0125 and 1.2 steps of 64 inner elements (2.5 us with two workgroups on a CU; 13 us measured for 272
// parts), six of the shorter steps of 64 x 64 tiles with four wave groups (4 ... 8 is level; 12: 8x 256 x 1024, Muon, 155 us instead of
// 150). A workgroup whose neighbour on the CU has ended runs up to twice as fast, so only half of what sticks out counts. A part has at
// least 4 steps.
void schedule(const Tables& tab, const std::vector<Tile>& tiles, int slots, double join_cost, Launch& launch, std::vector<NsItem>& join, long long& n_slots) {
  auto item = [&](auto... v) { return tab.item(v...); };
  std::vector<int> order(tiles.size()), parts(tiles.size(), 1), late;
  for (size_t i = 0; i < tiles.size(); ++i) order[i] = (int)i;
  std::stable_sort(order.begin(), order.end(), [&](int u, int v) { return tiles[u].steps > tiles[v].steps; });
  long long total = 0;
  std::vector<int> whole;
  for (int i : order) {
    total += tiles[i].steps + 2;
    whole.push_back(tiles[i].steps);
  }
  const double even = (double)total / slots;
  auto seen = [&](long long t) { return slots > 256 ? 0.5 * ((double)t + even) : (double)t; };
  double best = 0.95 * seen(makespan(whole, slots, (long long)(1.05 * even), &late));
  if (tiles.size() < 16u * slots && best > even) {
    std::vector<char> is_late(tiles.size(), 0);
    for (int k : late) is_late[k] = 1;
    int choice = 1;
    for (int p : {2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16}) {
      std::vector<int> pieces;
      long long count = 0;
      for (size_t k = 0; k < order.size(); ++k) {
        const int steps = whole[k], q = is_late[k] ? std::max(1, std::min(p, steps / 4)) : 1;
        for (int j = 0; j < q; ++j) pieces.push_back((int)((long long)steps * (j + 1) / q - (long long)steps * j / q));
        if (q > 1) count += q;
      }
      std::sort(pieces.begin(), pieces.end(), std::greater<int>());
      const double t = seen(makespan(pieces, slots, 0, nullptr)) + join_cost + 0.0125 * (double)count;
      if (t < best) {
        best = t;
        choice = p;
      }
    }
    for (size_t k = 0; k < order.size(); ++k)
      if (is_late[k]) parts[order[k]] = std::max(1, std::min(choice, whole[k] / 4));
  }
  // whole tiles in their blocks; a part of the inner axis, of all the split tiles of a matrix, is a group: one XCD alone reads it
  bool fresh = true;
  for (size_t i = 0; i < tiles.size(); ++i) {
    const Tile& t = tiles[i];
    fresh |= t.fresh;
    if (parts[i] > 1) continue;
    launch.add(fresh, item(t.matrix, t.ti, t.tj, 0, t.steps, -1, 1));
    fresh = false;
  }
  for (size_t i = 0; i < tiles.size();) {
    size_t end = i;
    while (end < tiles.size() && tiles[end].matrix == tiles[i].matrix) ++end;
    int most = 1;
    std::vector<int> slot(end - i, -1);
    for (size_t k = i; k < end; ++k) {
      if (parts[k] == 1) continue;
      most = std::max(most, parts[k]);
      slot[k - i] = (int)n_slots;
      join.push_back(item(tiles[k].matrix, tiles[k].ti, tiles[k].tj, 0, tiles[k].steps, (int)n_slots, parts[k]));
      n_slots += parts[k];
    }
    for (int j = 0; j < most && most > 1; ++j) {
      bool first = true;
      for (size_t k = i; k < end; ++k) {
        const int q = parts[k];
        if (q == 1 || j >= q) continue;
        const int k0 = (int)((long long)tiles[k].steps * j / q), k1 = (int)((long long)tiles[k].steps * (j + 1) / q);
        launch.add(first, item(tiles[k].matrix, tiles[k].ti, tiles[k].tj, k0, k1 - k0, slot[k - i] + j, 1));
        first = false;
      }
    }
    i = end;
  }
  launch.place();
}

inline int over(long long v, int t) { return (int)((v + t - 1) / t); }

// tiles on and below the diagonal of an m x m matrix, in blocks of `side` x `side` tiles: f(first of a block, row, column)
template <typename F>
void lower_blocks(int tiles, int side, F f) {
  for (int bi = 0; bi < tiles; bi += side)
    for (int bj = 0; bj <= bi; bj += side) {
      bool fresh = true;
      for (int i = bi; i < std::min(tiles, bi + side); ++i)
        for (int j = bj; j <= std::min(i, bj + side - 1); ++j, fresh = false) f(fresh, i, j);
    }
}

// The whole schedule of a set; false for shapes that it does not take.
bool build(const DasNsShape* shapes, int n, double top, DasNsPlan* plan, Tables& t) {
  std::vector<std::pair<long long, long long>> spans;
  long long n_mat = 0, n_chunks = 0;
  enum Class { SMALL, TILED, THIN };
  auto class_of = [](const DasNsShape& s) {
    const int m = std::min(s.rows, s.cols), nn = std::max(s.rows, s.cols);
    if (m > SMALL_M) return TILED;
    return small_lds(m, nn) <= SMALL_LDS && (long long)up16(m) * up64(nn) <= 4 * SMALL_QUADS * SMALL_TPB ? SMALL : THIN;
  };
  for (int g = 0; g < n; ++g) {
    const DasNsShape& s = shapes[g];
    if (s.off < 0 || s.off > (1LL << 60) || s.count < 1 || s.rows < 1 || s.cols < 1 || s.rows > (1 << 20) || s.cols > (1 << 20)) return false;
    const long long m = std::min(s.rows, s.cols), nn = std::max(s.rows, s.cols);
    n_mat += s.count;
    if (class_of(s) != SMALL) n_chunks += (long long)s.count * over(m, 64) * over(nn, 128) * 2;
    // (a launch has fewer than 2^32 threads: 1024 for a small matrix, 256 for a block)
    if (n_mat >= (1 << 22) || n_chunks >= (1 << 24) || m > (1 << 15)) return false;
    spans.push_back({s.off, s.off + (long long)s.count * s.rows * s.cols});
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return false;   // two workgroups would write the same elements
  plan->extent = spans.back().second;

  long long lower128 = 0, all128 = 0, lower64 = 0, all64 = 0;
  for (const Class cls : {SMALL, TILED, THIN}) {   // the order of the matrix and block tables
    for (int g = 0; g < n; ++g) {
      const DasNsShape& s = shapes[g];
      if (class_of(s) != cls) continue;
      for (int i = 0; i < s.count; ++i) {
        NsMatrix M = {};
        M.rows = s.rows; M.cols = s.cols; M.m = std::min(s.rows, s.cols); M.n = std::max(s.rows, s.cols);
        M.tall = s.rows > s.cols;
        M.thin = cls == THIN;
        M.ldx = over(M.n, 128) * 128; M.lda = over(M.m, 64) * 64;
        M.src = s.off + (long long)i * s.rows * s.cols;
        M.group = g; M.index = i;
        // X's largest entry is its norm's bound: as near to f16's end as a factor of two allows
        M.scale = (float)std::ldexp(1.0, (int)std::floor(std::log2(32768.0 / top)));
        // about m, and top^2 gscale within f16
        M.gscale = (float)std::ldexp(1.0, std::min((int)std::lround(std::log2((double)M.m)), (int)std::floor(std::log2(32768.0 / (top * top)))));
        if (cls == SMALL) {
          plan->n_small++;
          plan->small_lds = std::max(plan->small_lds, (int)small_lds(M.m, M.n));
          plan->small_quads = std::max(plan->small_quads, over((long long)up16(M.m) * up64(M.n), 4 * SMALL_TPB));
        } else {
          long long &x = cls == THIN ? plan->thin_x_elems : plan->x_elems, &a = cls == THIN ? plan->thin_a_elems : plan->a_elems;
          M.x = x; M.a = a; M.chunk0 = (int)t.chunks.size();
          x += (long long)M.m * M.ldx;
          a += (long long)M.m * M.lda;
          int k = 0;
          const int q = (int)t.mats.size();
          for (int r = 0; r < (M.tall ? M.ldx : M.lda) / CHUNK; ++r)
            for (int c = 0; c < (M.tall ? M.lda : M.ldx) / CHUNK; ++c) t.chunks.push_back(make_int4(q, r, c, k++));
          M.chunks = k;
          if (cls == TILED) {
            const long long tm = over(M.m, 128);
            lower128 += tm * (tm + 1) / 2;
            all128 += tm * (M.ldx / 128);
            lower64 += (long long)(M.lda / 64) * (M.lda / 64 + 1) / 2;
            all64 += (long long)(M.lda / 64) * (M.ldx / 64);
          } else {
            // at most 64 slices: the chain's workgroup reads all their parts
            const int pieces = M.ldx / THIN_COLS, per = over(pieces, 64), frags = up16(M.m) * up16(M.m) / 256;
            t.thin.push_back(make_int2((int)t.slices.size(), over(pieces, per)));
            for (int p = 0; p < pieces; p += per) {
              NsItem piece = {};
              piece.matrix = q; piece.k0 = p; piece.kn = std::min(per, pieces - p); piece.slot = (int)plan->thin_slots; piece.slots = frags;
              t.slices.push_back(piece);
              plan->thin_slots += frags;
            }
          }
        }
        t.mats.push_back(M);
      }
    }
    if (cls == TILED) plan->n_tile_chunks = (int)t.chunks.size();
  }
  const int tiled_end = (int)(t.mats.size() - t.thin.size());
  // Products and updates: 64 x 64 tiles whose inner axis four wave groups share while the 256 CUs have them in two rounds (9x 512x512,
  // Muon: 314 us, 372 with 128 x 128 ones), else 128 x 128 (24x 512x512: 435 us, 576 with 64 x 64 ones). Where a CU gets one of those,
  // two wave groups share it: at most 256 of an update, which has no second round to fill (512-channel bottleneck, 272 tiles: 233 us, 254
  // with two groups), under 384 of a product, whose long ones are split (2048x2048, 136 tiles: 1084 -> 853 us).
  plan->product_tile = lower64 > 512 ? 128 : 64;
  plan->product_kg = plan->product_tile == 64 ? 4 : lower128 >= 384 ? 1 : 2;
  plan->update_tile = all64 > 512 ? 128 : 64;
  plan->update_kg = plan->update_tile == 64 ? 4 : all128 > 256 ? 1 : 2;
  // X X^T, whose inner axis is long and may be split: 64 x 64 tiles and four wave groups for one round of the CUs (256 x 2304 123 us, 131
  // with 128 x 128 ones; 512 x 512 157, 165; 1024 x 1024 249, 254; but 12x 512 x 2048, 432 tiles: 486, 470 with 128 x 128 ones), then 128
  // x 128; where there are fewer than 384 of those, two wave groups share a tile (one workgroup a CU, not two)
  plan->gram_tile = lower64 <= 256 ? 64 : 128;
  plan->gram_kg = lower64 <= 256 ? 4 : lower128 >= 384 ? 1 : 2;
  // blocks of up to 8 x 8 tiles, smaller where one would be more than a 16th of the launch (half of an XCD's part)
  auto side_for = [](long long launch, int steps) {
    int side = 8;
    while (side > 1 && (long long)side * side * (steps + 2) * 16 > launch) side /= 2;
    return side;
  };
  long long product_cost = 0, update_cost = 0, gram_cost = 0;
  for (int q = plan->n_small; q < tiled_end; ++q) {
    const NsMatrix& M = t.mats[q];
    const long long p = over(M.m, plan->product_tile), r = over(M.m, plan->update_tile), w = over(M.m, plan->gram_tile);
    product_cost += p * (p + 1) / 2 * (M.lda / 64 + 2);
    update_cost += r * (M.ldx / plan->update_tile) * (M.lda / 64 + 2);
    gram_cost += w * (w + 1) / 2 * (M.ldx / 64 + 2);
  }
  std::vector<Tile> gram, product;
  for (int q = plan->n_small; q < tiled_end; ++q) {
    const NsMatrix& M = t.mats[q];
    lower_blocks(over(M.m, plan->gram_tile), side_for(gram_cost, M.ldx / 64),
                 [&](bool fresh, int i, int j) { gram.push_back(Tile{fresh, q, i, j, M.ldx / 64}); });
    lower_blocks(over(M.m, plan->product_tile), side_for(product_cost, M.lda / 64),
                 [&](bool fresh, int i, int j) { product.push_back(Tile{fresh, q, i, j, M.lda / 64}); });
    const int rows = over(M.m, plan->update_tile), cols = M.ldx / plan->update_tile, side = side_for(update_cost, M.lda / 64);
    for (int bj = 0; bj < cols; bj += side)
      for (int bi = 0; bi < rows; bi += side)
        for (int j = bj; j < std::min(cols, bj + side); ++j)
          for (int i = bi; i < std::min(rows, bi + side); ++i) t.update.add(i == bi && j == bj, t.item(q, i, j, 0, M.lda / 64, -1, 1));
  }
  schedule(t, gram, plan->gram_kg == 1 ? 512 : 256, plan->gram_kg == 4 ? 6.0 : 1.2, t.gram, t.gram_join, plan->gram_slots);
  if (plan->product_tile == 128) {
    schedule(t, product, plan->product_kg == 1 ? 512 : 256, 1.2, t.product, t.product_join, plan->product_slots);
  } else {
    for (const Tile& p : product) t.product.add(p.fresh, t.item(p.matrix, p.ti, p.tj, 0, p.steps, -1, 1));
    t.product.place();
  }
  t.update.place();
  // (KG x 256 threads for an item, 16 x 256 for a joined tile)
  return std::max({t.gram.order.size(), t.product.order.size(), t.update.order.size()}) < (1u << 22) &&
         std::max(t.gram_join.size(), t.product_join.size()) < (1u << 20);
}

}  // namespace

extern "C" int das_ns_plan(const DasNsShape* shapes, int n, int steps, const float* coef, float eps, DasNsPlan* plan, void* tables,
                           long long table_bytes) {
  Bounds bound[DAS_NS_MAX_STEPS];
  if (!shapes || n < 1 || !coef || !plan || steps < 1 || steps > DAS_NS_MAX_STEPS || !(eps >= 0.f) || !std::isfinite(eps) ||
      !polynomial_bounds(coef, steps, bound))
    return DAS_ERR_ARG;
  double top = 1.0;
  for (int k = 0; k < steps; ++k) top = std::max(top, bound[k].top);
  try {
    DasNsPlan p;
    memset(&p, 0, sizeof(p));
    Tables t;
    if (!build(shapes, n, top, &p, t)) return DAS_ERR_ARG;
    p.n_groups = n; p.n_matrices = (int)t.mats.size(); p.n_chunks = (int)t.chunks.size();
    p.n_gram = (int)t.gram.order.size(); p.n_product = (int)t.product.order.size(); p.n_update = (int)t.update.order.size();
    p.n_thin = (int)t.thin.size(); p.n_slices = (int)t.slices.size();
    p.n_gram_join = (int)t.gram_join.size(); p.n_product_join = (int)t.product_join.size();
    p.steps = steps; p.eps = eps;
    for (int k = 0; k < steps; ++k) p.phase_end[k] = phase_end(bound, steps, k);
    memcpy(p.coef, coef, sizeof(float) * 3 * steps);
    char* out = nullptr;
    auto put_table = [&](const auto& v, long long& at) {
      at = p.table_bytes;
      const long long bytes = (long long)(v.size() * sizeof(v[0]));
      if (out && bytes) memcpy(out + at, v.data(), bytes);
      p.table_bytes += up256(bytes);
    };
    for (int pass = 0; pass < (tables ? 2 : 1); ++pass) {
      if (pass) {
        if (table_bytes < p.table_bytes) return DAS_ERR_ARG;
        out = (char*)tables;
        memset(tables, 0, p.table_bytes);
      }
      p.table_bytes = 0;
      put_table(t.mats, p.mat_at);
      put_table(t.chunks, p.chunk_at);
      put_table(t.gram.order, p.gram_at);
      put_table(t.gram_join, p.gram_join_at);
      put_table(t.product.order, p.product_at);
      put_table(t.product_join, p.product_join_at);
      put_table(t.update.order, p.update_at);
      put_table(t.slices, p.slice_at);
      put_table(t.thin, p.thin_at);
    }
    *plan = p;
  } catch (...) {   // (no memory for the tables)
    return DAS_ERR_ARG;
  }
  return DAS_OK;
}

extern "C" long long das_ns_ws_bytes(const DasNsPlan* p) {
  if (!p) return -1;
  return std::max(256LL, carve(p, nullptr).bytes);
}

extern "C" int das_orthogonalize(const DasNsPlan* plan, const void* tables_dev, const DasNsSource* srcs, int n_srcs, int in_dtype,
                                 void* out, int out_dtype, void* ws, void* stream) {
  DAS_PROF(stream);
  if (!plan_valid(plan, tables_dev, ws) || !srcs || n_srcs != plan->n_groups || !out || out_dtype < DAS_F32 || out_dtype > DAS_F16 ||
      in_dtype < DAS_F32 || in_dtype > DAS_F16)
    return DAS_ERR_ARG;
  for (int i = 0; i < n_srcs; ++i)
    if (!srcs[i].base) return DAS_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const char* tab = (const char*)tables_dev;
  const Work w = carve(plan, ws);
  const NsMatrix* mats = (const NsMatrix*)(tab + plan->mat_at);
  const MuonIn none = {};
  const Result res = {out, out_dtype, nullptr, 1.f, 0.f, 0};
  Fork fork(s, worth_a_fork(plan));
  // one launch for every 64 source tensors (one in all but unusual sets): its workgroups of other tensors' blocks end at once
  for (int first = 0; first < n_srcs; first += Sources::MAX) {
    Sources a;
    a.first = first;
    a.count = std::min(Sources::MAX, n_srcs - first);
    for (int i = 0; i < Sources::MAX; ++i) a.s[i] = srcs[first + std::min(i, a.count - 1)];
    int st = DAS_OK;
    if (in_dtype == DAS_F32) st = launch_small<float, false>(plan, tab, a, none, res, fork.stream());
    else if (in_dtype == DAS_BF16) st = launch_small<bf16_t, false>(plan, tab, a, none, res, fork.stream());
    else st = launch_small<_Float16, false>(plan, tab, a, none, res, fork.stream());
    if (st != DAS_OK) return st;
    auto launch = [&](auto kernel) {
      launch_ingest(plan, tab, fork, s, [&](const int4* chunks, int n, hipStream_t on) {
        hipLaunchKernelGGL(kernel, dim3(n), dim3(TPB), 0, on, mats, chunks, a, none, w.x[0], w.xt, w.part);
      });
    };
    if (in_dtype == DAS_F32) launch(ingest_kernel<float, false>);
    else if (in_dtype == DAS_BF16) launch(ingest_kernel<bf16_t, false>);
    else launch(ingest_kernel<_Float16, false>);
    DAS_CHECK_LAUNCH();
  }
  return the_rest<false>(plan, tab, w, res, s, fork);
}

extern "C" int das_muon_step(const DasNsPlan* plan, const void* tables_dev, float* p, const float* g, float* buf, double lr,
                             double momentum, double weight_decay, int nesterov, int lr_scale, float grad_scale, float max_norm,
                             const float* grad_sumsq, void* ws, void* stream) {
  DAS_PROF(stream);
  if (!plan_valid(plan, tables_dev, ws) || !p || !g || !buf || !(momentum >= 0 && momentum < 1) || !(lr >= 0) ||
      !(weight_decay >= 0) || (max_norm > 0.f && !grad_sumsq) || lr_scale < 0 || lr_scale > 1)
    return DAS_ERR_ARG;
  if (((uintptr_t)p | (uintptr_t)g | (uintptr_t)buf) & 3) return DAS_ERR_ARG;
  const long long bytes = 4 * plan->extent;
  if (buffers_overlap(p, g, bytes) || buffers_overlap(p, buf, bytes) || buffers_overlap(g, buf, bytes)) return DAS_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const char* tab = (const char*)tables_dev;
  const Work w = carve(plan, ws);
  const MuonIn mu = {g, buf, (float)momentum, (float)(1.0 - momentum), grad_scale, max_norm, nesterov, grad_sumsq};
  const Result res = {nullptr, 0, p, (float)(1.0 - lr * weight_decay), (float)lr, lr_scale};
  Fork fork(s, worth_a_fork(plan));
  const int st = launch_small<float, true>(plan, tab, Sources{}, mu, res, fork.stream());
  if (st != DAS_OK) return st;
  launch_ingest(plan, tab, fork, s, [&](const int4* chunks, int n, hipStream_t on) {
    hipLaunchKernelGGL((ingest_kernel<float, true>), dim3(n), dim3(TPB), 0, on, (const NsMatrix*)(tab + plan->mat_at), chunks, Sources{}, mu,
                       w.x[0], w.xt, w.part);
  });
  DAS_CHECK_LAUNCH();
  return the_rest<true>(plan, tab, w, res, s, fork);
}
