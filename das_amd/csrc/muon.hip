// Newton-Schulz orthogonalisation of a ragged set of matrices, and the Muon step around it (include/das_hip.h).
//
// For U (rows x cols; m = min, n = max; transposed if rows > cols, so X is m x n):  X = U / (|U|_F + eps), then `steps` times
// X = (a I + b X X^T + c (X X^T)^2) X: in singular values s -> s (a + b s^2 + c s^4). All matrices of a set go through the same launches:
// a table (built once on the host, das_ns_plan) lists every tile of every matrix, one workgroup per tile.
//
// Two precisions, by the type of the result.
// f16 / bf16 results: X, G and Z are f16 (11 bits; bf16's 8 would make the error 8 times larger at the same matrix-pipe rate), sums f32.
//   G = X X^T   Z = a I + b G + c G G   X = Z X                            15 m m n + 5 m^3 flops for five steps
//   (a symmetric product is computed on and below its diagonal). 1e-3 off 64-bit arithmetic for a training run's gradients.
// f32 results (parameters, whose last bits a learning rate of 1e-2 already reaches): every operand is a pair of f16, high + low part, 22
//   bits, and a product is three (high high + high low + low high). To pay for it the m x n matrix is touched as seldom as possible: Z(G)
//   commutes with G, so several steps can be taken on m x m matrices alone,
//     Q = Z Q,  G' = X' X'^T = Z G Z      and X' = Q X at the end of such a phase:   18 m m n + 42 m^3 for five steps
//   (plain steps with three products: 45 m m n + 15 m^3). A phase ends before an error of G, which grows by (a + b s^2 + c s^4)^2 a step
//   in the direction of small singular values s while G's true entries there grow alike but start smaller, has grown 256-fold: with
//   the default polynomial three steps, then two. 5e-5 ... 2e-4 off 64-bit arithmetic for any spectrum (f32 throughout: 1e-6 ... 5e-5).
//
// Scales keep entries among f16's normal numbers: X is kept times S = 2^round(log2 sqrt(n)) (an orthogonal X has entries of 1 /
// sqrt(n)), G times gscale, about m (its trace starts at one). Row lengths are padded with zeros (ldx, lda) to whole stages of the inner axis.
#include <algorithm>
#include <cmath>
#include <cstring>
#include <type_traits>
#include <vector>

#include "common.h"
#include "prof.h"

namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));

constexpr int TPB = 256;
constexpr int CHUNK = 64;   // side of the blocks that ingest_kernel / normalise_kernel work on

struct NsMatrix {           // one matrix, as the kernels see it
  long long src;            // element offset in the flat buffers / in the result
  long long x, a;           // element offsets in the work areas X (m x ldx) and A, B (m x lda)
  int rows, cols, m, n, ldx, lda;
  int group, index;         // source tensor and matrix in it (das_orthogonalize)
  int chunk0, chunks;       // its blocks in the partial-sum table
  float scale, gscale;      // S; what G is kept times
  int tall;                 // rows > cols: X holds the transpose
};
struct Partial {            // of one 64 x 64 block: sum of squares of (u 2^-e), and e
  float ss;
  int e;
};

// N (4 or 8) neighbouring values of a row of a work matrix (SPLIT: 32 high parts, then their 32 low parts, and so on along the row)
template <bool SPLIT>
__device__ __forceinline__ long long at(int ld, int r, int c) {
  return SPLIT ? (long long)r * (2 * ld) + (c >> 5) * 64 + (c & 31) : (long long)r * ld + c;
}
template <bool SPLIT, int N>
__device__ __forceinline__ void put(_Float16* base, int ld, int r, int c, const float (&v)[N]) {
  typedef _Float16 vec_t __attribute__((ext_vector_type(N)));
  _Float16* p = base + at<SPLIT>(ld, r, c);
  vec_t h, l;
#pragma unroll
  for (int e = 0; e < N; ++e) {
    h[e] = (_Float16)v[e];
    l[e] = (_Float16)(v[e] - (float)h[e]);
  }
  *reinterpret_cast<vec_t*>(p) = h;
  if constexpr (SPLIT) *reinterpret_cast<vec_t*>(p + 32) = l;
}
template <bool SPLIT, int N>
__device__ __forceinline__ void get(const _Float16* base, int ld, int r, int c, float (&v)[N]) {
  typedef _Float16 vec_t __attribute__((ext_vector_type(N)));
  const _Float16* p = base + at<SPLIT>(ld, r, c);
  const vec_t h = *reinterpret_cast<const vec_t*>(p);
  vec_t l = {};
  if constexpr (SPLIT) l = *reinterpret_cast<const vec_t*>(p + 32);
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
  float momentum, grad_scale, max_norm;
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

template <typename T>
__device__ __forceinline__ float load_as_f32(const void* base, long long i) {
  const T v = reinterpret_cast<const T*>(base)[i];
  if constexpr (std::is_same<T, bf16_t>::value) return bf16_to_f32(v);
  else return (float)v;
}

// One 64 x 64 block of U: update the momentum (Muon), find the block's exponent e (largest entry in [1/2, 1) 2^(e + 10)) and sum of
// squares, store u 2^-e in X's layout (transposed through LDS for tall matrices), zeros in the padding. The exponent keeps gradients
// of any magnitude inside f16's range until the norm is known; normalise_kernel rounds a second time.
template <typename T, bool MUON, bool SPLIT>
__global__ __launch_bounds__(TPB) void ingest_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ chunks,
                                                     Sources src, MuonIn mu, _Float16* __restrict__ X, Partial* __restrict__ part) {
  __shared__ float tile[CHUNK][CHUNK + 1];
  __shared__ float red[4];
  const int4 ch = chunks[blockIdx.x];
  const NsMatrix M = mats[ch.x];
  if (!MUON && (unsigned)(M.group - src.first) >= (unsigned)src.count) return;   // (whole workgroups)
  const int r0 = ch.y * CHUNK, c0 = ch.z * CHUNK;
  const int c4 = (threadIdx.x & 15) * 4, rr = threadIdx.x >> 4;
  float coef = 1.f;
  if constexpr (MUON) {
    coef = mu.grad_scale;
    if (mu.max_norm > 0.f) {
      const float k = mu.max_norm / (sqrtf(*mu.sumsq) * mu.grad_scale + 1e-6f);
      coef *= k > 1.f ? 1.f : k;   // (a NaN norm stays NaN)
    }
  }
  float u[4][4], big = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = r0 + rr + k * 16;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int c = c0 + c4 + j;
      float v = 0.f;
      if (r < M.rows && c < M.cols) {
        if constexpr (MUON) {
          const long long i = M.src + (long long)r * M.cols + c;
          const float g = mu.g[i] * coef;
          const float b = mu.momentum * mu.buf[i] + (1.f - mu.momentum) * g;
          mu.buf[i] = b;
          v = mu.nesterov ? (1.f - mu.momentum) * g + mu.momentum * b : b;
        } else {
          const DasNsSource& s = src.s[M.group - src.first];
          v = load_as_f32<T>(s.base, M.index * s.batch_stride + r * s.row_stride + c);
        }
      }
      u[k][j] = v;
      big = fmaxf(big, fabsf(v));   // (NaN is passed over here and stays NaN in u)
    }
  }
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
    put<SPLIT>(X + (SPLIT ? 2 : 1) * M.x, M.ldx, r, x_c0 + c4, u[k]);
  }
}

// X <- X 2^e S / (|U|_F + eps), block by block. Every workgroup sums its matrix's partials itself, in one fixed order, in f64.
template <bool SPLIT>
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
    _Float16* x = X + (SPLIT ? 2 : 1) * M.x;
    float v[4];
    get<SPLIT>(x, M.ldx, r, x_c0 + c4, v);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] *= f;
    put<SPLIT>(x, M.ldx, r, x_c0 + c4, v);
  }
}

// ------------------------------------------------------------------ products
// T x T tile (T = 128 or 64) of one matrix by four waves of T/2 x T/2, v_mfma_f32_16x16x32_f16: lane l holds row l % 16 of A (column of
// B), inner elements (l / 16) * 8 ... + 8, and gets column l % 16, rows (l / 16) * 4 ... + 4 of the result.
//
// A stage is 128 bytes of every row of both operands: 64 inner elements, or (SPLIT) 32 high parts and their 32 low parts, which lie next to
// each other in memory so that both forms read whole 128-byte lines. It is copied global -> LDS without passing registers, into
// one of two buffers while the other is multiplied; the fragments are read before the next copies are issued, so no LDS read waits for them.
//   plain:  acc += A0 B0 + A1 B1   (two halves of the inner axis)
//   SPLIT:  acc += Ah Bh + Ah Bl + Al Bh   (the low x low part is 2^-22 of the product)
// LDS images. Rows by rows (gram, product, and B of the update): two panels of T rows x 64 bytes, 16-byte slot s of row r holds source
// slot s ^ (r / 2 % 4): eight neighbouring rows cover all banks. Columns of X (update): inner rows as they are in memory, 32-byte units
// swizzled by row, read with ds_read_tr16_b64 (four inner rows x 16 columns a 16-lane group, one column a lane).
typedef short i16x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ void copy16(const void* src, char* lds_wave_base) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds_wave_base, 16, 0, 0);
}

template <int T>
struct RowsOperand {        // T rows of a matrix whose rows run along the inner axis
  const char* src[T / 32];
  __device__ __forceinline__ void init(const _Float16* base, int pitch, int row0, int rows) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      const int q = wave * (T / 32) + i, r = (q >> 1) * 16 + (lane >> 2), kg = (lane & 3) ^ ((r >> 1) & 3);
      src[i] = (const char*)(base + (long long)min(row0 + r, rows - 1) * pitch + (q & 1) * 32 + kg * 8);   // (rows past the end: stand-ins)
    }
  }
  __device__ __forceinline__ void issue(char* lds) {
    const int wave = threadIdx.x >> 6;
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

template <int T, bool SPLIT>
struct ColsOperand {        // T columns of a matrix whose rows run across the inner axis
  static constexpr int ROWB = SPLIT ? T * 4 : T * 2, LPR = ROWB / 16, ROWS = SPLIT ? 32 : 64;   // bytes and lanes of a row, rows of a stage
  const char* base;
  int pitch, rows, row;     // bytes; rows of the matrix; this lane's row in the first copy
  int slot;
  static __device__ __forceinline__ int swz(int r) {
    return ROWB >= 256 ? ((r & 3) | ((r >> 1) & 4)) : (((r >> 1) & 1) | ((r >> 2) & 2));
  }
  __device__ __forceinline__ void init(const _Float16* x, int pitch_elems, int col0, int rows_) {
    base = (const char*)(x + col0 * (SPLIT ? 2 : 1));
    pitch = pitch_elems * 2;
    rows = rows_;
    row = 0;
  }
  __device__ __forceinline__ void issue(char* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
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
    const int unit = SPLIT ? (c >> 5) * 4 + p * 2 + ((c >> 4) & 1) : c >> 4;
    i16x4_t v[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = (SPLIT ? 0 : p * 32) + (lane >> 4) * 8 + h * 4 + (q >> 2);
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

template <int T, bool SPLIT, typename OB>
__device__ __forceinline__ void multiply(RowsOperand<T>& a, OB& b, int stages, char* smem, Acc<T>& acc) {
  constexpr int HALF = T * 128, N = T / 32;   // bytes of one operand's stage; fragments a wave has of each operand
  const int wave = threadIdx.x >> 6, wr = (wave >> 1) * (T / 2), wc = (wave & 1) * (T / 2);
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  a.issue(smem);
  b.issue(smem + HALF);
  __syncthreads();
  for (int k = 0; k < stages; ++k) {
    const char* cur = smem + (k & 1) * 2 * HALF;
    char* nxt = smem + ((k & 1) ^ 1) * 2 * HALF;
    f16x8_t fa[2][N], fb[2][N];
#pragma unroll
    for (int p = 0; p < 2; ++p)
#pragma unroll
      for (int t = 0; t < N; ++t) {
        fa[p][t] = RowsOperand<T>::frag(cur, wr, t, p);
        fb[p][t] = OB::frag(cur + HALF, wc, t, p);
      }
    if (k + 1 < stages) {
      a.issue(nxt);
      b.issue(nxt + HALF);
    }
#pragma unroll
    for (int q = 0; q < (SPLIT ? 3 : 2); ++q)   // plain: 00 11; split: low parts first (10, 01), then 00
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const int pa = SPLIT ? q == 0 : q, pb = SPLIT ? q == 1 : q;
          acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[pa][i], fb[pb][j], acc[i][j], 0, 0, 0);
        }
    __syncthreads();
  }
}

// The tile through LDS, row by row: f(row, col, eight values of the row). TRANSPOSED: rows and columns of the tile exchanged.
template <int T, bool TRANSPOSED, typename F>
__device__ __forceinline__ void store_tile(const Acc<T>& acc, char* smem, F f) {
  constexpr int P = T + 4;   // floats of a row: the four row groups of a fragment start 16 banks apart
  float* buf = reinterpret_cast<float*>(smem);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int major = (TRANSPOSED ? wave & 1 : wave >> 1) * (T / 2), minor = (TRANSPOSED ? wave >> 1 : wave & 1) * (T / 2);
  for (int r0 = 0; r0 < T; r0 += 64) {
    __syncthreads();
    if (T == 64 || major == r0) {
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
    constexpr int TPR = T / 8, RPS = TPB / TPR;
#pragma unroll
    for (int s = 0; s < 64 / RPS; ++s) {
      const int r = s * RPS + threadIdx.x / TPR, c = (threadIdx.x % TPR) * 8;
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
};

// Symmetric m x m results, tiles on and below the diagonal, each stored as it is and transposed.
//   GRAM:     G = X X^T times (gscale / S^2)      POLY: Z = a I + b G + c G G      PRODUCT: P Q of symmetric P, Q that commute
// Columns m ... lda are stored as zeros: the inner axis of the next product.
template <int T, bool SPLIT, SymKind KIND>
__global__ __launch_bounds__(TPB, 2) void sym_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ tiles, SymArgs s) {
  __shared__ __align__(16) char smem[4 * T * 128];
  const int4 t = tiles[blockIdx.x];
  const NsMatrix M = mats[t.x];
  const int z = blockIdx.y, i0 = t.y * T, j0 = t.z * T;
  const int ld = KIND == GRAM ? M.ldx : M.lda, pitch = SPLIT ? 2 * ld : ld;
  const _Float16* P = s.p[z] + (SPLIT ? 2 : 1) * (KIND == GRAM ? M.x : M.a);
  const _Float16* Q = s.q[z] + (SPLIT ? 2 : 1) * (KIND == GRAM ? M.x : M.a);
  RowsOperand<T> a, b;
  a.init(P, pitch, i0, M.m);
  b.init(Q, pitch, j0, M.m);
  Acc<T> acc;
  multiply<T, SPLIT>(a, b, pitch / 64, smem, acc);
  _Float16* out = s.out[z] + (SPLIT ? 2 : 1) * M.a;
  const float f = KIND == GRAM ? M.gscale / (M.scale * M.scale) : 1.f, cb = s.b / M.gscale, cc = s.c / (M.gscale * M.gscale);
  auto store = [&](int r, int c, float (&v)[8]) {
    if (r >= M.m || c >= M.lda) return;
    if constexpr (KIND == POLY) {
      float g[8];
      get<SPLIT>(P, M.lda, r, c, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = cc * v[e] + cb * g[e] + (r == c + e ? s.a : 0.f);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= f;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e >= M.m) v[e] = 0.f;
    put<SPLIT>(out, M.lda, r, c, v);
  };
  store_tile<T, false>(acc, smem, [&](int r, int c, float (&v)[8]) { store(i0 + r, j0 + c, v); });
  if (i0 != j0) store_tile<T, true>(acc, smem, [&](int r, int c, float (&v)[8]) { store(j0 + r, i0 + c, v); });
}

struct Result {             // where the last product goes
  void* out;                // das_orthogonalize
  int out_dtype;
  float* p;                 // das_muon_step: p = keep p - lr f X
  float keep, lr;
  int lr_scale;
};

// X' = Q X: Q's rows by X's columns. LAST: the result leaves the work area (and its scale S), transposed back where needed.
template <int T, bool SPLIT, bool LAST>
__global__ __launch_bounds__(TPB, 2) void update_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ tiles,
                                                        const _Float16* __restrict__ Q, const _Float16* __restrict__ X,
                                                        _Float16* __restrict__ Y, Result res) {
  __shared__ __align__(16) char smem[4 * T * 128];
  const int4 t = tiles[blockIdx.x];
  const NsMatrix M = mats[t.x];
  const int i0 = t.y * T, j0 = t.z * T;
  constexpr int W = SPLIT ? 2 : 1;
  RowsOperand<T> a;
  ColsOperand<T, SPLIT> b;
  a.init(Q + W * M.a, W * M.lda, i0, M.m);
  b.init(X + W * M.x, W * M.ldx, j0, M.m);
  Acc<T> acc;
  multiply<T, SPLIT>(a, b, W * M.lda / 64, smem, acc);
  if constexpr (!LAST) {
    store_tile<T, false>(acc, smem, [&](int r, int c, float (&v)[8]) {
      if (i0 + r < M.m) put<SPLIT>(Y + W * M.x, M.ldx, i0 + r, j0 + c, v);   // (columns n ... ldx: zero, as X's are)
    });
  } else {
    float f = 1.f / M.scale;
    if (res.p) {
      const float r = (float)M.rows, c = (float)M.cols;
      f *= res.lr * (res.lr_scale ? 0.2f * sqrtf(fmaxf(r, c)) : sqrtf(fmaxf(1.f, r / c)));
    }
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
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) p[e] = v[e];
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
    if (M.tall) store_tile<T, true>(acc, smem, [&](int r, int c, float (&v)[8]) { emit(j0 + r, i0 + c, v); });
    else store_tile<T, false>(acc, smem, [&](int r, int c, float (&v)[8]) { emit(i0 + r, j0 + c, v); });
  }
}

// ------------------------------------------------------------------ host side
inline long long up256(long long v) { return (v + 255) / 256 * 256; }

constexpr int N_AREAS = 5;   // m x m work matrices: G, R, Z, two of Q (the f16 form uses G and Z)
struct Work {
  _Float16 *x[2], *a[N_AREAS];
  Partial* part;
  long long bytes;
};
Work carve(const DasNsPlan* p, bool split, void* ws) {
  const long long xb = up256((split ? 4 : 2) * p->x_elems), ab = up256((split ? 4 : 2) * p->a_elems);
  const int areas = split ? N_AREAS : 2;
  char* c = (char*)ws;
  Work w = {};
  auto take = [&](long long n) { char* r = c; if (c) c += n; w.bytes += n; return r; };
  for (int i = 0; i < 2; ++i) w.x[i] = (_Float16*)take(xb);
  for (int i = 0; i < areas; ++i) w.a[i] = (_Float16*)take(ab);
  w.part = (Partial*)take(up256((long long)sizeof(Partial) * p->n_chunks));
  return w;
}

bool plan_valid(const DasNsPlan* p, const void* tables, const void* ws) {
  return p && tables && ws && p->n_matrices > 0 && p->n_chunks > 0 && p->n_gram > 0 && p->n_update > 0 && p->steps > 0 &&
         p->steps <= DAS_NS_MAX_STEPS && (p->gram_tile == 64 || p->gram_tile == 128) && (p->update_tile == 64 || p->update_tile == 128) &&
         !(((uintptr_t)tables | (uintptr_t)ws) & 15);
}

struct Bounds {              // of step k over the singular values that can reach it
  double top;                // |X| before the step
  double factor;             // max |a + b s^2 + c s^4|
};
// What f16 and the phases of f32 results have to hold: X's norm, Z's norm step by step. false: outside f16's range.
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

template <bool SPLIT>
int iterate(const DasNsPlan* p, const char* tab, Work w, const Result& res, hipStream_t s) {
  const NsMatrix* mats = (const NsMatrix*)(tab + p->mat_at);
  const int4 *chunks = (const int4*)(tab + p->chunk_at), *gram = (const int4*)(tab + p->gram_at), *upd = (const int4*)(tab + p->update_at);
  auto sym = [&](auto kind, int products, const SymArgs& a) {
    constexpr SymKind K = decltype(kind)::value;
    if (p->gram_tile == 128)
      hipLaunchKernelGGL((sym_kernel<128, SPLIT, K>), dim3(p->n_gram, products), dim3(TPB), 0, s, mats, gram, a);
    else
      hipLaunchKernelGGL((sym_kernel<64, SPLIT, K>), dim3(p->n_gram, products), dim3(TPB), 0, s, mats, gram, a);
  };
  auto update = [&](auto last, const _Float16* q, const _Float16* x, _Float16* y) {
    constexpr bool L = decltype(last)::value;
    if (p->update_tile == 128)
      hipLaunchKernelGGL((update_kernel<128, SPLIT, L>), dim3(p->n_update), dim3(TPB), 0, s, mats, upd, q, x, y, res);
    else
      hipLaunchKernelGGL((update_kernel<64, SPLIT, L>), dim3(p->n_update), dim3(TPB), 0, s, mats, upd, q, x, y, res);
  };
  const std::integral_constant<SymKind, GRAM> gram_k;
  const std::integral_constant<SymKind, POLY> poly_k;
  const std::integral_constant<SymKind, PRODUCT> product_k;
  hipLaunchKernelGGL(normalise_kernel<SPLIT>, dim3(p->n_chunks), dim3(TPB), 0, s, mats, chunks, p->eps, w.x[0], w.part);
  DAS_CHECK_LAUNCH();
  Bounds bound[DAS_NS_MAX_STEPS];
  if (!polynomial_bounds(p->coef, p->steps, bound)) return DAS_ERR_ARG;
  _Float16 *X = w.x[0], *Y = w.x[1], *G = w.a[0], *R = w.a[1], *Z = w.a[SPLIT ? 2 : 1];
  for (int k = 0; k < p->steps;) {
    // steps k ... end - 1 are one phase
    int end = k + 1;
    if (SPLIT) {
      double growth = bound[k].factor * bound[k].factor;
      while (end < p->steps && growth <= 256.0) {
        growth *= bound[end].factor * bound[end].factor;
        ++end;
      }
    }
    sym(gram_k, 1, SymArgs{{X}, {X}, {G}, 0.f, 0.f, 0.f});
    _Float16 *q = nullptr, *spare = w.a[SPLIT ? 3 : 1], *other = SPLIT ? w.a[4] : nullptr;   // (q: the phase's product so far)
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

}  // namespace

extern "C" int das_ns_plan(const DasNsShape* shapes, int n, int steps, const float* coef, float eps, DasNsPlan* plan, void* tables,
                           long long table_bytes) {
  Bounds bound[DAS_NS_MAX_STEPS];
  if (!shapes || n < 1 || !coef || !plan || steps < 1 || steps > DAS_NS_MAX_STEPS || !(eps >= 0.f) || !std::isfinite(eps) ||
      !polynomial_bounds(coef, steps, bound))
    return DAS_ERR_ARG;
  memset(plan, 0, sizeof(*plan));
  auto tiles = [&](int t, bool sym) {
    long long c = 0;
    for (int g = 0; g < n; ++g) {
      const long long m = std::min(shapes[g].rows, shapes[g].cols), nn = std::max(shapes[g].rows, shapes[g].cols);
      const long long tm = (m + t - 1) / t, tn = (nn + 127) / 128 * (128 / t);
      c += shapes[g].count * (sym ? tm * (tm + 1) / 2 : tm * tn);
    }
    return c;
  };
  long long n_mat = 0, n_chunks = 0;
  double top = 1.0;
  for (int k = 0; k < steps; ++k) top = std::max(top, bound[k].top);
  std::vector<std::pair<long long, long long>> spans;
  for (int g = 0; g < n; ++g) {
    const DasNsShape& s = shapes[g];
    if (s.off < 0 || s.count < 1 || s.rows < 1 || s.cols < 1 || s.rows > (1 << 20) || s.cols > (1 << 20)) return DAS_ERR_ARG;
    const long long m = std::min(s.rows, s.cols), nn = std::max(s.rows, s.cols);
    const long long ldx = (nn + 127) / 128 * 128, lda = (m + 63) / 64 * 64;
    n_mat += s.count;
    n_chunks += s.count * (lda / 64) * (ldx / 64);
    plan->x_elems += s.count * m * ldx;
    plan->a_elems += s.count * m * lda;
    if (n_mat > (1 << 24) || n_chunks > (1 << 26) || m > (1 << 15)) return DAS_ERR_ARG;
    spans.push_back({s.off, s.off + (long long)s.count * s.rows * s.cols});
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return DAS_ERR_ARG;   // two workgroups would write the same elements
  plan->gram_tile = tiles(128, true) >= 256 ? 128 : 64;
  plan->update_tile = tiles(128, false) >= 256 ? 128 : 64;
  const long long n_gram = tiles(plan->gram_tile, true), n_upd = tiles(plan->update_tile, false);
  if (n_gram > (1 << 26) || n_upd > (1 << 26)) return DAS_ERR_ARG;
  plan->n_groups = n; plan->n_matrices = (int)n_mat; plan->n_chunks = (int)n_chunks; plan->n_gram = (int)n_gram;
  plan->n_update = (int)n_upd; plan->steps = steps; plan->eps = eps; plan->extent = spans.back().second;
  memcpy(plan->coef, coef, sizeof(float) * 3 * steps);
  plan->mat_at = 0;
  plan->chunk_at = up256(n_mat * (long long)sizeof(NsMatrix));
  plan->gram_at = plan->chunk_at + up256(16 * n_chunks);
  plan->update_at = plan->gram_at + up256(16 * n_gram);
  plan->table_bytes = plan->update_at + up256(16 * n_upd);
  if (!tables) return DAS_OK;
  if (table_bytes < plan->table_bytes) return DAS_ERR_ARG;
  memset(tables, 0, plan->table_bytes);
  char* tab = (char*)tables;
  NsMatrix* mats = (NsMatrix*)(tab + plan->mat_at);
  int4 *chunk = (int4*)(tab + plan->chunk_at), *gram = (int4*)(tab + plan->gram_at), *upd = (int4*)(tab + plan->update_at);
  long long x = 0, a = 0;
  int q = 0, c = 0;
  for (int g = 0; g < n; ++g) {
    const DasNsShape& s = shapes[g];
    for (int i = 0; i < s.count; ++i, ++q) {
      NsMatrix& M = mats[q];
      M.rows = s.rows; M.cols = s.cols; M.m = std::min(s.rows, s.cols); M.n = std::max(s.rows, s.cols);
      M.tall = s.rows > s.cols;
      M.ldx = (M.n + 127) / 128 * 128; M.lda = (M.m + 63) / 64 * 64;
      M.src = s.off + (long long)i * s.rows * s.cols;
      M.x = x; M.a = a; M.group = g; M.index = i; M.chunk0 = c;
      M.scale = (float)std::ldexp(1.0, (int)std::lround(0.5 * std::log2((double)M.n)));
      // about m, and top^2 gscale within f16
      M.gscale = (float)std::ldexp(1.0, std::min((int)std::lround(std::log2((double)M.m)), (int)std::floor(std::log2(32768.0 / (top * top)))));
      x += (long long)M.m * M.ldx; a += (long long)M.m * M.lda;
      int k = 0;
      for (int r = 0; r < (M.tall ? M.ldx : M.lda) / CHUNK; ++r)
        for (int cc = 0; cc < (M.tall ? M.lda : M.ldx) / CHUNK; ++cc) chunk[c++] = make_int4(q, r, cc, k++);
      M.chunks = k;
    }
  }
  // longest inner axis first: the last workgroups to start are the shortest ones
  std::vector<int> order(n_mat);
  for (int i = 0; i < (int)n_mat; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int u, int v) { return mats[u].n > mats[v].n; });
  auto across = [](int v, int t) { return (v + t - 1) / t; };
  int t = 0;
  for (int i : order)
    for (int r = 0; r < across(mats[i].m, plan->gram_tile); ++r)
      for (int j = 0; j <= r; ++j) gram[t++] = make_int4(i, r, j, 0);
  std::stable_sort(order.begin(), order.end(), [&](int u, int v) { return mats[u].m > mats[v].m; });
  t = 0;
  for (int i : order)
    for (int j = 0; j < mats[i].ldx / plan->update_tile; ++j)
      for (int r = 0; r < across(mats[i].m, plan->update_tile); ++r) upd[t++] = make_int4(i, r, j, 0);
  return DAS_OK;
}

extern "C" long long das_ns_ws_bytes(const DasNsPlan* p, int f32_result) {
  if (!p) return -1;
  return carve(p, f32_result != 0, nullptr).bytes;
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
  const bool split = out_dtype == DAS_F32;
  const Work w = carve(plan, split, ws);
  const NsMatrix* mats = (const NsMatrix*)(tab + plan->mat_at);
  const int4* chunks = (const int4*)(tab + plan->chunk_at);
  const MuonIn none = {};
  // one launch for every 64 source tensors (one in all but unusual sets): its workgroups of other tensors' blocks end at once
  for (int first = 0; first < n_srcs; first += Sources::MAX) {
    Sources a;
    a.first = first;
    a.count = std::min(Sources::MAX, n_srcs - first);
    for (int i = 0; i < Sources::MAX; ++i) a.s[i] = srcs[first + std::min(i, a.count - 1)];
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(plan->n_chunks), dim3(TPB), 0, s, mats, chunks, a, none, w.x[0], w.part);
    };
    if (in_dtype == DAS_F32) split ? launch(ingest_kernel<float, false, true>) : launch(ingest_kernel<float, false, false>);
    else if (in_dtype == DAS_BF16) split ? launch(ingest_kernel<bf16_t, false, true>) : launch(ingest_kernel<bf16_t, false, false>);
    else split ? launch(ingest_kernel<_Float16, false, true>) : launch(ingest_kernel<_Float16, false, false>);
    DAS_CHECK_LAUNCH();
  }
  const Result res = {out, out_dtype, nullptr, 1.f, 0.f, 0};
  return split ? iterate<true>(plan, tab, w, res, s) : iterate<false>(plan, tab, w, res, s);
}

extern "C" int das_muon_step(const DasNsPlan* plan, const void* tables_dev, float* p, const float* g, float* buf, float lr,
                             float momentum, float weight_decay, int nesterov, int lr_scale, float grad_scale, float max_norm,
                             const float* grad_sumsq, void* ws, void* stream) {
  DAS_PROF(stream);
  if (!plan_valid(plan, tables_dev, ws) || !p || !g || !buf || !(momentum >= 0.f && momentum < 1.f) || !(lr >= 0.f) ||
      !(weight_decay >= 0.f) || (max_norm > 0.f && !grad_sumsq) || lr_scale < 0 || lr_scale > 1)
    return DAS_ERR_ARG;
  if (((uintptr_t)p | (uintptr_t)g | (uintptr_t)buf) & 3) return DAS_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const char* tab = (const char*)tables_dev;
  const Work w = carve(plan, true, ws);
  const MuonIn mu = {g, buf, momentum, grad_scale, max_norm, nesterov, grad_sumsq};
  hipLaunchKernelGGL((ingest_kernel<float, true, true>), dim3(plan->n_chunks), dim3(TPB), 0, s, (const NsMatrix*)(tab + plan->mat_at),
                     (const int4*)(tab + plan->chunk_at), Sources{}, mu, w.x[0], w.part);
  DAS_CHECK_LAUNCH();
  const Result res = {nullptr, 0, p, (float)(1.0 - (double)lr * (double)weight_decay), lr, lr_scale};
  return iterate<true>(plan, tab, w, res, s);
}
