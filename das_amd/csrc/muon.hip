// Newton-Schulz orthogonalisation of a ragged set of matrices, and the Muon step around it (include/das_hip.h).
//
// For U (rows x cols; m = min, n = max; transposed if rows > cols, so X is m x n):  X = U / (|U|_F + eps), then `steps` times
//   A = X X^T (m x m, symmetric)      gram_kernel<false>
//   B = a I + b A + c A A             gram_kernel<true>   (A A = A A^T: the same product of rows by rows; B is symmetric too)
//   X = B X                           update_kernel       (the last one writes the result / the parameter)
// In singular values this is s -> s (a + b s^2 + c s^4). All matrices of a set go through the same launches: a table (built once on
// the host, das_ns_plan) lists every tile of every matrix, one workgroup per tile.
//
// Storage. X, A and B are f16 (11 bits; bf16's 8 would make the error 8 times larger at the same matrix-pipe rate), products sum in
// f32. X is kept times S = 2^round(log2 sqrt(n)): an orthogonal X has entries of 1 / sqrt(n), so S X is around one and
// its small entries stay normal numbers. A has entries up to 1.5, B up to a few units. Row lengths are padded to multiples of 64 with
// zeros (ldx, lda), which is the inner-loop step of every product: no tile has a tail along its inner axis.
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
constexpr int TILE = 64;    // side of an output tile

struct NsMatrix {           // one matrix, as the kernels see it
  long long src;            // element offset in the flat buffers / in the result
  long long x, a;           // element offsets in the work areas X (m x ldx) and A, B (m x lda)
  int rows, cols, m, n, ldx, lda;
  int group, index;         // source tensor and matrix in it (das_orthogonalize)
  int chunk0, chunks;       // its blocks in the partial-sum table
  float scale;              // S
  int tall;                 // rows > cols: X holds the transpose
};
struct Partial {            // of one 64 x 64 block: sum of squares of (u 2^-e), and e
  float ss;
  int e;
};

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

// One 64 x 64 block of U: update the momentum (Muon), find the block's exponent e (largest entry in [0.5, 1) 2^e) and sum of squares,
// store u 2^-e as f16 in X's layout (transposed through LDS for tall matrices), zeros in the padding. The exponent keeps gradients of any
// magnitude inside f16's range until the norm is known; normalise_kernel rounds a second time, both roundings 2^-11.
template <typename T, bool MUON>
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
  if (big > 0.f && big <= 3.4028235e38f) (void)frexpf(big, &e);
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
    f16x4_t h;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = (_Float16)u[k][j];
    *reinterpret_cast<f16x4_t*>(X + M.x + (long long)r * M.ldx + x_c0 + c4) = h;
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
    f16x4_t* p = reinterpret_cast<f16x4_t*>(X + M.x + (long long)r * M.ldx + x_c0 + c4);
    f16x4_t h = *p;
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = (_Float16)((float)h[j] * f);
    *p = h;
  }
}

// ------------------------------------------------------------------ products
// 64 x 64 tile, four waves of 32 x 32, inner step 64. v_mfma_f32_16x16x32_f16: lane l gives row l % 16 of A (column of B), inner
// elements (l / 16) * 8 ... + 8; it gets column l % 16, rows (l / 16) * 4 ... + 4 of the result.
constexpr int PITCH = TILE + 8;   // f16 elements per LDS row

__device__ __forceinline__ void stage_rows(const _Float16* src, int ld, int row0, int rows, int k0, _Float16* dst) {
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int v = threadIdx.x + it * TPB, r = v >> 3, c = (v & 7) * 8;
    const int gr = min(row0 + r, rows - 1);   // (rows past the end are stand-ins whose results are dropped)
    *reinterpret_cast<uint4*>(dst + r * PITCH + c) = *reinterpret_cast<const uint4*>(src + (long long)gr * ld + k0 + c);
  }
}

__device__ __forceinline__ void mma_step(const _Float16* a, const _Float16* b, f32x4_t (&acc)[2][2]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wr = (wave >> 1) * 32, wc = (wave & 1) * 32;
#pragma unroll
  for (int kk = 0; kk < TILE; kk += 32) {
    f16x8_t fa[2], fb[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      fa[t] = *reinterpret_cast<const f16x8_t*>(a + (wr + t * 16 + (lane & 15)) * PITCH + kk + (lane >> 4) * 8);
      fb[t] = *reinterpret_cast<const f16x8_t*>(b + (wc + t * 16 + (lane & 15)) * PITCH + kk + (lane >> 4) * 8);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(fa[i], fb[j], acc[i][j], 0, 0, 0);
  }
}

// POLY false: A = X X^T / S^2.  POLY true: B = a I + b A + c A A^T.  Tiles on and below the diagonal; each is stored twice, as it is and
// transposed, so that the result is exactly symmetric. Columns m ... lda are stored as zeros (inner axis of the next product).
template <bool POLY>
__global__ __launch_bounds__(TPB) void gram_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ tiles,
                                                   const _Float16* __restrict__ in, _Float16* __restrict__ out, float ca, float cb,
                                                   float cc) {
  __shared__ __align__(16) _Float16 sa[TILE * PITCH], sb[TILE * PITCH];
  const int4 t = tiles[blockIdx.x];
  const NsMatrix M = mats[t.x];
  const _Float16* src = in + (POLY ? M.a : M.x);
  const int ld = POLY ? M.lda : M.ldx;
  const int i0 = t.y * TILE, j0 = t.z * TILE;
  f32x4_t acc[2][2] = {};
  for (int k = 0; k < ld; k += TILE) {
    __syncthreads();
    stage_rows(src, ld, i0, M.m, k, sa);
    stage_rows(src, ld, j0, M.m, k, sb);
    __syncthreads();
    mma_step(sa, sb, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const float inv = 1.f / (M.scale * M.scale);
  _Float16* dst = out + M.a;
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + (wave >> 1) * 32 + p * 16 + (lane >> 4) * 4 + e, j = j0 + (wave & 1) * 32 + q * 16 + (lane & 15);
        float v = acc[p][q][e];
        if (i < M.m && j < M.m) {
          if constexpr (POLY)
            v = cc * v + cb * (float)src[(long long)i * ld + j] + (i == j ? ca : 0.f);
          else
            v *= inv;
        } else {
          v = 0.f;
        }
        if (j0 == i0 && j > i) continue;   // (the diagonal tile's upper half comes from its lower one)
        if (i < M.m && j < M.lda) dst[(long long)i * M.lda + j] = (_Float16)v;
        if (j < M.m && i < M.lda && i != j) dst[(long long)j * M.lda + i] = (_Float16)v;
      }
}

struct Result {             // where the last product goes
  void* out;                // das_orthogonalize
  int out_dtype;
  float* p;                 // das_muon_step: p = keep p - lr f X
  float keep, lr;
  int lr_scale;
};

// X' = B X: B's rows by X's columns. LAST: the result leaves the work area (and its scale S), transposed back where needed.
template <bool LAST>
__global__ __launch_bounds__(TPB) void update_kernel(const NsMatrix* __restrict__ mats, const int4* __restrict__ tiles,
                                                     const _Float16* __restrict__ Bm, const _Float16* __restrict__ X,
                                                     _Float16* __restrict__ Y, Result res) {
  __shared__ __align__(16) _Float16 sa[TILE * PITCH], sb[TILE * PITCH];
  const int4 t = tiles[blockIdx.x];
  const NsMatrix M = mats[t.x];
  const int i0 = t.y * TILE, j0 = t.z * TILE;
  f32x4_t acc[2][2] = {};
  for (int k = 0; k < M.lda; k += TILE) {
    __syncthreads();
    stage_rows(Bm + M.a, M.lda, i0, M.m, k, sa);
#pragma unroll
    for (int it = 0; it < 2; ++it) {   // 64 rows (inner axis) x 64 columns of X, transposed into LDS
      const int v = threadIdx.x + it * TPB, r = v >> 3, c = (v & 7) * 8;
      f16x8_t x = {};
      if (k + r < M.m) x = *reinterpret_cast<const f16x8_t*>(X + M.x + (long long)(k + r) * M.ldx + j0 + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) sb[(c + e) * PITCH + r] = x[e];
    }
    __syncthreads();
    mma_step(sa, sb, acc);
  }
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  float f = 1.f / M.scale;
  if (LAST && res.p) {
    const float r = (float)M.rows, c = (float)M.cols;
    f *= res.lr * (res.lr_scale ? 0.2f * sqrtf(fmaxf(r, c)) : sqrtf(fmaxf(1.f, r / c)));
  }
#pragma unroll
  for (int p = 0; p < 2; ++p)
#pragma unroll
    for (int q = 0; q < 2; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + (wave >> 1) * 32 + p * 16 + (lane >> 4) * 4 + e, j = j0 + (wave & 1) * 32 + q * 16 + (lane & 15);
        const float v = acc[p][q][e];
        if constexpr (!LAST) {
          if (i < M.m) Y[M.x + (long long)i * M.ldx + j] = (_Float16)v;   // (j < ldx; zero from n on, as X is)
        } else if (i < M.m && j < M.n) {
          const long long o = M.src + (M.tall ? (long long)j * M.cols + i : (long long)i * M.cols + j);
          if (res.p)
            res.p[o] = res.keep * res.p[o] - f * v;
          else if (res.out_dtype == DAS_BF16)
            reinterpret_cast<bf16_t*>(res.out)[o] = f32_to_bf16(f * v);
          else
            reinterpret_cast<_Float16*>(res.out)[o] = (_Float16)(f * v);
        }
      }
}

// ------------------------------------------------------------------ host side
struct Work {
  _Float16 *x0, *x1, *a, *b;
  Partial* part;
};
inline long long up256(long long v) { return (v + 255) / 256 * 256; }
Work carve(const DasNsPlan* p, void* ws) {
  char* w = (char*)ws;
  const long long xb = up256(2 * p->x_elems), ab = up256(2 * p->a_elems);
  return Work{(_Float16*)w, (_Float16*)(w + xb), (_Float16*)(w + 2 * xb), (_Float16*)(w + 2 * xb + ab), (Partial*)(w + 2 * xb + 2 * ab)};
}

bool plan_valid(const DasNsPlan* p, const void* tables, const void* ws) {
  return p && tables && ws && p->n_matrices > 0 && p->n_chunks > 0 && p->n_gram > 0 && p->n_update > 0 && p->steps > 0 &&
         p->steps <= DAS_NS_MAX_STEPS && !(((uintptr_t)tables | (uintptr_t)ws) & 15);
}

int iterate(const DasNsPlan* p, const char* tab, Work w, const Result& res, hipStream_t s) {
  const NsMatrix* mats = (const NsMatrix*)(tab + p->mat_at);
  const int4 *chunks = (const int4*)(tab + p->chunk_at), *gram = (const int4*)(tab + p->gram_at), *upd = (const int4*)(tab + p->update_at);
  hipLaunchKernelGGL(normalise_kernel, dim3(p->n_chunks), dim3(TPB), 0, s, mats, chunks, p->eps, w.x0, w.part);
  DAS_CHECK_LAUNCH();
  for (int k = 0; k < p->steps; ++k) {
    const float *c = p->coef + 3 * k;
    hipLaunchKernelGGL(gram_kernel<false>, dim3(p->n_gram), dim3(TPB), 0, s, mats, gram, w.x0, w.a, 0.f, 0.f, 0.f);
    hipLaunchKernelGGL(gram_kernel<true>, dim3(p->n_gram), dim3(TPB), 0, s, mats, gram, w.a, w.b, c[0], c[1], c[2]);
    if (k + 1 < p->steps)
      hipLaunchKernelGGL(update_kernel<false>, dim3(p->n_update), dim3(TPB), 0, s, mats, upd, w.b, w.x0, w.x1, res);
    else
      hipLaunchKernelGGL(update_kernel<true>, dim3(p->n_update), dim3(TPB), 0, s, mats, upd, w.b, w.x0, w.x1, res);
    DAS_CHECK_LAUNCH();
    std::swap(w.x0, w.x1);
  }
  return DAS_OK;
}

// largest |p_k(...p_1(s))| over s in [0, 1], step by step on a grid: X's spectral norm, what f16 has to hold
bool polynomial_bounded(const float* coef, int steps) {
  double hi = 1.0;
  for (int k = 0; k < steps; ++k) {
    const double a = coef[3 * k], b = coef[3 * k + 1], c = coef[3 * k + 2];
    if (!std::isfinite(a) || !std::isfinite(b) || !std::isfinite(c)) return false;
    double next = 0.0;
    for (int i = 0; i <= 4096; ++i) {
      const double x = hi * i / 4096, y = x * x;
      next = std::max(next, std::fabs(x * (a + b * y + c * y * y)));
    }
    hi = next;
    if (!(hi <= 16.0) || std::fabs(a) + std::fabs(b) * hi * hi + std::fabs(c) * hi * hi * hi * hi > 30000.0) return false;
  }
  return true;
}

}  // namespace

extern "C" int das_ns_plan(const DasNsShape* shapes, int n, int steps, const float* coef, float eps, DasNsPlan* plan, void* tables,
                           long long table_bytes) {
  if (!shapes || n < 1 || !coef || !plan || steps < 1 || steps > DAS_NS_MAX_STEPS || !(eps >= 0.f) || !std::isfinite(eps) ||
      !polynomial_bounded(coef, steps))
    return DAS_ERR_ARG;
  memset(plan, 0, sizeof(*plan));
  long long n_mat = 0, n_chunks = 0, n_gram = 0, n_upd = 0;
  std::vector<std::pair<long long, long long>> spans;
  for (int g = 0; g < n; ++g) {
    const DasNsShape& s = shapes[g];
    if (s.off < 0 || s.count < 1 || s.rows < 1 || s.cols < 1 || s.rows > (1 << 20) || s.cols > (1 << 20)) return DAS_ERR_ARG;
    const long long m = std::min(s.rows, s.cols), nn = std::max(s.rows, s.cols);
    const long long tm = (m + TILE - 1) / TILE, tn = (nn + TILE - 1) / TILE;
    n_mat += s.count;
    n_chunks += s.count * tm * tn;
    n_gram += s.count * (tm * (tm + 1) / 2);
    n_upd += s.count * tm * tn;
    if (n_mat > (1 << 24) || n_chunks > (1 << 26) || n_gram > (1 << 26) || n_upd > (1 << 26)) return DAS_ERR_ARG;
    spans.push_back({s.off, s.off + (long long)s.count * s.rows * s.cols});
  }
  std::sort(spans.begin(), spans.end());
  for (size_t i = 1; i < spans.size(); ++i)
    if (spans[i].first < spans[i - 1].second) return DAS_ERR_ARG;   // two workgroups would write the same elements
  plan->n_groups = n; plan->n_matrices = (int)n_mat; plan->n_chunks = (int)n_chunks; plan->n_gram = (int)n_gram;
  plan->n_update = (int)n_upd; plan->steps = steps; plan->eps = eps; plan->extent = spans.back().second;
  memcpy(plan->coef, coef, sizeof(float) * 3 * steps);
  plan->mat_at = 0;
  plan->chunk_at = up256(n_mat * (long long)sizeof(NsMatrix));
  plan->gram_at = plan->chunk_at + up256(16 * n_chunks);
  plan->update_at = plan->gram_at + up256(16 * n_gram);
  plan->table_bytes = plan->update_at + up256(16 * n_upd);
  for (int g = 0; g < n; ++g) {
    const long long m = std::min(shapes[g].rows, shapes[g].cols), nn = std::max(shapes[g].rows, shapes[g].cols);
    plan->x_elems += shapes[g].count * m * ((nn + 63) / 64 * 64);
    plan->a_elems += shapes[g].count * m * ((m + 63) / 64 * 64);
  }
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
      M.ldx = (M.n + 63) / 64 * 64; M.lda = (M.m + 63) / 64 * 64;
      M.src = s.off + (long long)i * s.rows * s.cols;
      M.x = x; M.a = a; M.group = g; M.index = i; M.chunk0 = c;
      M.scale = (float)std::ldexp(1.0, (int)std::lround(0.5 * std::log2((double)M.n)));
      x += (long long)M.m * M.ldx; a += (long long)M.m * M.lda;
      int k = 0;
      for (int r = 0; r < (M.rows + CHUNK - 1) / CHUNK; ++r)
        for (int cc = 0; cc < (M.cols + CHUNK - 1) / CHUNK; ++cc) chunk[c++] = make_int4(q, r, cc, k++);
      M.chunks = k;
    }
  }
  // longest inner axis first: the last workgroups to start are the shortest ones
  std::vector<int> order(n_mat);
  for (int i = 0; i < (int)n_mat; ++i) order[i] = i;
  std::stable_sort(order.begin(), order.end(), [&](int u, int v) { return mats[u].n > mats[v].n; });
  int t = 0;
  for (int i : order)
    for (int r = 0; r < mats[i].lda / TILE; ++r)
      for (int j = 0; j <= r; ++j) gram[t++] = make_int4(i, r, j, 0);
  std::stable_sort(order.begin(), order.end(), [&](int u, int v) { return mats[u].m > mats[v].m; });
  t = 0;
  for (int i : order)
    for (int j = 0; j < mats[i].ldx / TILE; ++j)
      for (int r = 0; r < mats[i].lda / TILE; ++r) upd[t++] = make_int4(i, r, j, 0);
  return DAS_OK;
}

extern "C" long long das_ns_ws_bytes(const DasNsPlan* p) {
  if (!p) return -1;
  return 2 * up256(2 * p->x_elems) + 2 * up256(2 * p->a_elems) + up256((long long)sizeof(Partial) * p->n_chunks);
}

extern "C" int das_orthogonalize(const DasNsPlan* plan, const void* tables_dev, const DasNsSource* srcs, int n_srcs, int in_dtype,
                                 void* out, int out_dtype, void* ws, void* stream) {
  DAS_PROF(stream);
  if (!plan_valid(plan, tables_dev, ws) || !srcs || n_srcs != plan->n_groups || !out || (out_dtype != DAS_BF16 && out_dtype != DAS_F16) ||
      in_dtype < DAS_F32 || in_dtype > DAS_F16)
    return DAS_ERR_ARG;
  for (int i = 0; i < n_srcs; ++i)
    if (!srcs[i].base) return DAS_ERR_ARG;
  hipStream_t s = (hipStream_t)stream;
  const char* tab = (const char*)tables_dev;
  const Work w = carve(plan, ws);
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
      hipLaunchKernelGGL(kernel, dim3(plan->n_chunks), dim3(TPB), 0, s, mats, chunks, a, none, w.x0, w.part);
    };
    if (in_dtype == DAS_F32) launch(ingest_kernel<float, false>);
    else if (in_dtype == DAS_BF16) launch(ingest_kernel<bf16_t, false>);
    else launch(ingest_kernel<_Float16, false>);
    DAS_CHECK_LAUNCH();
  }
  const Result res = {out, out_dtype, nullptr, 1.f, 0.f, 0};
  return iterate(plan, tab, w, res, s);
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
  const Work w = carve(plan, ws);
  const MuonIn mu = {g, buf, momentum, grad_scale, max_norm, nesterov, grad_sumsq};
  hipLaunchKernelGGL((ingest_kernel<float, true>), dim3(plan->n_chunks), dim3(TPB), 0, s, (const NsMatrix*)(tab + plan->mat_at),
                     (const int4*)(tab + plan->chunk_at), Sources{}, mu, w.x0, w.part);
  DAS_CHECK_LAUNCH();
  const Result res = {nullptr, 0, p, (float)(1.0 - (double)lr * (double)weight_decay), lr, lr_scale};
  return iterate(plan, tab, w, res, s);
}
