// Cross entropy of a linear head for few rows against many classes (the operator of linear_ce.hip): scoring one token, a step of a short
// batch.  gfx950, wave64.
//
//   z_iv = x_i . w_v + b_v,  loss_i = log sum_v exp z_iv - z_i,t(i),  dz_iv = g_i (exp(z_iv - lse_i) - [v = t(i)])
//   dx_i = sum_v dz_iv w_v,  dw_v = sum_i dz_iv x_i,  db_v = sum_i dz_iv
//
// Bound by the bytes of w and dw: w is read once forward and once backward, dw is written once, and nothing else is as large -- the
// logits of at most 32 rows are kept in float32 instead of being formed again, and nothing is packed or scaled.  Forward: the matrix
// instructions of 16 x 16, operands straight from memory into registers whatever their stride or alignment (float32 ones on the float32
// instruction), four waves share K.  Backward: one launch in which some workgroups read w for dx (sums over their classes, joined in
// order by another launch) and others write dw and db, each forming its classes' dz in LDS first; products on the float32 matrix
// instruction, which takes 30 us for 16 rows, 65536 classes and 1024 features, less than the bytes.
//
// 65536 x 1024 (134 MB bfloat16, 268 MB float32), in a graph: one row, forward 33 and 57 us (4.1 and 4.7 TB/s); with backward 93 and
// 186 us (three times the bytes: 4.4 TB/s); 16 rows 105 and 206 us.  The products of dx and dw on the vector units took 84 us in all for one
// row of bfloat16, but 203 us for 16.
#include <algorithm>

#include "linear_ce_direct.h"

namespace {

constexpr int kClasses = 64;           // of a workgroup, forward
constexpr int kPitch = kClasses + 4;

struct Part { float m, s; };      // other classes' largest logit, sum of exp(z - m)
__device__ __forceinline__ Part merge(Part p, Part q) {
  const float m = fmaxf(p.m, q.m);
  if (m == -INFINITY) return {m, p.s + q.s};      // nothing, or NaN
  return {m, p.s * expf(p.m - m) + q.s * expf(q.m - m)};
}

// 64 classes by 16 NB rows per workgroup: logits (kept for the backward), each row's part of the statistics, the target's logit
template <typename T, int NB>
__global__ __launch_bounds__(256) void ce_few_logits_kernel(int n, int d, int v, const T* __restrict__ x, long long ldx,
                                                            const T* __restrict__ w, long long ldw, const T* __restrict__ bias,
                                                            const void* __restrict__ target, int idx64, long long ignore,
                                                            float* __restrict__ z, long long ldz, Part* __restrict__ part,
                                                            float* __restrict__ zt) {
  __shared__ __attribute__((aligned(16))) float lds[4][16 * NB][kPitch];
  constexpr int B = kClasses / 16, U = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int v0 = blockIdx.x * kClasses, at = g * kVec<T>;
  bool on[NB];      // rows that do not count are not looked at
  const T *xr[NB], *wr[B];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int row = j * 16 + r;
    on[j] = row < n && load_index(target, row, idx64) != ignore;
    xr[j] = x + (long long)(on[j] ? row : 0) * ldx + at;
  }
#pragma unroll
  for (int i = 0; i < B; ++i) wr[i] = w + (long long)min(v0 + i * 16 + r, v - 1) * ldw + at;
  f32x4 acc[B][NB] = {};
  const int steps = d / kStep<T>;
  const u32x4 zero = {0, 0, 0, 0};
  int s = wave;
  for (; s + 4 * (U - 1) < steps; s += 4 * U) {
    u32x4 a[U][B], b[U][NB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + 4 * u) * kStep<T>;
#pragma unroll
      for (int i = 0; i < B; ++i) a[u][i] = load16(wr[i] + k);
#pragma unroll
      for (int j = 0; j < NB; ++j) b[u][j] = on[j] ? load16(xr[j] + k) : zero;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < B; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(a[u][i], b[u][j], acc[i][j]);
  }
  for (; s < steps; s += 4) {
    const int k = s * kStep<T>;
    u32x4 a[B], b[NB];
#pragma unroll
    for (int i = 0; i < B; ++i) a[i] = load16(wr[i] + k);
#pragma unroll
    for (int j = 0; j < NB; ++j) b[j] = on[j] ? load16(xr[j] + k) : zero;
#pragma unroll
    for (int i = 0; i < B; ++i)
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(a[i], b[j], acc[i][j]);
  }
  if (s == steps && steps * kStep<T> < d) {      // the wave whose turn it is
    const int k = steps * kStep<T>, left = d - k - at;
    u32x4 b[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) b[j] = on[j] ? load_raw(xr[j] + k, left) : zero;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const u32x4 a = load_raw(wr[i] + k, left);
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(a, b[j], acc[i][j]);
    }
  }
  // a lane has four consecutive classes of row lane % 16
#pragma unroll
  for (int i = 0; i < B; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j) *reinterpret_cast<f32x4*>(&lds[wave][j * 16 + r][i * 16 + g * 4]) = acc[i][j];
  __syncthreads();
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int row = j * 16 + (threadIdx.x >> 4), q = (threadIdx.x & 15) * 4, c = v0 + q;
    f32x4 y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x4 p = *reinterpret_cast<const f32x4*>(&lds[k][row][q]);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += p[e];
    }
    if (bias) {
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += to_f32(bias[min(c + e, v - 1)]);
    }
    if (z && row < n && c < ldz) *reinterpret_cast<f32x4*>(z + row * ldz + c) = y;
    const long long t = row < n ? load_index(target, row, idx64) : -1;
    Part p = {-INFINITY, 0.f};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (c + e == t && c + e < v) zt[row] = y[e];
      if (c + e != t && c + e < v) p.m = fmaxf(p.m, y[e]);
    }
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) p.m = fmaxf(p.m, __shfl_xor(p.m, o));
    const float ref = p.m == -INFINITY ? 0.f : p.m;
#pragma unroll
    for (int e = 0; e < 4; ++e) p.s += c + e != t && c + e < v ? expf(y[e] - ref) : 0.f;
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) p.s += __shfl_xor(p.s, o);
    if (row < n && q == 0) part[(long long)row * gridDim.x + blockIdx.x] = p;
  }
}

// one workgroup per row
__global__ __launch_bounds__(1024) void ce_few_rows_kernel(int v, int tiles, const Part* __restrict__ part, const float* __restrict__ zt,
                                                           const void* __restrict__ target, int idx64, long long ignore,
                                                           Row* __restrict__ stat, int* __restrict__ tgt, float* __restrict__ row_loss) {
  __shared__ float tmp[2][16];
  const int i = blockIdx.x, tid = threadIdx.x;
  const long long t = load_index(target, i, idx64);
  Part p = {-INFINITY, 0.f};
#pragma unroll 4
  for (int k = tid; k < tiles; k += 1024) p = merge(p, part[(long long)i * tiles + k]);
  const float wm = wave_max(p.m);
  if ((tid & 63) == 0) tmp[0][tid >> 6] = wm;
  __syncthreads();
  float m = tmp[0][0];
#pragma unroll
  for (int k = 1; k < 16; ++k) m = fmaxf(m, tmp[0][k]);
  const float ws = wave_sum(p.m == -INFINITY ? p.s : p.s * expf(p.m - m));      // (-inf: nothing, or NaN)
  if ((tid & 63) == 0) tmp[1][tid >> 6] = ws;
  __syncthreads();
  if (tid == 0) {
    float sum = 0.f;
    for (int k = 0; k < 16; ++k) sum += tmp[1][k];
    Row r = {kNaN, kNaN, kNaN, kNaN};
    if (t == ignore) r.loss = 0.f;
    else if (t >= 0 && t < v) r = row_of(m, sum, zt[i]);
    stat[i] = r;
    tgt[i] = t == ignore ? -2 : t >= 0 && t < v ? (int)t : -1;
    row_loss[i] = r.loss;
  }
}

__global__ __launch_bounds__(64) void ce_few_total_kernel(int n, int mean, const float* __restrict__ row_loss,
                                                          const int* __restrict__ tgt, float* __restrict__ loss) {
  const bool on = (int)threadIdx.x < n && tgt[threadIdx.x] != -2;
  const double sum = wave_sum(on ? (double)row_loss[threadIdx.x] : 0.0);
  const int rows = __popcll(__ballot(on));
  if (threadIdx.x == 0) *loss = (float)(mean ? sum / rows : sum);
}

struct FewGrads {
  int n, d, v, chunk, reduction;
  int dxs, subs;                 // workgroups that form dx, chunks of classes
  int groups, teams;             // groups of 16 x 16 bytes of columns; waves that share a group's classes
  long long ldx, ldw, ldz, lds;  // lds: of the slabs' rows
  const void *x, *w;
  const float *z, *gout;
  const Row* stat;
  const int* tgt;
  float* slab;                   // [workgroup, team][row][lds]
  void *dw, *db;
};
constexpr int kChunk = 256;      // classes whose dz a workgroup holds in LDS, at most

// Workgroups [0, dxs): slabs of dx, every dxs-th chunk of classes; [dxs, dxs + subs): dw and db of a chunk.  A wave has a group of columns:
// lane l the sixteen bytes l % 16 of it, so that the instruction for element e of them gets columns V (l % 16) + e from the lanes as they
// were loaded.  dx: K are four classes, one per sixteen lanes; dw: K are four rows, the outputs of a lane are V columns of four classes.
template <typename T, int NB>
__global__ __launch_bounds__(256, 2) void ce_few_grads_kernel(FewGrads f) {
  constexpr int V = kVec<T>, NR = 16 * NB, P = NR + 1, G = 16 / V;      // G: groups of columns whose sums of dx a wave has at a time
  __shared__ float dz[kChunk * P];      // [class][row]
  __shared__ float fac[NR], top[NR], inv[NR], att[NR];
  __shared__ int tg[NR];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const int team = wave & (f.teams - 1), step = 4 / f.teams, passes = (f.groups + step * G - 1) / (step * G);
  if (tid < NR) {
    const int t = tid < f.n ? f.tgt[tid] : -2;
    const uint64_t on = __ballot(t != -2);
    const int rows = __popcll(on);
    const Row s = tid < f.n ? f.stat[tid] : Row{0.f, 0.f, 0.f, 0.f};
    fac[tid] = f.reduction == 0 ? (tid < f.n ? f.gout[tid] : 0.f) : f.reduction == 1 ? f.gout[0] / rows : f.gout[0];
    top[tid] = s.top;
    inv[tid] = s.inv;
    att[tid] = s.at_target;
    tg[tid] = t;
  }
  __syncthreads();
  // g (p - t) of `count` classes from c0 on; zeros in rows that do not count and behind the classes, up to the next sixteen
  auto fill = [&](int c0, int count) {
    const int padded = (count + 15) & ~15;
    for (int idx = tid; idx < padded * NR; idx += 256) {
      const int i = idx / padded, c = idx - i * padded;
      float y = 0.f;
      if (i < f.n && c < count && tg[i] != -2)
        y = fac[i] * (tg[i] == c0 + c ? att[i] : inv[i] * expf(f.z[i * f.ldz + c0 + c] - top[i]));
      dz[c * P + i] = y;
    }
    __syncthreads();
  };
  if ((int)blockIdx.x < f.dxs) {
    const T* w = (const T*)f.w;
    for (int pass = 0; pass < passes; ++pass) {
      const int first = (pass * step + wave / f.teams) * G, col = (first * 16 + r) * V;
      const int mine = min(G, f.groups - first);      // groups of this wave, none at all if negative
      f32x4 acc[G][V][NB] = {};
      auto add = [&](int q, int c, const u32x4& raw) {
        float y[V], a[NB];
        unpack<T>(raw, y);
#pragma unroll
        for (int j = 0; j < NB; ++j) a[j] = dz[(c + g) * P + j * 16 + r];
#pragma unroll
        for (int e = 0; e < V; ++e)
#pragma unroll
          for (int j = 0; j < NB; ++j) acc[q][e][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], y[e], acc[q][e][j], 0, 0, 0);
      };
      for (int sub = blockIdx.x; sub < f.subs; sub += f.dxs) {
        const int c0 = sub * f.chunk, count = min(f.chunk, f.v - c0);
        fill(c0, count);
        // (the matrix instructions need whole waves: only what is loaded depends on the lane)
        const T* at = w + col;
        const int last = f.v - 1, by = 4 * f.teams;
        int c = team * 4;
        if (mine > 0 && (f.d % V == 0 || (first + G) * 16 * V <= f.d)) {
          constexpr int U = 8 / G;
          long long to[G];      // (lanes behind the last column read others, for sums that are not stored)
#pragma unroll
          for (int q = 0; q < G; ++q) to[q] = col + q * 16 * V < f.d ? q * 16 * V : -(long long)col;
          for (; c + (U - 1) * by < count; c += U * by) {
            u32x4 raw[U][G];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int q = 0; q < G; ++q) raw[u][q] = load16(at + min(c0 + c + u * by + g, last) * f.ldw + to[q]);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
              for (int q = 0; q < G; ++q) add(q, c + u * by, raw[u][q]);
          }
        }
        for (; mine > 0 && c < count; c += by) {
#pragma unroll
          for (int q = 0; q < G; ++q)
            if (q < mine) add(q, c, load_raw(at + min(c0 + c + g, last) * f.ldw + q * 16 * V, f.d - col - q * 16 * V));
        }
        __syncthreads();
      }
#pragma unroll
      for (int q = 0; q < G; ++q)
#pragma unroll
        for (int j = 0; j < NB; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = j * 16 + g * 4 + k, at = col + q * 16 * V;
            float* out = f.slab + ((long long)(blockIdx.x * f.teams + team) * f.n + row) * f.lds + at;
            if (row < f.n) {
#pragma unroll
              for (int e = 0; e < V; e += 4)
                if (at + e < f.lds)
                  *reinterpret_cast<f32x4*>(out + e) =
                      f32x4{acc[q][e][j][k], acc[q][e + 1][j][k], acc[q][e + 2][j][k], acc[q][e + 3][j][k]};
            }
          }
    }
  } else {
    const int c0 = (int)(blockIdx.x - f.dxs) * f.chunk, count = min(f.chunk, f.v - c0);
    fill(c0, count);
    if (f.db && tid < count) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < NR; ++i) sum += dz[tid * P + i];
      ((T*)f.db)[c0 + tid] = from_f32<T>(sum);
    }
    if (!f.dw) return;
    const T* x = (const T*)f.x;
    for (int group = wave / f.teams; group < f.groups; group += step) {
      const int col = (group * 16 + r) * V, left = f.d - col;
      float xr[NB * 4][V];
#pragma unroll
      for (int i = 0; i < NB * 4; ++i) {
        if (tg[i * 4 + g] != -2) {
          load_part(x + (i * 4 + g) * f.ldx + col, left, xr[i]);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) xr[i][e] = 0.f;
        }
      }
      for (int c = team * 16; c < count; c += 16 * f.teams) {
        f32x4 acc[V] = {};
#pragma unroll
        for (int i = 0; i < NB * 4; ++i) {
          const float a = dz[(c + r) * P + i * 4 + g];
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, xr[i][e], acc[e], 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int cls = c + g * 4 + k;
          float y[V];
#pragma unroll
          for (int e = 0; e < V; ++e) y[e] = acc[e][k];
          if (cls < count) store_part((T*)f.dw + (long long)(c0 + cls) * f.d + col, left, y);
        }
      }
    }
  }
}

// dx: the slabs in order, 64 columns of a row per workgroup, sixteen parts of the slabs side by side
template <typename T>
__global__ __launch_bounds__(256) void ce_few_join_kernel(int n, int d, int slabs, const float* __restrict__ slab, long long ld,
                                                          const int* __restrict__ tgt, T* __restrict__ dx) {
  __shared__ f32x4 tmp[16][16];
  const int per = (d + 63) / 64, i = blockIdx.x / per, c = (int)(blockIdx.x % per) * 64 + (threadIdx.x & 15) * 4, part = threadIdx.x >> 4;
  const int each = (slabs + 15) / 16;
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (c < d) {
#pragma unroll 8
    for (int s = part * each; s < min(slabs, (part + 1) * each); ++s) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(slab + ((long long)s * n + i) * ld + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] += y[e];
    }
  }
  tmp[part][threadIdx.x & 15] = x;
  __syncthreads();
  if (part || c >= d) return;
  for (int k = 1; k < 16; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += tmp[k][threadIdx.x][e];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < d) dx[(long long)i * d + c + e] = from_f32<T>(tgt[i] == -2 ? 0.f : x[e]);
}

struct FewKeep { long long ldz, z, stat, tgt, loss, bytes; };
inline FewKeep few_keep(long long n, int v, int train) {
  FewKeep k;
  k.ldz = round_up(v, 4);
  k.z = 0;
  k.stat = train ? round_up(4 * n * k.ldz, 256) : 0;
  k.tgt = k.stat + 16 * kFewRowsCe;
  k.loss = k.tgt + 4 * kFewRowsCe;
  k.bytes = k.loss + 4 * kFewRowsCe;
  return k;
}
struct FewPlan { int groups, teams, chunk, subs, dxs; };
inline FewPlan few_plan(long long n, int d, int v, int dtype) {
  FewPlan p;
  const int columns = dtype == ISTNET_VOCAB_F32 ? 64 : 128;
  p.groups = (d + columns - 1) / columns;
  p.teams = p.groups == 1 ? 4 : p.groups == 2 ? 2 : 1;
  p.chunk = (int)std::min<long long>(kChunk, round_up((v + 511) / 512, 16));      // some 512 workgroups
  p.subs = (v + p.chunk - 1) / p.chunk;
  // slabs that are small beside w: 64 MB, or 32 of them where there are that many features
  const long long most = std::max<long long>(32, (64ll << 20) / (4 * n * d * p.teams));
  p.dxs = (int)std::min<long long>({p.subs, (n <= 16 ? 512 : 256) / p.teams, most});
  return p;
}
#define FEW_BLOCKS(n, NB, ...)                                           \
  do {                                                                   \
    if ((n) <= 16) { constexpr int NB = 1; __VA_ARGS__; }                \
    else { constexpr int NB = 2; __VA_ARGS__; }                          \
  } while (0)

}  // namespace

long long vocab_few_ce_keep(long long n, int v, int train) { return few_keep(n, v, train).bytes; }

long long vocab_few_ce_scratch(long long n, int d, int v, int dtype, int backward) {
  const long long tiles = (v + kClasses - 1) / kClasses;
  const FewPlan p = few_plan(n, d, v, dtype);
  return backward ? 4ll * p.dxs * p.teams * n * round_up(d, 4) : 8 * n * tiles + 4 * kFewRowsCe;
}

int vocab_few_ce_forward(int n, int d, int v, int dtype, int idx64, int train, const void* x, long long ldx, const void* w,
                         long long ldw, const void* bias, const void* target, long long ignore, int reduction, float* loss, void* keep,
                         void* ws, hipStream_t st) {
  const FewKeep k = few_keep(n, v, train);
  const int tiles = (v + kClasses - 1) / kClasses;
  char* kb = (char*)keep;
  float *z = train ? (float*)(kb + k.z) : nullptr, *row_loss = reduction == 0 ? loss : (float*)(kb + k.loss);
  Part* part = (Part*)ws;
  float* zt = (float*)((char*)ws + 8ll * n * tiles);
  int* tgt = (int*)(kb + k.tgt);
  VOCAB_DISPATCH(dtype, T, FEW_BLOCKS(n, NB, hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_few_logits_kernel<T, NB>), dim3(tiles), dim3(256), 0,
                                                                st, n, d, v, (const T*)x, ldx, (const T*)w, ldw, (const T*)bias, target,
                                                                idx64, ignore, z, k.ldz, part, zt)));
  hipLaunchKernelGGL(ce_few_rows_kernel, dim3(n), dim3(1024), 0, st, v, tiles, part, zt, target, idx64, ignore, (Row*)(kb + k.stat), tgt,
                     row_loss);
  if (reduction != 0) hipLaunchKernelGGL(ce_few_total_kernel, dim3(1), dim3(64), 0, st, n, reduction == 1, row_loss, tgt, loss);
  return launch_status();
}

int vocab_few_ce_backward(int n, int d, int v, int dtype, const void* x, long long ldx, const void* w, long long ldw, int reduction,
                          const float* gout, const void* keep, void* ws, void* dx, void* dw, void* db, hipStream_t st) {
  const FewKeep k = few_keep(n, v, 1);
  const FewPlan p = few_plan(n, d, v, dtype);
  const char* kb = (const char*)keep;
  FewGrads f = {};
  f.n = n;
  f.d = d;
  f.v = v;
  f.chunk = p.chunk;
  f.groups = p.groups;
  f.teams = p.teams;
  f.reduction = reduction;
  f.dxs = dx ? p.dxs : 0;
  f.subs = p.subs;
  f.ldx = ldx;
  f.ldw = ldw;
  f.ldz = k.ldz;
  f.lds = round_up(d, 4);
  f.x = x;
  f.w = w;
  f.z = (const float*)(kb + k.z);
  f.gout = gout;
  f.stat = (const Row*)(kb + k.stat);
  f.tgt = (const int*)(kb + k.tgt);
  f.slab = (float*)ws;
  f.dw = dw;
  f.db = db;
  const int wgs = f.dxs + (dw || db ? p.subs : 0);
  VOCAB_DISPATCH(dtype, T, {
    FEW_BLOCKS(n, NB, hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_few_grads_kernel<T, NB>), dim3(wgs), dim3(256), 0, st, f));
    if (dx)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_few_join_kernel<T>), dim3(n * ((d + 63) / 64)), dim3(256), 0, st, n, d,
                         p.dxs * p.teams, f.slab, f.lds, f.tgt, (T*)dx);
  });
  return launch_status();
}
