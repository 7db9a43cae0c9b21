// Cross entropy of a linear head for many rows against few classes (the operator of linear_ce.hip): a category or a bin for each of many
// points.  gfx950, wave64.
//
//   z_iv = x_i . w_v + b_v,  loss_i = log sum_v exp z_iv - z_i,t(i),  dz_iv = g_i (exp(z_iv - lse_i) - [v = t(i)])
//   dx_i = sum_v dz_iv w_v,  dw_v = sum_i dz_iv x_i,  db_v = sum_i dz_iv
//
// Bound by the bytes of x and dx: x is read once forward and once backward, dx is written once; w fits the caches.  A wave has all
// classes of its rows, so that one launch gives logits, statistics, losses and p - t (kept in float32, V numbers a row); nothing is
// packed, and rows that do not count are skipped where they lie.  Backward: one launch in which some workgroups form dx and others sums of
// dw and db over their rows, which another launch joins in order.  Products of p - t run on the float32 matrix instruction.
//
// 32768 x 128 float32, 30% of the rows without a class, 64 classes: 20 us forward, 22 us backward and 9 us for the two launches that join
// (17 MB of x, 8 MB of p - t, 17 MB of dx: 2 TB/s; a few waits for memory in a row, with two to four workgroups on a compute unit).
// 300000 x 64, 10 classes: 28 and 40 us, 2.8 and 4.5 TB/s.
#include <algorithm>

#include "linear_ce_direct.h"

namespace {

constexpr int kTileRows = 128;      // rows of p - t in LDS, backward
constexpr int row_blocks(int vb) { return vb == 4 ? 1 : 2; }      // of 16 rows, for a wave, forward

// 64 NB rows per workgroup, 16 NB per wave; VB: blocks of 16 classes
template <typename T, int VB>
__global__ __launch_bounds__(256) void ce_classes_rows_kernel(int n, int d, int v, const T* __restrict__ x, long long ldx,
                                                              const T* __restrict__ w, long long ldw, const T* __restrict__ bias,
                                                              const void* __restrict__ target, int idx64, long long ignore,
                                                              float* __restrict__ dz, long long ldz, int* __restrict__ on_row,
                                                              float* __restrict__ row_loss, double2* __restrict__ part) {
  __shared__ double2 sums[4];
  constexpr int NB = row_blocks(VB), U = 4;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), r = lane & 15, g = lane >> 4;
  const int row0 = (blockIdx.x * 4 + wave) * 16 * NB + r, at = g * kVec<T>;
  bool on[NB];
  long long t[NB];
  const T *xr[NB], *wr[VB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int row = row0 + j * 16;
    t[j] = row < n ? load_index(target, row, idx64) : ignore;
    on[j] = row < n && t[j] != ignore;      // other rows are not looked at
    xr[j] = x + (long long)(on[j] ? row : 0) * ldx + at;
  }
#pragma unroll
  for (int i = 0; i < VB; ++i) wr[i] = w + (long long)min(i * 16 + r, v - 1) * ldw + at;
  f32x4 acc[VB][NB] = {}, shift[VB] = {};      // shift: the bias of the lane's classes, 16 i + 4 g + 0..3
  if (bias) {
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) shift[i][e] = to_f32(bias[min(i * 16 + g * 4 + e, v - 1)]);
  }
  const int steps = d / kStep<T>;
  const u32x4 zero = {0, 0, 0, 0};
  int s = 0;
  for (; s + U <= steps; s += U) {
    u32x4 a[U][VB], b[U][NB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (s + u) * kStep<T>;
#pragma unroll
      for (int j = 0; j < NB; ++j) b[u][j] = on[j] ? load16(xr[j] + k) : zero;
#pragma unroll
      for (int i = 0; i < VB; ++i) a[u][i] = load16(wr[i] + k);
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < VB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(a[u][i], b[u][j], acc[i][j]);
  }
  for (; s * kStep<T> < d; ++s) {
    const int k = s * kStep<T>, left = d - k - at;
    u32x4 b[NB];
#pragma unroll
    for (int j = 0; j < NB; ++j) b[j] = on[j] ? load_raw(xr[j] + k, left) : zero;
#pragma unroll
    for (int i = 0; i < VB; ++i) {
      const u32x4 a = load_raw(wr[i] + k, left);
#pragma unroll
      for (int j = 0; j < NB; ++j) acc[i][j] = multiply<T>(a, b[j], acc[i][j]);
    }
  }
  // a lane has classes 16 i + 4 g + 0..3 of row lane % 16 of each block of rows
  double sum = 0.0, rows = 0.0;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int row = row0 + j * 16;
    float m = -INFINITY, zt = 0.f;
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = i * 16 + g * 4 + e;
        acc[i][j][e] += shift[i][e];
        if (c == t[j]) zt += acc[i][j][e];
        else if (c < v) m = fmaxf(m, acc[i][j][e]);
      }
    m = fmaxf(m, __shfl_xor(m, 16));
    m = fmaxf(m, __shfl_xor(m, 32));
    zt += __shfl_xor(zt, 16);      // one lane has it, the others zero
    zt += __shfl_xor(zt, 32);
    const float ref = m == -INFINITY ? 0.f : m;
    float others = 0.f;
#pragma unroll
    for (int i = 0; i < VB; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int c = i * 16 + g * 4 + e;
        others += c != t[j] && c < v ? expf(acc[i][j][e] - ref) : 0.f;
      }
    others += __shfl_xor(others, 16);
    others += __shfl_xor(others, 32);
    Row q = {kNaN, kNaN, kNaN, kNaN};
    if (t[j] >= 0 && t[j] < v) q = row_of(m, others, zt);
    if (!on[j]) q.loss = 0.f;
    if (dz && row < n) {
#pragma unroll
      for (int i = 0; i < VB; ++i) {
        const int c0 = i * 16 + g * 4;
        f32x4 y;
#pragma unroll
        for (int e = 0; e < 4; ++e)
          y[e] = !on[j] || c0 + e >= v ? 0.f : c0 + e == t[j] ? q.at_target : q.inv * expf(acc[i][j][e] - q.top);
        if (c0 < ldz) *reinterpret_cast<f32x4*>(dz + row * ldz + c0) = y;
      }
    }
    if (g == 0 && row < n) {
      if (on_row) on_row[row] = on[j];
      if (row_loss) row_loss[row] = q.loss;
      sum += q.loss;
      rows += on[j];
    }
  }
  if (!part) return;
  sum = wave_sum(sum);
  rows = wave_sum(rows);
  if (lane == 0) sums[wave] = make_double2(sum, rows);
  __syncthreads();
  if (threadIdx.x == 0)
    part[blockIdx.x] = make_double2(sums[0].x + sums[1].x + sums[2].x + sums[3].x, sums[0].y + sums[1].y + sums[2].y + sums[3].y);
}

__global__ __launch_bounds__(1024) void ce_classes_total_kernel(int parts, int mean, const double2* __restrict__ part,
                                                                float* __restrict__ loss, float* __restrict__ count) {
  __shared__ double2 tmp[16];
  double sum = 0.0, rows = 0.0;
#pragma unroll 4
  for (int i = threadIdx.x; i < parts; i += 1024) {
    sum += part[i].x;
    rows += part[i].y;
  }
  sum = wave_sum(sum);
  rows = wave_sum(rows);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = make_double2(sum, rows);
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = rows = 0.0;
    for (int w = 0; w < 16; ++w) { sum += tmp[w].x; rows += tmp[w].y; }
    *loss = (float)(mean ? sum / rows : sum);
    *count = (float)rows;
  }
}

struct ClassGrads {
  int n, d, v, reduction;
  int dxs;                       // workgroups that form dx, 128 rows each
  int slices, turns;             // slices of the rows for dw; workgroups of a slice
  int groups, units, teams;      // groups of columns for dx and for dw (0: no dw); waves that share a group's rows
  long long ldx, ldw, ldz, lds;
  const void *x, *w;
  const float *dz, *gout, *count;
  const int* on;
  float *slab, *col;             // [slice, team][class][lds], [slice][class]
  void *dx, *dw;
  int db;
};

// Workgroups [0, dxs): dx of 128 rows; the rest: dw of a slice of the rows, as sums over it.  A wave has a group of columns: lane l the sixteen
// bytes l % 16 of it, so that the instruction for element e of them gets columns V (l % 16) + e from the lanes as they were loaded.
// dx: K are four classes; dw: K are four rows, one per sixteen lanes.
template <typename T, int VB>
__global__ __launch_bounds__(256, 2) void ce_classes_grads_kernel(ClassGrads f) {
  constexpr int V = kVec<T>, NV = 16 * VB, P = NV + 4;
  __shared__ float dz[kTileRows * P];      // [row][class]
  __shared__ int on[kTileRows];
  __shared__ float tmp[256];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), r = lane & 15, g = lane >> 4;
  const float rows = f.reduction == 1 ? *f.count : 1.f, whole = f.reduction == 0 ? 1.f : rows == 0.f ? 0.f : f.gout[0] / rows;
  // g (p - t) of `count` rows from row0 on; zeros behind them and behind the classes (and, as the forward left them, where a row does not
  // count)
  auto fill = [&](int row0, int count) {
    if (tid < kTileRows) on[tid] = tid < count ? f.on[row0 + tid] : 0;
#pragma unroll 4
    for (int idx = tid; idx < kTileRows * (NV / 4); idx += 256) {
      const int i = idx / (NV / 4), c = idx % (NV / 4) * 4;
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      if (i < count && c < f.ldz) {
        y = *reinterpret_cast<const f32x4*>(f.dz + (long long)(row0 + i) * f.ldz + c);
        const float by = f.reduction ? whole : f.on[row0 + i] ? f.gout[row0 + i] : 0.f;
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] *= by;
      }
      *reinterpret_cast<f32x4*>(&dz[i * P + c]) = y;
    }
    __syncthreads();
  };
  if ((int)blockIdx.x < f.dxs) {
    const int row0 = blockIdx.x * kTileRows, count = min(kTileRows, f.n - row0);
    fill(row0, count);
    const int step = 4 / f.teams, team = wave & (f.teams - 1);
    const T* w = (const T*)f.w;
    for (int group = wave / f.teams; group < f.groups; group += step) {
      const int col = (group * 16 + r) * V, left = f.d - col;
      u32x4 raw[VB * 4];
#pragma unroll
      for (int k = 0; k < VB * 4; ++k) raw[k] = load_raw(w + (long long)min(k * 4 + g, f.v - 1) * f.ldw + col, left);
      for (int b = team * 16; b < count; b += 16 * f.teams) {
        f32x4 acc[V] = {};
#pragma unroll
        for (int k = 0; k < VB * 4; ++k) {
          float y[V];
          asm volatile("" : "+v"(raw[k]));      // unpacked here: all of w in float32 would not fit the registers
          unpack<T>(raw[k], y);
          const float a = dz[(b + r) * P + k * 4 + g];
#pragma unroll
          for (int e = 0; e < V; ++e) acc[e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a, y[e], acc[e], 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int i = b + g * 4 + k;
          float y[V];
#pragma unroll
          for (int e = 0; e < V; ++e) y[e] = on[i] ? acc[e][k] : 0.f;
          if (i < count) store_part((T*)f.dx + (long long)(row0 + i) * f.d + col, left, y);
        }
      }
    }
  } else {
    const int wg = blockIdx.x - f.dxs, slice = wg / f.turns, turn = wg % f.turns;
    const int step = 4 / f.teams, team = wave & (f.teams - 1);
    const int group = turn * step + wave / f.teams, col = (group * 16 + r) * V, left = f.d - col;
    const T* x = (const T*)f.x;
    f32x4 acc[VB][V] = {};
    float sum = 0.f;
    auto add = [&](int i, const u32x4& raw) {      // rows i .. i + 3 of the tile
      float y[V], a[VB];
      unpack<T>(raw, y);
#pragma unroll
      for (int b = 0; b < VB; ++b) a[b] = dz[(i + g) * P + b * 16 + r];
#pragma unroll
      for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int e = 0; e < V; ++e) acc[b][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[b], y[e], acc[b][e], 0, 0, 0);
    };
    for (int row0 = slice * kTileRows; row0 < f.n; row0 += f.slices * kTileRows) {
      const int count = min(kTileRows, f.n - row0);
      fill(row0, count);
      if (group < f.units) {
        constexpr int U = VB * V >= 32 ? 4 : 8;
        // (lanes behind the last column read others, for sums that are not stored)
        const bool all = f.d % V == 0 || (group + 1) * 16 * V <= f.d;
        const T* at = x + (left > 0 ? col : 0);
        const int by = 4 * f.teams;
        const u32x4 zero = {0, 0, 0, 0};
        int i = team * 4;
        for (; all && i + (U - 1) * by < count; i += U * by) {
          u32x4 raw[U];
#pragma unroll
          for (int u = 0; u < U; ++u) {
            const int k = i + u * by + g;
            raw[u] = on[k] ? load16(at + (long long)(row0 + k) * f.ldx) : zero;
          }
#pragma unroll
          for (int u = 0; u < U; ++u) add(i + u * by, raw[u]);
        }
        for (; i < count; i += by) add(i, on[i + g] ? load_raw(x + (long long)(row0 + i + g) * f.ldx + col, left) : zero);
      }
      if (f.db && turn == 0) {
#pragma unroll 8
        for (int i = tid / NV; i < kTileRows; i += 256 / NV) sum += dz[i * P + tid % NV];
      }
      __syncthreads();
    }
    if (group < f.units && f.dw) {
#pragma unroll
      for (int b = 0; b < VB; ++b)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int c = b * 16 + g * 4 + k;
          float* out = f.slab + ((long long)(slice * f.teams + team) * f.v + c) * f.lds + col;
          if (c < f.v) {
#pragma unroll
            for (int e = 0; e < V; e += 4)
              if (col + e < f.lds) *reinterpret_cast<f32x4*>(out + e) = f32x4{acc[b][e][k], acc[b][e + 1][k], acc[b][e + 2][k], acc[b][e + 3][k]};
          }
        }
    }
    if (f.db && turn == 0) {
      tmp[tid] = sum;
      __syncthreads();
      if (tid < f.v) {
        for (int k = tid + NV; k < 256; k += NV) sum += tmp[k];
        f.col[(long long)slice * f.v + tid] = sum;
      }
    }
  }
}

// dw: the slabs in order, 64 columns of a class per workgroup, 64 parts of the slabs side by side; the last workgroup: db
template <typename T>
__global__ __launch_bounds__(1024) void ce_classes_join_kernel(int d, int v, int slabs, const float* __restrict__ slab, long long ld,
                                                               int slices, const float* __restrict__ col, T* __restrict__ dw,
                                                               T* __restrict__ db) {
  __shared__ f32x4 tmp[64][16];
  const int per = (d + 63) / 64;
  if (db && blockIdx.x == gridDim.x - 1) {
    float* part = (float*)tmp;      // [part][class]
    const int lanes = v <= 16 ? 16 : v <= 32 ? 32 : 64, parts = 1024 / lanes, c = threadIdx.x % lanes, p = threadIdx.x / lanes;
    const int each = (slices + parts - 1) / parts;
    float s = 0.f;
    if (c < v) {
#pragma unroll 8
      for (int k = p * each; k < min(slices, (p + 1) * each); ++k) s += col[(long long)k * v + c];
    }
    part[threadIdx.x] = s;
    __syncthreads();
    if (p || c >= v) return;
    for (int k = 1; k < parts; ++k) s += part[k * lanes + c];
    db[c] = from_f32<T>(s);
    return;
  }
  const int i = blockIdx.x / per, c = (int)(blockIdx.x % per) * 64 + (threadIdx.x & 15) * 4, part = threadIdx.x >> 4;
  const int each = (slabs + 63) / 64;
  f32x4 y = {0.f, 0.f, 0.f, 0.f};
  if (c < d) {
#pragma unroll 8
    for (int s = part * each; s < min(slabs, (part + 1) * each); ++s) {
      const f32x4 a = *reinterpret_cast<const f32x4*>(slab + ((long long)s * v + i) * ld + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] += a[e];
    }
  }
  tmp[part][threadIdx.x & 15] = y;
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    __syncthreads();
    if (part < o)
#pragma unroll
      for (int e = 0; e < 4; ++e) tmp[part][threadIdx.x & 15][e] = y[e] += tmp[part + o][threadIdx.x & 15][e];
  }
  if (part || c >= d) return;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (c + e < d) dw[(long long)i * d + c + e] = from_f32<T>(y[e]);
}

struct ClassKeep { long long ldz, dz, on, count, bytes; };
inline ClassKeep class_keep(long long n, int v, int train) {
  ClassKeep k;
  k.ldz = round_up(v, 4);
  k.dz = 0;
  k.on = train ? round_up(4 * n * k.ldz, 256) : 0;
  k.count = k.on + (train ? round_up(4 * n, 256) : 0);
  k.bytes = k.count + 256;
  return k;
}
struct ClassPlan { int groups, teams, turns, slices; long long lds, slab, col, bytes; };
inline ClassPlan class_plan(long long n, int d, int v, int dtype) {
  ClassPlan p;
  const int columns = dtype == ISTNET_VOCAB_F32 ? 64 : 128;
  p.groups = (d + columns - 1) / columns;
  p.teams = p.groups == 1 ? 4 : p.groups == 2 ? 2 : 1;
  const int step = 4 / p.teams;
  p.turns = (p.groups + step - 1) / step;
  p.lds = round_up(d, 4);
  // some 512 workgroups, and no more than 32 MB of sums beyond 64 slices
  const long long tiles = (n + kTileRows - 1) / kTileRows, most = std::max<long long>(64, (32ll << 20) / (4 * p.lds * v * p.teams));
  p.slices = (int)std::min({tiles, most, std::max<long long>(16, 512 / p.turns)});
  p.slab = 0;
  p.col = round_up(4ll * p.slices * p.teams * v * p.lds, 256);
  p.bytes = p.col + 4ll * p.slices * v;
  return p;
}
#define CLASS_BLOCKS(v, VB, ...)                                             \
  do {                                                                       \
    if ((v) <= 16) { constexpr int VB = 1; __VA_ARGS__; }                    \
    else if ((v) <= 32) { constexpr int VB = 2; __VA_ARGS__; }               \
    else { constexpr int VB = 4; __VA_ARGS__; }                              \
  } while (0)

}  // namespace

long long vocab_class_ce_keep(long long n, int v, int train) { return class_keep(n, v, train).bytes; }

long long vocab_class_ce_scratch(long long n, int d, int v, int dtype, int backward) {
  return backward ? class_plan(n, d, v, dtype).bytes : 16 * ((n + 63) / 64);
}

int vocab_class_ce_forward(int n, int d, int v, int dtype, int idx64, int train, const void* x, long long ldx, const void* w,
                           long long ldw, const void* bias, const void* target, long long ignore, int reduction, float* loss, void* keep,
                           void* ws, hipStream_t st) {
  const ClassKeep k = class_keep(n, v, train);
  const int per = 64 * row_blocks(v <= 16 ? 1 : v <= 32 ? 2 : 4), tiles = (n + per - 1) / per;
  char* kb = (char*)keep;
  float *dz = train ? (float*)(kb + k.dz) : nullptr, *row_loss = reduction == 0 ? loss : nullptr;
  int* on = train ? (int*)(kb + k.on) : nullptr;
  double2* part = reduction == 0 ? nullptr : (double2*)ws;
  VOCAB_DISPATCH(dtype, T, CLASS_BLOCKS(v, VB, hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_classes_rows_kernel<T, VB>), dim3(tiles), dim3(256), 0,
                                                                  st, n, d, v, (const T*)x, ldx, (const T*)w, ldw, (const T*)bias, target,
                                                                  idx64, ignore, dz, k.ldz, on, row_loss, part)));
  if (reduction != 0)
    hipLaunchKernelGGL(ce_classes_total_kernel, dim3(1), dim3(1024), 0, st, tiles, reduction == 1, part, loss, (float*)(kb + k.count));
  return launch_status();
}

int vocab_class_ce_backward(int n, int d, int v, int dtype, const void* x, long long ldx, const void* w, long long ldw, int reduction,
                            const float* gout, const void* keep, void* ws, void* dx, void* dw, void* db, hipStream_t st) {
  const ClassKeep k = class_keep(n, v, 1);
  const ClassPlan p = class_plan(n, d, v, dtype);
  const char* kb = (const char*)keep;
  ClassGrads f = {};
  f.n = n;
  f.d = d;
  f.v = v;
  f.reduction = reduction;
  f.dxs = dx ? (n + kTileRows - 1) / kTileRows : 0;
  f.slices = p.slices;
  f.turns = dw ? p.turns : 1;
  f.groups = p.groups;
  f.units = dw ? p.groups : 0;
  f.teams = p.teams;
  f.ldx = ldx;
  f.ldw = ldw;
  f.ldz = k.ldz;
  f.lds = p.lds;
  f.x = x;
  f.w = w;
  f.dz = (const float*)(kb + k.dz);
  f.gout = gout;
  f.count = (const float*)(kb + k.count);
  f.on = (const int*)(kb + k.on);
  f.slab = (float*)((char*)ws + p.slab);
  f.col = (float*)((char*)ws + p.col);
  f.dx = dx;
  f.dw = dw;
  f.db = db != nullptr;
  const int wgs = f.dxs + (dw || db ? f.slices * f.turns : 0), joins = (dw ? v * ((d + 63) / 64) : 0) + (db ? 1 : 0);
  VOCAB_DISPATCH(dtype, T, {
    CLASS_BLOCKS(v, VB, hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_classes_grads_kernel<T, VB>), dim3(wgs), dim3(256), 0, st, f));
    if (joins)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_classes_join_kernel<T>), dim3(joins), dim3(1024), 0, st, d, v, p.slices * p.teams, f.slab,
                         p.lds, p.slices, f.col, (T*)dw, (T*)db);
  });
  return launch_status();
}
