// Softmax cross entropy of a linear head over a large vocabulary without its logits (include/istnet_vocab.h).  gfx950, wave64.
//
//   z_iv = x_i . w_v + b_v,   lse_i = log sum_v exp z_iv,   loss_i = lse_i - z_i,t(i)
//   dz_iv = g_i (exp(z_iv - lse_i) - [v = t(i)]),   dx = dz w,   dw = dz^T x,   db_v = sum_i dz_iv
//
// Four matrix products on the matrix cores, one kernel template for all of them:
//   forward     z tile = w x^T, never stored: its epilogue leaves (maximum, sum of exponentials) per row and 256 classes
//   backward    the z tile again, its epilogue writes p - [v = t] of one piece of the vocabulary (16 bits), then
//               dw = (p - t)^T x for that piece and dx += (p - t) w over it
// so the logits cost a second product (8 N V D operations instead of 6) and the memory is that of one piece.
//
// Rows whose target is ignore_index are left out before the products: the rows that count are packed (padded to whole tiles with
// zeros), so masked rows cost nothing and whatever they hold is not looked at.
//
// Numbers.  The logits of bfloat16 and float16 operands are exact products summed in float32.  A float32 operand is held as two
// float16 numbers to a common power of two, x = 2^-e (hi + lo), and a product is hi hi + hi lo + lo hi: 22 bits of each factor, the
// dropped lo lo is 2^-22 of the product at most; entries smaller than 2^-17 of the largest one keep an absolute error of 2^-39 of
// that.  Three half-precision products run at three times the rate of one float32 product on this chip.
// p - t is rounded once the target is taken off, always to float16 numbers scaled by 2^14, and always to more bits than the gradients
// have, because an error of p - t of the result's own rounding would add as much again to it: one number (11 bits) for bfloat16
// operands, which are turned into float16 ones with an exponent in common for this (exact down to 2^-29 of the largest entry), hi + lo
// (22 bits) for float16 and float32 ones.  All sums are float32.
#include <algorithm>

#include "vocab_common.h"

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kNaN = __builtin_nanf("");
constexpr int BK = 32;            // K per step: 64 bytes of a row
constexpr int kStages = 3;        // steps in LDS: one being read, two on their way
constexpr int kPad = 256;         // rows of packed operands are padded to whole tiles
constexpr float kDzScale = 16384.f;      // p - t in float16: 1 -> 2^14, so that p keeps its bits down to 2^-28

// ---- the product ----------------------------------------------------------------------------------------------------------

// An operand: `ld` elements between its rows.  Along-K rows ("KC"): row r of the tile is a row of memory, K is contiguous.
// Across-K rows ("KS"): K runs over the rows of memory and the tile's index is contiguous.  Rows beyond `last_row` and (KS) blocks
// of eight columns beyond `last_col8` are replaced by the last one: what they give is multiplied by zero or not stored.
struct Operand {
  const uint16_t* plane[2];      // float32: hi, lo; else both the same
  long long ld;
  int last_row, last_col8;
};

// What the backward needs of a row: p_v = inv * 2^(z_v - ref) in log2 units; the derivative at the target, p_t - 1, comes from the
// sum over the OTHER classes, so that it (and the loss) keep their relative precision where the target is almost certain.
struct __attribute__((aligned(16))) RowStat { float ref, inv, at_target, unused; };

struct Epilogue {
  // logits
  const float* scal;             // device scalars, see Scal
  const float* bias2;            // log2(e) * bias, -inf behind the last class
  int biased;
  const int* target;             // packed rows: class or < 0
  const RowStat* stat;           // per packed row
  float2* part;                  // [class tile][packed row]: largest of the other classes' logits in log2 units, sum of exponentials
  float* zt;                     // the target's logit as the product left it (with a bias: finished, in log2 units)
  uint16_t* dz[2];               // [packed row][piece], float16 hi (and lo)
  const int* rowmap;             // with weights: packed row -> row
  const float* weights;          // weights of the rows' losses where they are taken into p - t, or null
  long long ld_dz;
  int v, v0;                     // classes in all, first class of the piece
  int parts_ld;
  // gradients
  float* slab;                   // [split][row][ld_slab] float32
  long long slab_stride, ld_slab;
  int accumulate;
  void* out;                     // [row][d] final
  int out_rows, d, reduction;
  const float* gout;
};

// device scalars
// (kXScale, kWScale: of the packed operands; kXBack, kWBack: of those that the gradients are formed from)
enum Scal { kCount = 0, kLogitScale = 1, kXScale = 2, kWScale = 3, kGMax = 4, kXBack = 5, kWBack = 6, kScalars = 8 };

__device__ __forceinline__ int swz_kc(int row) { return ((row >> 1) ^ (row >> 3)) & 3; }
template <int R> __device__ __forceinline__ int swz_ks(int k) { return R >= 256 ? ((k & 3) | (((k >> 3) & 1) << 2)) : (k & 3); }

// sixteen bytes per lane from memory to LDS at `lds` + 16 * lane, past the registers.  Inline: the compiler would wait for every such
// load before the next LDS read; the waits are placed by hand.  Nothing else in these kernels uses m0, and it takes one wait state
// before the load may read it.
__device__ __forceinline__ void load_lds16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}
// all but the last N loads have landed, and what this wave has read from LDS is in its registers
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }
__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void*)p;
}

template <bool KS, int R, int WAVES> struct Stager {
  static constexpr int LOADS = R * 4 / (64 * WAVES);      // sixteen-byte chunks per lane and step
  static constexpr int CPR = KS ? R / 8 : 4;              // chunks per row of the tile in LDS
  uint32_t off[LOADS];
  __device__ __forceinline__ void init(const Operand& o, int first, int wave, int lane) {
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int p = (j * WAVES + wave) * 64 + lane, row = p / CPR, pos = p % CPR;
      if constexpr (KS) {
        const int c8 = min(first / 8 + ((((pos >> 2) ^ swz_ks<R>(row)) << 2) | (pos & 3)), o.last_col8);
        off[j] = (uint32_t)(row * o.ld * 2 + (long long)(c8 - first / 8) * 16);      // first / 8 <= last_col8: not negative beyond the tile
      } else {
        const int r = min(first + row, o.last_row) - first;
        off[j] = (uint32_t)(r * o.ld * 2 + ((pos ^ swz_kc(row)) << 4));
      }
    }
  }
  // step `k0` (first K) of the operand's plane
  __device__ __forceinline__ void issue(const Operand& o, int plane, int first, int k0, uint32_t lds, int wave, int lane) {
    if constexpr (KS) {
      const uint16_t* base = o.plane[plane] + (long long)k0 * o.ld + first;
      if (k0 + BK - 1 <= o.last_row) {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) load_lds16(base, off[j], lds + (j * WAVES + wave) * 1024);
      } else {
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
          const int row = ((j * WAVES + wave) * 64 + lane) / CPR, over = max(0, k0 + row - o.last_row);
          load_lds16(base, off[j] - (uint32_t)(over * o.ld * 2), lds + (j * WAVES + wave) * 1024);
        }
      }
    } else {
      const uint16_t* base = o.plane[plane] + (long long)first * o.ld + k0;
#pragma unroll
      for (int j = 0; j < LOADS; ++j) load_lds16(base, off[j], lds + (j * WAVES + wave) * 1024);
    }
  }
};

// lane addresses of an operand's fragments in its LDS tile
template <bool KS, int R, int BLOCKS> struct Reader {
  static constexpr int N = KS ? BLOCKS : 2;
  uint32_t at[N];
  __device__ __forceinline__ void init(int first, int lane) {
    if constexpr (KS) {
      const int k = ((lane >> 5) << 3) + ((lane & 15) >> 2);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b)
        at[b] = k * R * 2 + (((first / 32 + b) ^ swz_ks<R>(k)) << 6) + (((lane >> 4) & 1) << 5) + ((lane & 3) << 3);
    } else {
      const int row = first + (lane & 31);
#pragma unroll
      for (int s = 0; s < 2; ++s) at[s] = row * 64 + (((2 * s + (lane >> 5)) ^ swz_kc(row)) << 4);
    }
  }
  // the 32 x 16 fragment of block b, half s of the step
  __device__ __forceinline__ s16x8 get(const char* tile, int b, int s) const {
    typedef __attribute__((address_space(3))) s16x4 lds4;
    typedef __attribute__((address_space(3))) s16x8 lds8;
    const auto t = (const __attribute__((address_space(3))) char*)tile;
    if constexpr (KS) {
      const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(t + at[b] + s * 16 * R * 2));
      const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4*)(t + at[b] + s * 16 * R * 2 + 4 * R * 2));
      return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      return *(const lds8*)(t + at[s] + b * 32 * 64);
    }
  }
};

template <typename M> __device__ __forceinline__ f32x16 mfma(s16x8 a, s16x8 b, f32x16 c) {
  if constexpr (__is_same(M, bf16))
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(b16x8, a), __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(h16x8, a), __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}

// (maximum, sum of 2^(x - maximum)) of two sets; an empty one is (-inf, 0), a NaN sum stays NaN
__device__ __forceinline__ float2 merge(float2 p, float2 q) {
  const float m = fmaxf(p.x, q.x);
  if (m == -INFINITY) return make_float2(m, p.y + q.y);
  return make_float2(m, p.y * exp2_raw(p.x - m) + q.y * exp2_raw(q.x - m));
}

// Workgroup -> tile.  Consecutive workgroups go to different XCDs, each with an L2 of its own: every XCD gets a run of tiles, and a run
// walks blocks of 8 tiles of M by all of N, so that the 64 tiles an XCD works on at a time share 8 + 8 panels.
__device__ __forceinline__ void tile_of(int wg, int total, int tm, int tn, int* m, int* n, int* split) {
  const int q = total >> 3, r = total & 7, x = wg & 7;
  int id = x * q + min(x, r) + (wg >> 3);
  const int per = tm * tn;
  *split = id / per;
  id -= *split * per;
  const int g = id / (8 * tn), in = id - g * 8 * tn, gm = min(8, tm - g * 8);
  *m = g * 8 + in % gm;
  *n = in / gm;
}

enum { kLse = 0, kDz = 1, kSlab = 2, kOut = 3 };

// C (M x N) = A (M x K) B (N x K)^T, tile MT x NT, four waves of MT / 2 x NT / 2.  M: matrix element type; SEGS: products of planes
// that make one up, walked one after the other along K, small ones first (1: hi hi; 2: hi lo, hi hi; 3: lo hi, hi lo, hi hi);
// PD: planes of p - t that are written; T: element type of the final output.  The lane of column n holds rows 8 j + 4 (lane / 32) + 0..3 of every 32 x 32 block.
// ROWS_N / ROWS_K: the packed rows are the N dimension (tiles behind the last row leave) / the K dimension (it ends there).
template <typename M, int SEGS, int PD, bool AKS, bool BKS, int MT, int NT, int EPI, typename T>
__global__ __launch_bounds__(256, 2) void ce_gemm_kernel(Operand a, Operand b, int tm, int tn, int ksteps, int per_split, int rows_n,
                                                         int rows_k, Epilogue e) {
  constexpr int WAVES = 4, MB = MT / 64, NB = NT / 64;
  constexpr int ABYTES = MT * 64, BBYTES = NT * 64, STAGE = ABYTES + BBYTES;
  __shared__ __attribute__((aligned(1024))) char lds[kStages * STAGE];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave & 1, wn = wave >> 1;
  int mt, nt, split;
  tile_of(blockIdx.x, gridDim.x, tm, tn, &mt, &nt, &split);
  const int count = (rows_n || rows_k) ? (int)e.scal[kCount] : 0;
  if (rows_n && nt * NT >= count) return;
  if (rows_k) ksteps = (count + BK - 1) / BK;
  const int all = ksteps * SEGS;
  const int t0 = per_split ? min(all, split * per_split) : 0, t1 = per_split ? min(all, t0 + per_split) : all;
  const int m0 = mt * MT, n0 = nt * NT;

  f32x16 acc[MB][NB];
#pragma unroll
  for (int i = 0; i < MB; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  Stager<AKS, MT, WAVES> sa;
  Stager<BKS, NT, WAVES> sb;
  sa.init(a, m0, wave, lane);
  sb.init(b, n0, wave, lane);
  Reader<AKS, MT, MB> ra;
  Reader<BKS, NT, NB> rb;
  ra.init(wm * MT / 2, lane);
  rb.init(wn * NT / 2, lane);
  constexpr int LOADS = Stager<AKS, MT, WAVES>::LOADS + Stager<BKS, NT, WAVES>::LOADS;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(lds_address(lds));

  int seg = SEGS > 1 ? t0 / max(ksteps, 1) : 0, k = t0 - seg * ksteps, slot = 0;      // of the next step to load
  auto issue = [&]() {
    const int pa = SEGS == 3 ? (seg == 0) : 0, pb = SEGS == 3 ? (seg == 1) : SEGS == 2 ? (seg == 0) : 0;
    sa.issue(a, pa, m0, k * BK, lds0 + slot * STAGE, wave, lane);
    sb.issue(b, pb, n0, k * BK, lds0 + slot * STAGE + ABYTES, wave, lane);
    slot = slot == kStages - 1 ? 0 : slot + 1;
    if (++k == ksteps) { k = 0; ++seg; }
  };
  if (t0 < t1) issue();
  if (t0 + 1 < t1) issue();
  int from = 0;
  for (int t = t0; t < t1; ++t) {
    // this step's loads have landed (those of the next may still be under way), for every wave; and every wave is done with the slot
    // of the step before, which is the one the next loads go to
    if (t + 1 < t1) wait_loads<LOADS>(); else wait_loads<0>();
    barrier();
    if (t + 2 < t1) issue();
    const char* at = lds + from * STAGE;
    from = from == kStages - 1 ? 0 : from + 1;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      s16x8 fa[MB], fb[NB];
#pragma unroll
      for (int i = 0; i < MB; ++i) fa[i] = ra.get(at, i, s);
#pragma unroll
      for (int j = 0; j < NB; ++j) fb[j] = rb.get(at + ABYTES, j, s);
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j] = mfma<M>(fa[i], fb[j], acc[i][j]);
    }
  }
  wait_loads<0>();
  barrier();      // the tiles' LDS is free

  const int half = lane >> 5, col = lane & 31;
  // logits in log2 units: without a bias they stay as the product left them and are scaled inside the exponential
  const float c = EPI <= kDz && !e.biased ? e.scal[kLogitScale] : 1.f;
  const int mw = m0 + wm * (MT / 2);
  auto finish_logits = [&](int j) {
    if (e.biased) {
      const float scale = e.scal[kLogitScale];
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 bb = *reinterpret_cast<const f32x4*>(e.bias2 + e.v0 + mw + i * 32 + g * 8 + half * 4);
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[i][j][g * 4 + r] = __builtin_fmaf(acc[i][j][g * 4 + r], scale, bb[r]);
        }
    } else if (e.v0 + m0 + MT > e.v) {
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (e.v0 + mw + i * 32 + (r >> 2) * 8 + half * 4 + (r & 3) >= e.v) acc[i][j][r] = -INFINITY;
    }
  };
  if constexpr (EPI == kLse) {
    float2* pair = reinterpret_cast<float2*>(lds);
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = n0 + wn * (NT / 2) + j * 32 + col;
      finish_logits(j);
      const int t = e.target[n] - mw;
      if (__any(t >= 0 && t < MT / 2)) {
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (t == i * 32 + (r >> 2) * 8 + half * 4 + (r & 3)) {
              e.zt[n] = acc[i][j][r];
              acc[i][j][r] = -INFINITY;
            }
      }
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
      m = fmaxf(m, __shfl_xor(m, 32)) * c;
      const float ref = m == -INFINITY ? 0.f : m;
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += exp2_raw(__builtin_fmaf(acc[i][j][r], c, -ref));
      s += __shfl_xor(s, 32);
      if (half == 0) pair[wm * NT + wn * (NT / 2) + j * 32 + col] = make_float2(m, s);
    }
    __syncthreads();
    if (threadIdx.x < NT) {
      e.part[(long long)mt * e.parts_ld + n0 + threadIdx.x] = merge(pair[threadIdx.x], pair[NT + threadIdx.x]);
    }
  } else if constexpr (EPI == kDz) {
    // per wave NT / 2 rows of MT / 2 classes, written row by row: pitch MT / 2 + 8 elements keeps the rows' writes apart
    constexpr int PITCH = MT / 2 + 8, ROWS = NT / 2;
    static_assert(4 * ROWS * PITCH * 2 <= kStages * STAGE, "the epilogue's rows fit the tiles' LDS");
    uint16_t* mine = reinterpret_cast<uint16_t*>(lds) + wave * ROWS * PITCH;
#pragma unroll
    for (int pl = 0; pl < PD; ++pl) {
#pragma unroll
      for (int j = 0; j < NB; ++j) {
        const int n = n0 + wn * (NT / 2) + j * 32 + col;
        if (pl == 0) {
          finish_logits(j);
          const RowStat st = e.stat[n];
          float one = kDzScale;
          if (e.weights) one *= n < count ? e.weights[e.rowmap[n]] / e.scal[kGMax] : 0.f;
          const float w = one * st.inv;
#pragma unroll
          for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = w * exp2_raw(__builtin_fmaf(acc[i][j][r], c, -st.ref));
          const int t = e.target[n] - e.v0 - mw;
          if (__any(t >= 0 && t < MT / 2)) {
            const float x = one * st.at_target;
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
              for (int r = 0; r < 16; ++r) acc[i][j][r] = t == i * 32 + (r >> 2) * 8 + half * 4 + (r & 3) ? x : acc[i][j][r];
          }
        }
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            uint16_t h[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const float x = acc[i][j][g * 4 + r];
              const f16 y = (f16)x;
              h[r] = __builtin_bit_cast(uint16_t, y);
              if (PD == 2 && pl == 0) acc[i][j][g * 4 + r] = x - (float)y;
            }
            *reinterpret_cast<uint2*>(mine + (j * 32 + col) * PITCH + i * 32 + g * 8 + half * 4) =
                make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
          }
      }
      // a wave reads what it wrote itself: LDS keeps its order
      constexpr int CH = MT / 16;      // sixteen-byte chunks of a row
      uint16_t* out = e.dz[pl] + (long long)(n0 + wn * ROWS) * e.ld_dz + mw;
      asm volatile("" ::: "memory");
#pragma unroll
      for (int q = 0; q < ROWS * CH / 64; ++q) {
        const int p = q * 64 + lane, row = p / CH, ch = p % CH;
        *reinterpret_cast<u32x4*>(out + row * e.ld_dz + ch * 8) = *reinterpret_cast<const u32x4*>(mine + row * PITCH + ch * 8);
      }
      asm volatile("" ::: "memory");
    }
  } else if constexpr (EPI == kSlab) {
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      float* row = e.slab + split * e.slab_stride + (long long)(n0 + wn * (NT / 2) + j * 32 + col) * e.ld_slab;
#pragma unroll
      for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          f32x4* p = reinterpret_cast<f32x4*>(row + m0 + wm * (MT / 2) + i * 32 + g * 8 + half * 4);
          f32x4 x;
#pragma unroll
          for (int r = 0; r < 4; ++r) x[r] = acc[i][j][g * 4 + r];
          if (e.accumulate) {
            const f32x4 y = *p;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] += y[r];
          }
          *p = x;
        }
    }
  } else {
    const float rows = e.scal[kCount];
    const float g = e.reduction == 0 ? e.scal[kGMax] : e.reduction == 1 ? e.gout[0] / rows : e.gout[0];
    const float f = rows == 0.f ? 0.f : g / kDzScale / e.scal[kXBack];
#pragma unroll
    for (int j = 0; j < NB; ++j) {
      const int n = n0 + wn * (NT / 2) + j * 32 + col;
      if (n < e.out_rows) {
        T* row = reinterpret_cast<T*>(e.out) + (long long)n * e.d;
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int m = m0 + wm * (MT / 2) + i * 32 + q * 8 + half * 4;
            if ((e.d & 3) == 0 && m < e.d) {
              if constexpr (sizeof(T) == 4) {
                f32x4 x;
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = f * acc[i][j][q * 4 + r];
                *reinterpret_cast<f32x4*>(row + m) = x;
              } else {
                uint16_t h[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) h[r] = __builtin_bit_cast(uint16_t, from_f32<T>(f * acc[i][j][q * 4 + r]));
                *reinterpret_cast<uint2*>(row + m) = make_uint2(h[0] | ((uint32_t)h[1] << 16), h[2] | ((uint32_t)h[3] << 16));
              }
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (m + r < e.d) row[m + r] = from_f32<T>(f * acc[i][j][q * 4 + r]);
            }
          }
      }
    }
  }
}

// ---- before and after the products -------------------------------------------------------------------------------------------

// largest magnitude of a row (infinities as they come, NaN passed over), this lane's part
template <typename T> __device__ __forceinline__ float row_amax(const T* row, int d, float m) {
  for (int c = (threadIdx.x & 63) * kVec<T>; c < d; c += 64 * kVec<T>) {
    float f[kVec<T>];
    load_part(row + c, d - c, f);
#pragma unroll
    for (int i = 0; i < kVec<T>; ++i) m = fmaxf(m, fabsf(f[i]));
  }
  return m;
}
__device__ __forceinline__ void store_amax(float m, float* tmp, float* part) {
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) part[blockIdx.x] = fmaxf(fmaxf(tmp[0], tmp[1]), fmaxf(tmp[2], tmp[3]));
}
// the largest magnitude of the rows of x that count ([0, xwgs)) and of w, one value per workgroup
__global__ __launch_bounds__(256) void ce_amax_kernel(int n, int v, int d, const float* __restrict__ x, long long ldx,
                                                      const float* __restrict__ w, long long ldw, const void* __restrict__ target,
                                                      int idx64, long long ignore, int xwgs, float* __restrict__ part) {
  __shared__ float tmp[4];
  const int wave = threadIdx.x >> 6;
  float m = 0.f;
  if ((int)blockIdx.x < xwgs) {
    for (int r = blockIdx.x * 4 + wave; r < n; r += xwgs * 4)
      if (load_index(target, r, idx64) != ignore) m = row_amax(x + r * ldx, d, m);
  } else {
    for (int r = (blockIdx.x - xwgs) * 4 + wave; r < v; r += (gridDim.x - xwgs) * 4) m = row_amax(w + r * ldw, d, m);
  }
  store_amax(m, tmp, part);
}
// the same of packed rows
__global__ __launch_bounds__(256) void ce_amax_packed_kernel(int kp, const bf16* __restrict__ xp, const float* __restrict__ scal, int v,
                                                             int d, const bf16* __restrict__ w, long long ldw, int xwgs,
                                                             float* __restrict__ part) {
  __shared__ float tmp[4];
  const int wave = threadIdx.x >> 6, count = (int)scal[kCount];
  float m = 0.f;
  if ((int)blockIdx.x < xwgs) {
    for (int r = blockIdx.x * 4 + wave; r < count; r += xwgs * 4) m = row_amax(xp + (long long)r * kp, kp, m);
  } else {
    for (int r = (blockIdx.x - xwgs) * 4 + wave; r < v; r += (gridDim.x - xwgs) * 4) m = row_amax(w + r * ldw, d, m);
  }
  store_amax(m, tmp, part);
}

// counted rows per block of 256
__global__ __launch_bounds__(256) void ce_count_kernel(int n, const void* __restrict__ target, int idx64, long long ignore,
                                                       int* __restrict__ blocks) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  const int c = __syncthreads_count(i < n && load_index(target, i, idx64) != ignore);
  if (threadIdx.x == 0) blocks[blockIdx.x] = c;
}

__device__ __forceinline__ float scale_for(float amax) {      // power of two that takes amax to [2^14, 2^15)
  if (!(amax > 0.f) || amax > 3.4e38f) return 1.f;
  int ex;
  frexpf(amax, &ex);                                          // amax = f 2^ex, f in [1/2, 1)
  return ldexpf(1.f, max(-126, min(126, 15 - ex)));
}

// rows counted before each block of 256 (in place where ce_count_kernel left the counts), number of rows, scales
__global__ __launch_bounds__(1024) void ce_plan_kernel(int n, int counted, const void* __restrict__ target, int idx64, long long ignore,
                                                       int split, int xwgs, int wgs, const float* __restrict__ amax,
                                                       int* __restrict__ blocks, float* __restrict__ scal) {
  __shared__ int tmp[16];
  __shared__ float tmx[16], tmw[16];
  const int nb = (n + 255) / 256, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (!counted) {
    for (int b = wave; b < nb; b += 16) {
      int c = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int i = b * 256 + j * 64 + lane;
        c += __popcll(__ballot(i < n && load_index(target, i < n ? i : 0, idx64) != ignore));
      }
      if (lane == 0) blocks[b] = c;
    }
    __syncthreads();
  }
  int carry = 0;
  for (int base = 0; base < nb; base += 1024) {
    const int b = base + threadIdx.x, x = b < nb ? blocks[b] : 0;
    int s = x;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int y = __shfl_up(s, o);
      if (lane >= o) s += y;
    }
    if (lane == 63) tmp[wave] = s;
    __syncthreads();
    int before = 0, all = 0;
    for (int w = 0; w < 16; ++w) {
      before += w < wave ? tmp[w] : 0;
      all += tmp[w];
    }
    __syncthreads();
    if (b < nb) blocks[b] = carry + before + s - x;
    carry += all;
  }
  float mx = 0.f, mw = 0.f;
  if (split) {
    for (int i = threadIdx.x; i < wgs; i += 1024) {
      if (i < xwgs) mx = fmaxf(mx, amax[i]); else mw = fmaxf(mw, amax[i]);
    }
    mx = wave_max(mx);
    mw = wave_max(mw);
    if (lane == 0) { tmx[wave] = mx; tmw[wave] = mw; }
    __syncthreads();
    for (int w = 0; w < 16; ++w) { mx = fmaxf(mx, tmx[w]); mw = fmaxf(mw, tmw[w]); }
  }
  if (threadIdx.x == 0) {
    const float sx = split ? scale_for(mx) : 1.f, sw = split ? scale_for(mw) : 1.f;
    scal[kCount] = (float)carry;
    scal[kLogitScale] = kLog2e / sx / sw;
    scal[kXScale] = sx;
    scal[kWScale] = sw;
    scal[kGMax] = 1.f;
    scal[kXBack] = sx;
    scal[kWBack] = sw;
  }
}

// scales of bfloat16 operands as float16 ones
__global__ __launch_bounds__(1024) void ce_scales_kernel(int xwgs, int wgs, const float* __restrict__ amax, float* __restrict__ scal) {
  __shared__ float tmx[16], tmw[16];
  const int i = threadIdx.x, lane = i & 63, wave = i >> 6;
  const float m = i < wgs ? amax[i] : 0.f, mx = wave_max(i < xwgs ? m : 0.f), mw = wave_max(i < xwgs ? 0.f : m);
  if (lane == 0) { tmx[wave] = mx; tmw[wave] = mw; }
  __syncthreads();
  if (i == 0) {
    float x = 0.f, w = 0.f;
    for (int k = 0; k < 16; ++k) { x = fmaxf(x, tmx[k]); w = fmaxf(w, tmw[k]); }
    scal[kXBack] = scale_for(x);
    scal[kWBack] = scale_for(w);
  }
}

// eight elements of a row, scaled and rounded (P == 2: split), as they lie in the packed operand
template <typename T, int P>
__device__ __forceinline__ void pack8(const T* src, int left, float scale, u32x4* hi, u32x4* lo) {
  float f[8];
  if constexpr (sizeof(T) == 2) {
    load_part(src, left, f);
    if (scale != 1.f) {
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] *= scale;
    }
    *hi = pack<T>(f);
  } else {
    float g[4], h[4];
    load_part(src, left, g);
    load_part(src + 4, left - 4, h);
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[i] = g[i] * scale; f[4 + i] = h[i] * scale; }
    float r[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) r[i] = f[i] - (float)(f16)f[i];
    *hi = pack<f16>(f);
    *lo = pack<f16>(r);
  }
}

// Packed rows of x (and of w where its own rows cannot be read as they are), the bias in log2 units.  Workgroups [0, xwgs): 16 rows of
// x each; the next 16: the zeros behind the last packed row; the rest: 4 rows of w each step, and the bias.
constexpr int kPackRows = 16;
template <typename T, int P>
__global__ __launch_bounds__(256) void ce_pack_kernel(int n, int v, int d, int kp, int vp, const T* __restrict__ x, long long ldx,
                                                      const T* __restrict__ w, long long ldw, const T* __restrict__ bias,
                                                      const void* __restrict__ target, int idx64, long long ignore, int xwgs,
                                                      int pack_w, const int* __restrict__ blocks, const float* __restrict__ scal,
                                                      uint16_t* __restrict__ xp, long long xplane, uint16_t* __restrict__ wp,
                                                      long long wplane, float* __restrict__ bias2, int* __restrict__ rowmap,
                                                      int* __restrict__ inverse, int* __restrict__ tgt, float* __restrict__ row_loss) {
  __shared__ int flag[4];
  __shared__ int where[256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wg = blockIdx.x;
  if (wg < xwgs) {
    const int block = wg / (256 / kPackRows), i = block * 256 + threadIdx.x;
    const long long t = i < n ? load_index(target, i, idx64) : ignore;
    const bool on = i < n && t != ignore;
    const uint64_t m = __ballot(on);
    if (lane == 0) flag[wave] = __popcll(m);
    __syncthreads();
    int at = blocks[block] + __popcll(m & ((1ull << lane) - 1));
    for (int j = 0; j < wave; ++j) at += flag[j];
    where[threadIdx.x] = on ? at : -1;
    const int r0 = (wg % (256 / kPackRows)) * kPackRows;
    if ((int)threadIdx.x >= r0 && (int)threadIdx.x < r0 + kPackRows && i < n) {
      inverse[i] = on ? at : -1;
      if (on) {
        rowmap[at] = i;
        tgt[at] = (t >= 0 && t < v) ? (int)t : -1;
      } else if (row_loss) {
        row_loss[i] = 0.f;
      }
    }
    __syncthreads();
    const float s = scal[kXScale];
    for (int r = r0 + wave; r < r0 + kPackRows; r += 4) {
      const int to = where[r];
      if (to < 0) continue;
      const T* src = x + (long long)(block * 256 + r) * ldx;
      for (int c = lane * 8; c < kp; c += 512) {
        u32x4 hi, lo;
        pack8<T, P>(src + c, d - c, s, &hi, &lo);
        store16(xp + (long long)to * kp + c, hi);
        if constexpr (P == 2) store16(xp + xplane + (long long)to * kp + c, lo);
      }
    }
  } else if (wg < xwgs + kPad / kPackRows) {
    const int count = (int)scal[kCount], end = (count + kPad - 1) / kPad * kPad, r0 = count + (wg - xwgs) * kPackRows;
    const u32x4 zero = {0, 0, 0, 0};
    for (int r = r0 + wave; r < min(end, r0 + kPackRows); r += 4) {
      for (int c = lane * 8; c < kp; c += 512) {
        store16(xp + (long long)r * kp + c, zero);
        if constexpr (P == 2) store16(xp + xplane + (long long)r * kp + c, zero);
      }
      if (lane == 0) tgt[r] = -2;
    }
  } else {
    const int first = wg - xwgs - kPad / kPackRows, wgs = gridDim.x - xwgs - kPad / kPackRows;
    for (int c = first * 256 + threadIdx.x; c < vp; c += wgs * 256)
      bias2[c] = c >= v ? -INFINITY : bias ? kLog2e * to_f32(bias[c]) : 0.f;
    if (pack_w) {
      const float s = scal[kWScale];
      for (int r = first * 4 + wave; r < v; r += wgs * 4) {
        const T* src = w + r * ldw;
        for (int c = lane * 8; c < kp; c += 512) {
          u32x4 hi, lo;
          pack8<T, P>(src + c, d - c, s, &hi, &lo);
          store16(wp + (long long)r * kp + c, hi);
          if constexpr (P == 2) store16(wp + wplane + (long long)r * kp + c, lo);
        }
      }
    }
  }
}

// statistics and loss of 16 packed rows per workgroup, from the tiles' partial sums
__global__ __launch_bounds__(256) void ce_finish_kernel(int tiles, int parts_ld, int biased, const float2* __restrict__ part,
                                                        const float* __restrict__ zt, const int* __restrict__ tgt,
                                                        const int* __restrict__ rowmap, const float* __restrict__ scal,
                                                        RowStat* __restrict__ stat, float* __restrict__ packed_loss,
                                                        float* __restrict__ row_loss) {
  __shared__ float2 tmp[16][17];
  const int count = (int)scal[kCount], t = threadIdx.x & 15, j = threadIdx.x >> 4, row = blockIdx.x * 16 + t;
  if (blockIdx.x * 16 >= (count + kPad - 1) / kPad * kPad) return;
  float2 ms = make_float2(-INFINITY, 0.f);
  if (row < count) {
#pragma unroll 4
    for (int k = j; k < tiles; k += 16) ms = merge(ms, part[(long long)k * parts_ld + row]);
  }
  tmp[j][t] = ms;
  __syncthreads();
  if (j == 0) {
    if (row < count) {
      for (int k = 1; k < 16; ++k) ms = merge(ms, tmp[k][t]);
      // ms: the other classes.  d = target's logit above their largest; loss = log(1 + rest), rest = others over target
      RowStat r = {kNaN, kNaN, kNaN, 0.f};
      float loss = kNaN;
      if (tgt[row] >= 0) {
        const float c = biased ? 1.f : scal[kLogitScale], z = zt[row];
        const float d = ms.x == -INFINITY ? INFINITY : __builtin_fmaf(z, c, -ms.x);
        r.ref = d > 0.f ? z * c : ms.x;
        const float others = ms.x == -INFINITY ? ms.y : ms.y * exp2_raw(ms.x - r.ref), mine = exp2_raw(__builtin_fmaf(z, c, -r.ref));
        r.inv = 1.f / (others + mine);
        if (d < -100.f) {
          loss = kLn2 * -d + logf(ms.y);
          r.at_target = -1.f + 0.f * loss;      // NaN stays NaN
          if (d == -INFINITY) r.at_target = -1.f;
        } else {
          const float rest = others / mine;
          loss = log1pf(rest);
          r.at_target = -rest / (1.f + rest);
        }
      }
      stat[row] = r;
      packed_loss[row] = loss;
      if (row_loss) row_loss[rowmap[row]] = loss;
    } else {
      stat[row] = {INFINITY, 1.f, 0.f, 0.f};      // a row of padding: every probability zero
    }
  }
}

__global__ __launch_bounds__(1024) void ce_total_kernel(int mean, const float* __restrict__ packed_loss, const float* __restrict__ scal,
                                                        float* __restrict__ loss) {
  __shared__ double tmp[16];
  const int count = (int)scal[kCount];
  double sum = 0.0;
  for (int i = threadIdx.x; i < count; i += 1024) sum += packed_loss[i];
  sum = wave_sum(sum);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < 16; ++w) sum += tmp[w];
    *loss = (float)(mean ? sum / count : sum);
  }
}

// largest |g| over the counted rows (weights of the rows' losses)
__global__ __launch_bounds__(1024) void ce_gmax_kernel(const float* __restrict__ gout, const int* __restrict__ rowmap,
                                                       float* __restrict__ scal) {
  __shared__ float tmp[16];
  const int count = (int)scal[kCount];
  float m = 0.f;
  for (int i = threadIdx.x; i < count; i += 1024) m = fmaxf(m, fabsf(gout[rowmap[i]]));
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) tmp[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < 16; ++w) m = fmaxf(m, tmp[w]);
    scal[kGMax] = m > 0.f ? m : 1.f;
  }
}

// eight elements as float16 (P == 2: hi and lo) whatever their type
template <typename T, int P>
__device__ __forceinline__ void pack8_f16(const T* src, int left, float scale, u32x4* hi, u32x4* lo) {
  if constexpr (__is_same(T, bf16)) {
    float f[8];
    load_part(src, left, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] *= scale;
    *hi = pack<f16>(f);
  } else {
    pack8<T, P>(src, left, scale, hi, lo);
  }
}

// Packed float16 rows that dw is formed from: of g_i / max |g| * x_i where the rows' losses have weights of their own, of x_i else.
template <typename T, int P>
__global__ __launch_bounds__(256) void ce_back_x_kernel(int d, int kp, const T* __restrict__ x, long long ldx,
                                                        const float* __restrict__ gout, const int* __restrict__ rowmap,
                                                        const float* __restrict__ scal, uint16_t* __restrict__ xp, long long xplane) {
  const int count = (int)scal[kCount], end = (count + kPad - 1) / kPad * kPad, lane = threadIdx.x & 63;
  const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= end) return;
  const int i = r < count ? rowmap[r] : -1;
  const float s = i < 0 ? 0.f : gout ? gout[i] / scal[kGMax] * scal[kXBack] : scal[kXBack];
  for (int c = lane * 8; c < kp; c += 512) {
    u32x4 hi = {0, 0, 0, 0}, lo = {0, 0, 0, 0};
    if (i >= 0) pack8_f16<T, P>(x + (long long)i * ldx + c, d - c, s, &hi, &lo);
    store16(xp + (long long)r * kp + c, hi);
    if constexpr (P == 2) store16(xp + xplane + (long long)r * kp + c, lo);
  }
}

// rows of a piece of bfloat16 w as float16
__global__ __launch_bounds__(256) void ce_back_w_kernel(int rows, int d, int kp, const bf16* __restrict__ w, long long ldw,
                                                        const float* __restrict__ scal, uint16_t* __restrict__ wp) {
  const int lane = threadIdx.x & 63;
  const float s = scal[kWBack];
  for (int r = blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += gridDim.x * 4) {
    for (int c = lane * 8; c < kp; c += 512) {
      u32x4 hi, lo;
      pack8_f16<bf16, 1>(w + r * ldw + c, d - c, s, &hi, &lo);
      store16(wp + (long long)r * kp + c, hi);
    }
  }
}

// dx: slabs added in order, scaled, back to the rows they belong to; rows that do not count get zeros
template <typename T>
__global__ __launch_bounds__(256) void ce_dx_kernel(int n, int d, int splits, const float* __restrict__ slab, long long slab_stride,
                                                    long long ld, const int* __restrict__ inverse, const float* __restrict__ gout,
                                                    int reduction, int folded, const float* __restrict__ scal, T* __restrict__ dx) {
  const int per = (d + 3) / 4;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, i = id / per;
  if (i >= n) return;
  const int c = (int)(id % per) * 4, at = inverse[i];
  f32x4 x = {0.f, 0.f, 0.f, 0.f};
  if (at >= 0) {
    const float* p = slab + at * ld + c;
    x = *reinterpret_cast<const f32x4*>(p);
    for (int s = 1; s < splits; ++s) {
      const f32x4 y = *reinterpret_cast<const f32x4*>(p + s * slab_stride);
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] += y[r];
    }
    const float g = (folded ? scal[kGMax] : reduction == 0 ? gout[i] : reduction == 1 ? gout[0] / scal[kCount] : gout[0]) / kDzScale /
                    scal[kWBack];
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] *= g;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (c + r < d) dx[i * d + c + r] = from_f32<T>(x[r]);
}

// dw where its product was split along the rows
template <typename T>
__global__ __launch_bounds__(256) void ce_dw_kernel(int rows, int d, int splits, const float* __restrict__ slab, long long slab_stride,
                                                    long long ld, const float* __restrict__ gout, int reduction,
                                                    const float* __restrict__ scal, T* __restrict__ dw) {
  const int per = (d + 3) / 4;
  const long long id = (long long)blockIdx.x * 256 + threadIdx.x, i = id / per;
  if (i >= rows) return;
  const int c = (int)(id % per) * 4;
  const float* p = slab + i * ld + c;
  f32x4 x = *reinterpret_cast<const f32x4*>(p);
  for (int s = 1; s < splits; ++s) {
    const f32x4 y = *reinterpret_cast<const f32x4*>(p + s * slab_stride);
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] += y[r];
  }
  const float n = scal[kCount];
  const float g = n == 0.f ? 0.f : (reduction == 0 ? scal[kGMax] : reduction == 1 ? gout[0] / n : gout[0]) / kDzScale / scal[kXBack];
#pragma unroll
  for (int r = 0; r < 4; ++r)
    if (c + r < d) dw[i * d + c + r] = from_f32<T>(g * x[r]);
}

// db: column sums of p - t over the packed rows, `chunks` parts of the rows side by side, joined in order
template <int PD>
__global__ __launch_bounds__(256) void ce_colsum_kernel(int width, const uint16_t* __restrict__ hi, const uint16_t* __restrict__ lo,
                                                        long long ld, const float* __restrict__ gout, const int* __restrict__ rowmap,
                                                        const float* __restrict__ scal, int chunks, float* __restrict__ part) {
  const int c = (blockIdx.x * 64 + (threadIdx.x & 63)) * 8, chunk = blockIdx.y * 4 + (threadIdx.x >> 6);
  const int count = (int)scal[kCount], per = (count + chunks - 1) / chunks, a = chunk * per, b = min(count, a + per);
  if (c >= width) return;
  float s[8] = {};
#pragma unroll 4
  for (int r = a; r < b; ++r) {
    const float g = gout ? gout[rowmap[r]] : 1.f;
    float f[8];
    unpack<f16>(*reinterpret_cast<const u32x4*>(hi + r * ld + c), f);
    if constexpr (PD == 2) {
      float l[8];
      unpack<f16>(*reinterpret_cast<const u32x4*>(lo + r * ld + c), l);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] += l[i];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) s[i] += g * f[i];
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part[(long long)chunk * width + c + i] = s[i];
}
template <typename T>
__global__ __launch_bounds__(256) void ce_db_kernel(int rows, int width, int chunks, const float* __restrict__ part,
                                                    const float* __restrict__ gout, int reduction, int folded,
                                                    const float* __restrict__ scal, T* __restrict__ db) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= rows) return;
  double s = 0.0;
#pragma unroll 4
  for (int k = 0; k < chunks; ++k) s += part[(long long)k * width + c];
  const float n = scal[kCount];
  const float g = n == 0.f ? 0.f : (folded ? scal[kGMax] : reduction == 0 ? 1.f : reduction == 1 ? gout[0] / n : gout[0]) / kDzScale;
  db[c] = from_f32<T>((float)(g * s));
}

// ---- sizes and launches ------------------------------------------------------------------------------------------------------

constexpr int kMT = 256, kNT = 128;
constexpr int kChunks = 64;                              // parts of the rows of a bias gradient
constexpr long long kPieceBytes = 512ll << 20;           // memory of one piece of p - t

inline long long round_up(long long x, long long m) { return (x + m - 1) / m * m; }
inline bool ce_ok(long long n, int d, int v, int dtype) {
  return n >= 1 && n <= (1ll << 22) && d >= 1 && d <= (1 << 20) && v >= 1 && v <= (1 << 28) && dtype >= 0 && dtype <= 2 &&
         ((n + 127) / 128) * ((v + 255ll) / 256) <= (1ll << 23);      // a launch holds fewer than 2^32 threads
}
// rows of w that the matrix cores can be fed from as they lie: whole steps of K, sixteen-byte chunks
inline bool direct_w(int d, int dtype, const void* w, long long ldw) {
  return dtype != ISTNET_VOCAB_F32 && d % BK == 0 && ldw % 8 == 0 && ldw <= (1 << 22) && ((uintptr_t)w & 15) == 0;
}

struct Keep {      // what the backward needs, in the caller's `keep`
  long long np, kp, vp, planes;
  long long xp, wp, bias2, rowmap, inverse, tgt, stat, scal, bytes;
};
inline Keep keep_plan(long long n, int d, int v, int dtype, bool direct) {
  Keep k = {};
  k.planes = dtype == ISTNET_VOCAB_F32 ? 2 : 1;
  k.np = round_up(n, kPad) + kPad;      // zeros are written up to the next whole tile behind the last row
  k.kp = round_up(d, BK);
  k.vp = round_up(v, kMT);
  long long at = 0;
  auto take = [&](long long bytes) { const long long o = at; at += round_up(bytes, 256); return o; };
  k.xp = take(2 * k.planes * k.np * k.kp);
  k.wp = direct ? 0 : take(2 * k.planes * v * k.kp);
  k.bias2 = take(4 * k.vp);
  k.rowmap = take(4 * k.np);
  k.inverse = take(4 * k.np);
  k.tgt = take(4 * k.np);
  k.stat = take((long long)sizeof(RowStat) * k.np);
  k.scal = take(4 * kScalars);
  k.bytes = at;
  return k;
}
struct Forward { long long part, zt, loss, blocks, amax, bytes; int tiles; };
inline Forward forward_plan(const Keep& k) {
  Forward f = {};
  f.tiles = (int)(k.vp / kMT);
  long long at = 0;
  auto take = [&](long long bytes) { const long long o = at; at += round_up(bytes, 256); return o; };
  f.part = take(8ll * f.tiles * k.np);
  f.zt = take(4 * k.np);
  f.loss = take(4 * k.np);
  f.blocks = take(4 * (k.np / 256 + 1));
  f.amax = take(4 * 1024);
  f.bytes = at;
  return f;
}
struct Backward {
  int pieces, dx_splits, dx_per, dw_splits, dw_per;
  long long piece, dz, xb, wb, amax, dx_slab, dx_rows, dw_slab, dw_rows, col, ld, bytes;
};
inline Backward backward_plan(const Keep& k, long long n, int d, int v, int dtype, int reduction) {
  Backward b = {};
  const long long planes = dtype == ISTNET_VOCAB_BF16 ? 1 : 2;      // of p - t
  const long long most = std::max<long long>(kMT, kPieceBytes / (2 * planes * k.np) / kMT * kMT);
  b.pieces = (int)((k.vp + most - 1) / most);
  b.piece = round_up((k.vp + b.pieces - 1) / b.pieces, kMT);
  b.pieces = (int)((k.vp + b.piece - 1) / b.piece);
  b.ld = round_up(d, kMT);
  const long long dt = b.ld / kMT, seg = dtype == ISTNET_VOCAB_F32 ? 3 : planes;
  // two workgroups fit a compute unit: split K while that fills more of the 512 places, eight steps at least
  auto splits = [&](long long tiles, long long steps) {
    return std::max<long long>(1, std::min<long long>(512 / std::max<long long>(1, tiles), steps / 8));
  };
  const long long most_rows = std::min<long long>(v, b.piece), dx_steps = (most_rows + BK - 1) / BK * seg, dw_steps = (n + BK - 1) / BK * seg;
  b.dx_rows = round_up(n, kNT);
  b.dw_rows = round_up(most_rows, kNT);
  b.dx_splits = (int)splits(dt * (b.dx_rows / kNT), dx_steps);
  b.dx_per = (int)((dx_steps + b.dx_splits - 1) / b.dx_splits);
  b.dw_splits = (int)splits(dt * (b.dw_rows / kNT), dw_steps);
  b.dw_per = (int)((dw_steps + b.dw_splits - 1) / b.dw_splits);
  long long at = 0;
  auto take = [&](long long bytes) { const long long o = at; at += round_up(bytes, 256); return o; };
  b.dz = take(2 * planes * k.np * b.piece);
  b.xb = dtype == ISTNET_VOCAB_BF16 || (dtype == ISTNET_VOCAB_F32 && reduction == 0) ? take(2 * k.planes * k.np * k.kp) : 0;
  b.wb = dtype == ISTNET_VOCAB_BF16 ? take(2 * most_rows * k.kp) : 0;
  b.amax = take(4 * 1024);
  b.dx_slab = take(4 * b.dx_splits * b.dx_rows * b.ld);
  b.dw_slab = b.dw_splits > 1 ? take(4 * b.dw_splits * b.dw_rows * b.ld) : 0;
  b.col = take(4ll * kChunks * b.piece);
  b.bytes = at;
  return b;
}

// element type of the logits' product, planes of the operands and of p - t, products of planes per product of the logits / gradients
template <typename T> struct Matrix;
template <> struct Matrix<float> { typedef f16 M; static constexpr int P = 2, PD = 2, LOGIT = 3, GRAD = 3; };
template <> struct Matrix<f16> { typedef f16 M; static constexpr int P = 1, PD = 2, LOGIT = 1, GRAD = 2; };
template <> struct Matrix<bf16> { typedef bf16 M; static constexpr int P = 1, PD = 1, LOGIT = 1, GRAD = 1; };

}  // namespace

extern "C" int istnet_linear_ce_keep_kib(long long n, int d, int v, int dtype, const void* w, long long ldw) {
  if (!ce_ok(n, d, v, dtype)) return -1;
  return (int)((keep_plan(n, d, v, dtype, direct_w(d, dtype, w, ldw)).bytes + 1023) / 1024);
}
extern "C" int istnet_linear_ce_scratch_kib(long long n, int d, int v, int dtype, int reduction, int backward) {
  if (!ce_ok(n, d, v, dtype) || reduction < 0 || reduction > 2) return -1;
  const Keep k = keep_plan(n, d, v, dtype, false);
  return (int)(((backward ? backward_plan(k, n, d, v, dtype, reduction).bytes : forward_plan(k).bytes) + 1023) / 1024);
}

extern "C" int istnet_linear_ce_forward(long long n, int d, int v, int dtype, int idx64, const void* x, long long ldx, const void* w,
                                        long long ldw, const void* bias, const void* target, long long ignore, int reduction,
                                        float* loss, void* keep, void* ws, void* stream) {
  if (!ce_ok(n, d, v, dtype) || !x || !w || !target || !loss || !keep || !ws || ldx < d || ldw < d || reduction < 0 || reduction > 2)
    return ISTNET_PN2_EINVAL;
  const hipStream_t st = (hipStream_t)stream;
  const bool direct = direct_w(d, dtype, w, ldw), split = dtype == ISTNET_VOCAB_F32;
  const Keep k = keep_plan(n, d, v, dtype, direct);
  const Forward f = forward_plan(k);
  char *kb = (char*)keep, *wb = (char*)ws;
  float* scal = (float*)(kb + k.scal);
  int* blocks = (int*)(wb + f.blocks);
  float *amax = (float*)(wb + f.amax), *packed_loss = (float*)(wb + f.loss), *row_loss = reduction == 0 ? loss : nullptr;
  uint16_t *xp = (uint16_t*)(kb + k.xp), *wp = (uint16_t*)(kb + k.wp);
  float *bias2 = (float*)(kb + k.bias2), *zt = (float*)(wb + f.zt);
  RowStat* stat = (RowStat*)(kb + k.stat);
  int *rowmap = (int*)(kb + k.rowmap), *inverse = (int*)(kb + k.inverse), *tgt = (int*)(kb + k.tgt);
  const int ax = split ? (int)std::min<long long>(256, (n + 3) / 4) : 0, aw = split ? (int)std::min<long long>(768, (v + 3ll) / 4) : 0;
  if (split)
    hipLaunchKernelGGL(ce_amax_kernel, dim3(ax + aw), dim3(256), 0, st, (int)n, v, d, (const float*)x, ldx, (const float*)w, ldw, target,
                       idx64, ignore, ax, amax);
  const int counted = n > 16384;      // up to here one workgroup counts the rows while it is at it
  if (counted)
    hipLaunchKernelGGL(ce_count_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, (int)n, target, idx64, ignore, blocks);
  hipLaunchKernelGGL(ce_plan_kernel, dim3(1), dim3(1024), 0, st, (int)n, counted, target, idx64, ignore, (int)split, ax, ax + aw, amax,
                     blocks, scal);
  const int xwgs = (int)((n + 255) / 256 * (256 / kPackRows));
  const int wwgs = direct ? (int)std::min<long long>(256, (k.vp + 255) / 256) : (int)std::min<long long>(2048, (v + 3ll) / 4);
  VOCAB_DISPATCH(dtype, T, {
    typedef Matrix<T> X;
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_pack_kernel<T, X::P>), dim3(xwgs + kPad / kPackRows + wwgs), dim3(256), 0, st, (int)n, v, d,
                       (int)k.kp, (int)k.vp, (const T*)x, ldx, (const T*)w, ldw, (const T*)bias, target, idx64, ignore, xwgs, !direct,
                       blocks, scal, xp, k.np * k.kp, wp, v * k.kp, bias2, rowmap, inverse, tgt, row_loss);
    const uint16_t* wd = direct ? (const uint16_t*)w : wp;
    const Operand A = {{wd, direct ? wd : wp + v * k.kp}, direct ? ldw : k.kp, v - 1, 0};
    const Operand B = {{xp, xp + (X::P - 1) * k.np * k.kp}, k.kp, (int)k.np - 1, 0};
    Epilogue e = {};
    e.scal = scal;
    e.bias2 = bias2;
    e.biased = bias != nullptr;
    e.target = tgt;
    e.part = (float2*)(wb + f.part);
    e.zt = zt;
    e.v = v;
    e.parts_ld = (int)k.np;
    const int tn = (int)((n + kNT - 1) / kNT);
    hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_gemm_kernel<typename X::M, X::LOGIT, 1, false, false, kMT, kNT, kLse, T>), dim3(f.tiles * tn),
                       dim3(256), 0, st, A, B, f.tiles, tn, (int)(k.kp / BK), 0, 1, 0, e);
  });
  hipLaunchKernelGGL(ce_finish_kernel, dim3((unsigned)(round_up(n, kPad) / 16)), dim3(256), 0, st, f.tiles, (int)k.np,
                     bias != nullptr, (const float2*)(wb + f.part), zt, tgt, rowmap, scal, stat, packed_loss, row_loss);
  if (reduction != 0)
    hipLaunchKernelGGL(ce_total_kernel, dim3(1), dim3(1024), 0, st, reduction == 1, packed_loss, scal, loss);
  return launch_status();
}

extern "C" int istnet_linear_ce_backward(long long n, int d, int v, int dtype, const void* x, long long ldx, const void* w, long long ldw,
                                         int has_bias, int reduction, const float* gout, void* keep, void* ws, void* dx, void* dw,
                                         void* db, void* stream) {
  if (!ce_ok(n, d, v, dtype) || !x || !w || !gout || !keep || !ws || ldx < d || ldw < d || reduction < 0 || reduction > 2)
    return ISTNET_PN2_EINVAL;
  const hipStream_t st = (hipStream_t)stream;
  const bool direct = direct_w(d, dtype, w, ldw);
  const Keep k = keep_plan(n, d, v, dtype, direct);
  const Backward b = backward_plan(k, n, d, v, dtype, reduction);
  char *kb = (char*)keep, *wb = (char*)ws;
  float* scal = (float*)(kb + k.scal);
  uint16_t *xp = (uint16_t*)(kb + k.xp), *wp = (uint16_t*)(kb + k.wp), *dz = (uint16_t*)(wb + b.dz);
  int *rowmap = (int*)(kb + k.rowmap), *inverse = (int*)(kb + k.inverse);
  const int tn = (int)((n + kNT - 1) / kNT), dt = (int)(b.ld / kMT);
  const bool weighted = reduction == 0, folded = weighted && dtype == ISTNET_VOCAB_F16, turned = dtype == ISTNET_VOCAB_BF16;
  if (weighted) hipLaunchKernelGGL(ce_gmax_kernel, dim3(1), dim3(1024), 0, st, gout, rowmap, scal);
  if (turned) {
    const int ax = (int)std::min<long long>(256, (n + 3) / 4), aw = (int)std::min<long long>(768, (v + 3ll) / 4);
    float* amax = (float*)(wb + b.amax);
    hipLaunchKernelGGL(ce_amax_packed_kernel, dim3(ax + aw), dim3(256), 0, st, (int)k.kp, (const bf16*)xp, scal, v, d,
                       (const bf16*)w, ldw, ax, amax);
    hipLaunchKernelGGL(ce_scales_kernel, dim3(1), dim3(1024), 0, st, ax, ax + aw, amax, scal);
  }
  VOCAB_DISPATCH(dtype, T, {
    typedef Matrix<T> X;
    typedef typename X::M M;
    constexpr int P = X::P, PD = X::PD;
    uint16_t* xb = xp;      // rows that dw is formed from
    if (dw && (turned || (weighted && !folded))) {
      xb = (uint16_t*)(wb + b.xb);
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_back_x_kernel<T, P>), dim3((unsigned)(round_up(n, kPad) / 4)), dim3(256), 0, st, d, (int)k.kp,
                         (const T*)x, ldx, weighted ? gout : nullptr, rowmap, scal, xb, k.np * k.kp);
    }
    const uint16_t* wd = direct ? (const uint16_t*)w : wp;
    const long long ldwd = direct ? ldw : k.kp, wplane = direct ? 0 : v * k.kp, xplane = (P - 1) * k.np * k.kp, dzp = k.np * b.piece;
    for (int piece = 0; piece < b.pieces; ++piece) {
      const int v0 = (int)(piece * b.piece), width = (int)std::min(b.piece, k.vp - v0), rows = std::min(width, v - v0);
      Epilogue e = {};
      e.scal = scal;
      e.bias2 = (float*)(kb + k.bias2);
      e.biased = has_bias;
      e.target = (int*)(kb + k.tgt);
      e.stat = (const RowStat*)(kb + k.stat);
      e.dz[0] = dz;
      e.dz[1] = dz + dzp;
      e.ld_dz = b.piece;
      e.rowmap = rowmap;
      e.weights = folded ? gout : nullptr;
      e.v = v;
      e.v0 = v0;
      const uint16_t* w0 = wd + v0 * ldwd;
      const Operand A = {{w0, w0 + (P - 1) * wplane}, ldwd, rows - 1, 0};
      const Operand B = {{xp, xp + xplane}, k.kp, (int)k.np - 1, 0};
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_gemm_kernel<M, X::LOGIT, PD, false, false, kMT, kNT, kDz, T>), dim3(width / kMT * tn),
                         dim3(256), 0, st, A, B, width / kMT, tn, (int)(k.kp / BK), 0, 1, 0, e);
      const Operand D = {{dz, dz + (PD - 1) * dzp}, b.piece, (int)k.np - 1, (int)b.piece / 8 - 1};
      if (dx) {
        Epilogue s = {};
        s.scal = scal;
        s.slab = (float*)(wb + b.dx_slab);
        s.slab_stride = b.dx_rows * b.ld;
        s.ld_slab = b.ld;
        s.accumulate = piece > 0;
        Operand Wt = {{w0, w0 + (P - 1) * wplane}, ldwd, rows - 1, (int)(direct ? d : k.kp) / 8 - 1};
        if (turned) {
          uint16_t* wf = (uint16_t*)(wb + b.wb);
          hipLaunchKernelGGL(ce_back_w_kernel, dim3(std::min((rows + 3) / 4, 2048)), dim3(256), 0, st, rows, d, (int)k.kp,
                             (const bf16*)w + v0 * ldw, ldw, scal, wf);
          Wt = {{wf, wf}, k.kp, rows - 1, (int)k.kp / 8 - 1};
        }
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_gemm_kernel<f16, X::GRAD, 1, true, false, kMT, kNT, kSlab, T>), dim3(dt * tn * b.dx_splits),
                           dim3(256), 0, st, Wt, D, dt, tn, (rows + BK - 1) / BK, b.dx_per, 1, 0, s);
      }
      if (dw) {
        Epilogue s = {};
        s.scal = scal;
        s.slab = (float*)(wb + b.dw_slab);
        s.slab_stride = b.dw_rows * b.ld;
        s.ld_slab = b.ld;
        T* dw0 = (T*)dw + (long long)v0 * d;
        s.out = dw0;
        s.out_rows = rows;
        s.d = d;
        s.reduction = reduction;
        s.gout = gout;
        const Operand Xt = {{xb, xb + xplane}, k.kp, (int)k.np - 1, (int)k.kp / 8 - 1};
        const int vt = (rows + kNT - 1) / kNT;
        if (b.dw_splits == 1) {
          hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_gemm_kernel<f16, X::GRAD, 1, true, true, kMT, kNT, kOut, T>), dim3(dt * vt), dim3(256), 0,
                             st, Xt, D, dt, vt, 0, 0, 0, 1, s);
        } else {
          hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_gemm_kernel<f16, X::GRAD, 1, true, true, kMT, kNT, kSlab, T>), dim3(dt * vt * b.dw_splits),
                             dim3(256), 0, st, Xt, D, dt, vt, 0, b.dw_per, 0, 1, s);
          hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_dw_kernel<T>), dim3((unsigned)(((long long)rows * ((d + 3) / 4) + 255) / 256)), dim3(256),
                             0, st, rows, d, b.dw_splits, s.slab, s.slab_stride, b.ld, gout, reduction, scal, dw0);
        }
      }
      if (db) {
        float* col = (float*)(wb + b.col);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_colsum_kernel<PD>), dim3((width + 511) / 512, kChunks / 4), dim3(256), 0, st, width, dz,
                           dz + (PD - 1) * dzp, b.piece, weighted && !folded ? gout : nullptr, rowmap, scal, kChunks, col);
        hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_db_kernel<T>), dim3((rows + 255) / 256), dim3(256), 0, st, rows, width, kChunks, col, gout,
                           reduction, folded, scal, (T*)db + v0);
      }
    }
    if (dx)
      hipLaunchKernelGGL(HIP_KERNEL_NAME(ce_dx_kernel<T>), dim3((unsigned)((n * ((d + 3) / 4) + 255) / 256)), dim3(256), 0, st, (int)n, d,
                         b.dx_splits, (const float*)(wb + b.dx_slab), b.dx_rows * b.ld, b.ld, inverse, gout, reduction, folded, scal,
                         (T*)dx);
  });
  return launch_status();
}
