// join_kernels.hip — what stands between two sublayers of a transformer block
// (gfx950 / MI355X):
//
//   n = Post(u) (or u) ;  y = scale * x + gate * n ;  h = Norm(y)
//
// Norm and Post are layer norms or root-mean-square norms; the gate is absent,
// one vector for all rows, one for each sample, or a whole tensor.
//
// Bound by HBM: the forward pass reads x, u and writes y, h; the backward pass
// reads x, u, dy, dh and writes dx, du, everything else of a row stays in
// registers.  A row belongs to one wave (D <= 1024) or one block (D <= 8192),
// at most 16 elements a lane.  Means and variances in fp32, the variance about
// the mean (two sums).  Both passes take y before its rounding: the backward
// one computes it again from x and u, which cost what reading y would.
//
// Sums over rows (weights, biases, gate): each block keeps its rows' sums in
// registers, writes them once, and a second kernel adds the blocks' parts in
// fixed order.  No atomics: results repeat bit for bit.
//
// bf16, 49152 rows of 768, one gate vector: forward 53 us (5.7 TB/s), backward
// 115 (3.9 TB/s), sums 5.  8192 rows of 4096 with both norms: 48, 77 and 4 us.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <cstdint>

#define JN_MAXD 8192

struct JoinArgs {
  const void *x, *u, *w, *b, *pw, *pb, *gate;
  void *y, *h;
  float *my, *ry, *mu, *ru;            // statistics of the rows
  const void *dy, *dh;                 // either may be null
  void *dx, *du, *dgate;               // dgate: whole-tensor gate only
  float* part;                         // [blocks][slots][D]
  int slot_w, slot_b, slot_pw, slot_pb, slot_g, slots;
  int64_t rows;                        // of a group
  int nb;                              // blocks of a group
  int D;
  int layer;                           // 1: mean subtracted
  int gate_kind;                       // 0 none, 1 one vector a group, 2 whole
  int64_t gate_step;                   // from one group's vector to the next
  float scale, eps, invD;
};

// 16 bytes at any address that is a multiple of two: rows of odd length are
// read as wide as others.
typedef uint32_t jn_u4 __attribute__((ext_vector_type(4)));
typedef jn_u4 jn_u4_any __attribute__((aligned(2)));

__device__ __forceinline__ float jn_f(float v) { return v; }
__device__ __forceinline__ float jn_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T jn_t(float v);
template <> __device__ __forceinline__ float jn_t(float v) { return v; }
template <> __device__ __forceinline__ __hip_bfloat16 jn_t(float v) { return __float2bfloat16(v); }

// A lane's share of a row: EPT elements in 16-byte vectors, TPR lanes a row.
template <typename T, int EPT, int TPR>
struct JnRow {
  static constexpr int VEC = 16 / sizeof(T), CH = EPT / VEC;
  jn_u4 c[CH];
  __device__ __forceinline__ static int at(int j, int lane) {
    return ((j / VEC) * TPR + lane) * VEC + j % VEC;
  }
  // past the row's end, and where there is no tensor: zeros
  __device__ __forceinline__ void load(const void* p, int64_t off, int lane, int D) {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e = (i * TPR + lane) * VEC;
      const T* from = (const T*)p + off + e;
      if (p != nullptr && e + VEC <= D) {
        c[i] = *(const jn_u4_any*)from;
      } else {
        c[i] = (jn_u4)(0u);
        if (p != nullptr && e < D)  // the end of a row of odd length
#pragma unroll
          for (int j = 0; j < VEC - 1; ++j)
            if (e + j < D) put(i * VEC + j, from[j]);
      }
    }
  }
  __device__ __forceinline__ void store(void* p, int64_t off, int lane, int D) const {
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int e = (i * TPR + lane) * VEC;
      T* to = (T*)p + off + e;
      if (e + VEC <= D) {
        *(jn_u4_any*)to = c[i];
      } else if (e < D) {
#pragma unroll
        for (int j = 0; j < VEC - 1; ++j)
          if (e + j < D) to[j] = of(i * VEC + j);
      }
    }
  }
  __device__ __forceinline__ T of(int j) const {
    if constexpr (sizeof(T) == 4) return __builtin_bit_cast(T, (uint32_t)c[j / 4][j % 4]);
    else return __builtin_bit_cast(T, (uint16_t)(c[j / 8][j % 8 / 2] >> (16 * (j & 1))));
  }
  __device__ __forceinline__ void put(int j, T v) {
    if constexpr (sizeof(T) == 4) {
      c[j / 4][j % 4] = __builtin_bit_cast(uint32_t, v);
    } else {
      const uint32_t b = __builtin_bit_cast(uint16_t, v), w = c[j / 8][j % 8 / 2];
      c[j / 8][j % 8 / 2] = j & 1 ? (w & 0xffffu) | (b << 16) : (w & 0xffff0000u) | b;
    }
  }
  __device__ __forceinline__ float get(int j) const { return jn_f(of(j)); }
  __device__ __forceinline__ void set(int j, float v) { put(j, jn_t<T>(v)); }
};

// The sum over a wave, in all lanes, without LDS: rotations within 16 lanes,
// then rows of 16 and halves swapped.  All lanes add the same pairs: one value.
__device__ __forceinline__ float jn_wave_sum(float x) {
#define JN_ROR(n)                                                              \
  x += __uint_as_float(__builtin_amdgcn_update_dpp(                            \
      0, __float_as_uint(x), 0x120 + (n), 0xf, 0xf, false))
  JN_ROR(8);
  JN_ROR(4);
  JN_ROR(2);
  JN_ROR(1);
#undef JN_ROR
  auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Sums over the lanes of a row.  `red`: room for two rounds of a block's waves.
template <int TPR>
__device__ __forceinline__ float2 jn_sum2(float a, float b, float2* red, int& turn) {
  a = jn_wave_sum(a);
  b = jn_wave_sum(b);
  if (TPR == 64) return make_float2(a, b);
  constexpr int W = TPR / 64;
  float2* r = red + turn * W;
  turn ^= 1;
  if ((threadIdx.x & 63) == 0) r[threadIdx.x >> 6] = make_float2(a, b);
  __syncthreads();
  a = b = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    a += r[i].x;
    b += r[i].y;
  }
  return make_float2(a, b);
}

template <int TPR>
__device__ __forceinline__ float jn_sum(float a, float2* red, int& turn) {
  return jn_sum2<TPR>(a, 0.0f, red, turn).x;
}

// mean (0 for the rms kind) and 1/sqrt(variance + eps) of a row in f
template <int EPT, int TPR, typename R>
__device__ __forceinline__ void jn_stats(const JoinArgs& a, const float* f, int lane,
                                         float& mean, float& rstd, float2* red, int& turn) {
  mean = 0.0f;
  if (a.layer) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < EPT; ++j) s += f[j];
    mean = jn_sum<TPR>(s, red, turn) * a.invD;
  }
  float q = 0.0f;
#pragma unroll
  for (int j = 0; j < EPT; ++j) {
    const float d = R::at(j, lane) < a.D ? f[j] - mean : 0.0f;
    q = fmaf(d, d, q);
  }
  q = jn_sum<TPR>(q, red, turn);
  rstd = 1.0f / sqrtf(fmaf(q, a.invD, a.eps));
}

// Rows of 64 lanes stand four to a block, others are a block each.
template <int TPR>
struct JnBlock {
  static constexpr int N = TPR < 128 ? 256 : TPR, ROWS = N / TPR;
};

// GATE: 0 none, 1 a vector, 2 x's shape
template <typename T, int EPT, int TPR, bool POST, int GATE>
__global__ void __launch_bounds__(JnBlock<TPR>::N) k_join_fwd(const JoinArgs a) {
  using R = JnRow<T, EPT, TPR>;
  constexpr int RPB = JnBlock<TPR>::ROWS;
  __shared__ float2 red[2 * (TPR / 64)];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int group = blockIdx.x / a.nb, blk = blockIdx.x - group * a.nb;
  const int D = a.D;
  int turn = 0;
  R w, b, pw, pb, gate;
  w.load(a.w, 0, lane, D);
  b.load(a.b, 0, lane, D);
  if (POST) {
    pw.load(a.pw, 0, lane, D);
    pb.load(a.pb, 0, lane, D);
  }
  if (GATE == 1) gate.load(a.gate, group * a.gate_step, lane, D);
  const int64_t step = (int64_t)a.nb * RPB;
  int64_t i = (int64_t)blk * RPB + sub;
  R xn, un, gn;  // the next row's, on their way
  auto load = [&](int64_t at) {
    const int64_t off = (group * a.rows + at) * D;
    xn.load(a.x, off, lane, D);
    un.load(a.u, off, lane, D);
    if (GATE == 2) gn.load(a.gate, off, lane, D);
  };
  if (i < a.rows) load(i);
  for (; i < a.rows; i += step) {
    const int64_t row = group * a.rows + i, off = row * D;
    R x = xn, u = un;
    if (GATE == 2) gate = gn;
    if (i + step < a.rows) load(i + step);
    float f[EPT];
#pragma unroll
    for (int j = 0; j < EPT; ++j) f[j] = u.get(j);
    if (POST) {
      float m, r;
      jn_stats<EPT, TPR, R>(a, f, lane, m, r, red, turn);
      if (lane == 0) {
        a.mu[row] = m;
        a.ru[row] = r;
      }
#pragma unroll
      for (int j = 0; j < EPT; ++j) f[j] = fmaf((f[j] - m) * r, pw.get(j), pb.get(j));
    }
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      const float g = GATE ? gate.get(j) * f[j] : f[j];
      f[j] = R::at(j, lane) < D ? fmaf(a.scale, x.get(j), g) : 0.0f;
      x.set(j, f[j]);
    }
    x.store(a.y, off, lane, D);
    float m, r;
    jn_stats<EPT, TPR, R>(a, f, lane, m, r, red, turn);
    if (lane == 0) {
      a.my[row] = m;
      a.ry[row] = r;
    }
#pragma unroll
    for (int j = 0; j < EPT; ++j) u.set(j, fmaf((f[j] - m) * r, w.get(j), b.get(j)));
    u.store(a.h, off, lane, D);
  }
}

// This block's sums of one slot, to its part: the rows in hand are added
// through LDS in fixed order.
template <int EPT, int TPR, typename R>
__device__ __forceinline__ void jn_part(const JoinArgs& a, const float* acc, int slot,
                                        int lane, int sub, float* lds) {
  constexpr int RPB = JnBlock<TPR>::ROWS;
  float* out = a.part + ((int64_t)blockIdx.x * a.slots + slot) * a.D;
  if (RPB == 1) {
#pragma unroll
    for (int j = 0; j < EPT; ++j)
      if (R::at(j, lane) < a.D) out[R::at(j, lane)] = acc[j];
    return;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < EPT; ++j) lds[sub * EPT * TPR + R::at(j, lane)] = acc[j];
  __syncthreads();
  for (int e = threadIdx.x; e < a.D; e += JnBlock<TPR>::N) {
    float s = 0.0f;
#pragma unroll
    for (int k = 0; k < RPB; ++k) s += lds[k * EPT * TPR + e];
    out[e] = s;
  }
}

// A lane's sums over the rows of its block, in registers or in its own places
// in LDS: 16 bytes a lane, so that a wave's accesses meet in no bank.  No other
// lane looks at them: no barrier.
template <int EPT, int TPR, bool LDS>
struct JnAcc {
  float r[LDS ? 1 : EPT];
  float4* at;
  static constexpr int BYTES = LDS ? EPT * TPR * 4 : 0;
  __device__ __forceinline__ void clear(char* lds, int lane) {
    at = (float4*)lds + lane;
#pragma unroll
    for (int j = 0; j < EPT; j += 4) {
      if constexpr (LDS) at[j / 4 * TPR] = make_float4(0, 0, 0, 0);
      else r[j] = r[j + 1] = r[j + 2] = r[j + 3] = 0.0f;
    }
  }
  // sum j becomes f(j, sum j)
  template <typename F> __device__ __forceinline__ void add(F f) {
#pragma unroll
    for (int j = 0; j < EPT; j += 4) {
      if constexpr (LDS) {
        float4 s = at[j / 4 * TPR];
        s.x = f(j, s.x);
        s.y = f(j + 1, s.y);
        s.z = f(j + 2, s.z);
        s.w = f(j + 3, s.w);
        at[j / 4 * TPR] = s;
      } else {
#pragma unroll
        for (int k = j; k < j + 4; ++k) r[k] = f(k, r[k]);
      }
    }
  }
  __device__ __forceinline__ void get(float* to) {
    add([&](int j, float s) { return to[j] = s; });
  }
};

template <typename T, int EPT, int TPR, bool POST, int GATE>
__global__ void __launch_bounds__(JnBlock<TPR>::N) k_join_bwd(const JoinArgs a) {
  using R = JnRow<T, EPT, TPR>;
  constexpr int RPB = JnBlock<TPR>::ROWS;
  __shared__ float2 red[2 * (TPR / 64)];
  __shared__ float lds[RPB == 1 ? 1 : RPB * EPT * TPR];
  // Five sums of 16 elements do not fit beside a row of 512 lanes: with Post
  // they went to scratch (4096 rows of 8192, a gate vector: 364 us, 126 so).
  constexpr bool FAR = POST && EPT == 16 && TPR == 512;
  using Near = JnAcc<EPT, TPR, false>;
  using Acc = JnAcc<EPT, TPR, FAR>;
  __shared__ __attribute__((aligned(16))) char sums[FAR ? (3 + (GATE == 1)) * Acc::BYTES : 16];
  const int lane = threadIdx.x % TPR, sub = threadIdx.x / TPR;
  const int group = blockIdx.x / a.nb, blk = blockIdx.x - group * a.nb;
  const int D = a.D;
  int turn = 0;
  R w, pw, pb, gate;
  Near aw;
  Acc ab, ag, apw, apb;
  aw.clear(nullptr, lane);
  ab.clear(sums, lane);
  if (POST) {
    apw.clear(sums + Acc::BYTES, lane);
    apb.clear(sums + 2 * Acc::BYTES, lane);
  }
  if (GATE == 1) ag.clear(sums + 3 * Acc::BYTES, lane);
  w.load(a.w, 0, lane, D);
  if (POST) {
    pw.load(a.pw, 0, lane, D);
    pb.load(a.pb, 0, lane, D);
  }
  if (GATE == 1) gate.load(a.gate, group * a.gate_step, lane, D);
  const int64_t step = (int64_t)a.nb * RPB;
  int64_t i = (int64_t)blk * RPB + sub;
  R xn, un, dyn, dhn, gn;  // the next row's, on their way
  float m1n = 0.0f, r1n = 0.0f, m2n = 0.0f, r2n = 1.0f;
  auto load = [&](int64_t at) {
    const int64_t row = group * a.rows + at, off = row * D;
    m1n = a.my[row];
    r1n = a.ry[row];
    if (POST) {
      m2n = a.mu[row];
      r2n = a.ru[row];
    }
    xn.load(a.x, off, lane, D);
    dhn.load(a.dh, off, lane, D);
    dyn.load(a.dy, off, lane, D);
    un.load(a.u, off, lane, D);
    if (GATE == 2) gn.load(a.gate, off, lane, D);
  };
  // the longest rows have no registers to hold another one
  constexpr bool AHEAD = TPR < 512 || EPT < 16;
  if (AHEAD && i < a.rows) load(i);
  for (; i < a.rows; i += step) {
    const int64_t row = group * a.rows + i, off = row * D;
    if (!AHEAD) load(i);
    R x = xn, u = un, dy = dyn, dh = dhn;
    if (GATE == 2) gate = gn;
    const float m1 = m1n, r1 = r1n, m2 = m2n, r2 = r2n;
    if (AHEAD && i + step < a.rows) load(i + step);
    float t[EPT];  // the whole gradient of y
    float y[EPT];  // y's normed value
    float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      float n = u.get(j);
      if (POST) n = fmaf((n - m2) * r2, pw.get(j), pb.get(j));
      if (GATE) n *= gate.get(j);
      const float xh = (fmaf(a.scale, x.get(j), n) - m1) * r1, g = dh.get(j);
      y[j] = xh;
      t[j] = g * w.get(j);
      s1 += t[j];
      s2 = fmaf(t[j], xh, s2);
    }
    aw.add([&](int j, float s) { return fmaf(dh.get(j), y[j], s); });
    ab.add([&](int j, float s) { return s + dh.get(j); });
    float2 s = jn_sum2<TPR>(s1, s2, red, turn);
    float c1 = a.layer ? s.x * a.invD : 0.0f, c2 = s.y * a.invD;
#pragma unroll
    for (int j = 0; j < EPT; ++j) {
      t[j] = fmaf(r1, fmaf(-y[j], c2, t[j] - c1), dy.get(j));
      x.set(j, a.scale * t[j]);
    }
    x.store(a.dx, off, lane, D);
    s1 = s2 = 0.0f;
    auto uh = [&](int j) { return POST ? (u.get(j) - m2) * r2 : u.get(j); };
    auto dg = [&](int j) {
      return t[j] * (POST ? fmaf(uh(j), pw.get(j), pb.get(j)) : uh(j));
    };
    if (GATE == 1) ag.add([&](int j, float s) { return s + dg(j); });
    if (GATE) {
#pragma unroll
      for (int j = 0; j < EPT; ++j) {
        if (GATE == 2) dy.set(j, dg(j));
        t[j] *= gate.get(j);
      }
    }
    if (POST) {
      apw.add([&](int j, float s) { return fmaf(t[j], uh(j), s); });
      apb.add([&](int j, float s) { return s + t[j]; });
#pragma unroll
      for (int j = 0; j < EPT; ++j) {
        t[j] *= pw.get(j);
        s1 += t[j];
        s2 = fmaf(t[j], uh(j), s2);
      }
    }
    if (GATE == 2 && a.dgate) dy.store(a.dgate, off, lane, D);
    if (POST) {
      s = jn_sum2<TPR>(s1, s2, red, turn);
      c1 = a.layer ? s.x * a.invD : 0.0f;
      c2 = s.y * a.invD * r2;
#pragma unroll
      for (int j = 0; j < EPT; ++j) t[j] = r2 * fmaf(m2 - u.get(j), c2, t[j] - c1);
    }
#pragma unroll
    for (int j = 0; j < EPT; ++j) u.set(j, t[j]);
    u.store(a.du, off, lane, D);
  }
  // lanes past the row's end held w = pw = 0 and are not written
  auto part = [&](auto& acc, int slot) {
    if (slot < 0) return;
    float f[EPT];
    acc.get(f);
    jn_part<EPT, TPR, R>(a, f, slot, lane, sub, lds);
  };
  part(aw, a.slot_w);
  part(ab, a.slot_b);
  if (GATE == 1) part(ag, a.slot_g);
  if (POST) {
    part(apw, a.slot_pw);
    part(apb, a.slot_pb);
  }
}

struct JoinSums {
  void* out[5];     // by slot
  const float* part;
  int slots, slot_g, groups, nb, D;
  int from;         // first of the sums that this launch takes
};

// out[slot][d] = sum over blocks of part[block][slot][d]; the gate's slot one
// sum for each group.  32 columns and 32 ranges of blocks a thread block.
template <typename T>
__global__ void __launch_bounds__(1024) k_join_sum(const JoinSums a) {
  __shared__ float lds[32][33];
  const int col = threadIdx.x & 31, rg = threadIdx.x >> 5;
  const int d = blockIdx.x * 32 + col;
  // y: first the slots summed over all blocks, then the gate's groups
  const bool each = a.slot_g >= 0 && a.groups > 1;
  const int whole = a.slots - (each ? 1 : 0), y = a.from + (int)blockIdx.y;
  int slot, first, count, g = 0;
  if (y < whole) {
    slot = y;
    if (each && slot >= a.slot_g) ++slot;
    first = 0;
    count = a.groups * a.nb;
  } else {
    slot = a.slot_g;
    g = y - whole;
    first = g * a.nb;
    count = a.nb;
  }
  float s = 0.0f;
  if (d < a.D) {
    const float* p = a.part + ((int64_t)first * a.slots + slot) * a.D + d;
    const int64_t step = (int64_t)a.slots * a.D;
#pragma unroll 8
    for (int i = rg; i < count; i += 32) s += p[i * step];
  }
  lds[rg][col] = s;
  __syncthreads();
  // the ranges of a column in one half wave
  s = lds[col][rg];
#pragma unroll
  for (int k = 16; k > 0; k >>= 1) s += __shfl_xor(s, k, 32);
  const int e = blockIdx.x * 32 + rg;
  if (col == 0 && e < a.D) ((T*)a.out[slot])[(int64_t)g * a.D + e] = jn_t<T>(s);
}

// ---------------------------------------------------------------------------

// Lanes and elements a lane for a row of D.  Eight elements a lane keep the
// backward kernel with Post, or in fp32, at two or three waves a SIMD (16 took
// 256 registers and left one); else 16 fit, with two, and one wave a row beats
// two (49152 rows of 768 backward: 116 us, as 128 lanes of 8 167).  A lane's
// vectors are 16 bytes wide even where that leaves a quarter of the lanes idle.
struct JnShape {
  int ept, tpr;
};
static constexpr JnShape jn_shape(int64_t D, bool lean) {
  if (D <= 512) return {8, 64};
  if (D <= 1024) return lean ? JnShape{8, 128} : JnShape{16, 64};
  if (D <= 2048) return {8, 256};
  if (D <= 4096) return lean ? JnShape{8, 512} : JnShape{16, 256};
  return {16, 512};
}

// DMAX: the longest row of the shape
template <typename T, bool BWD, bool POST, int GATE, int DMAX>
static void jn_go(hipStream_t s, int grid, const JoinArgs& a) {
  constexpr JnShape h = jn_shape(DMAX, BWD && (POST || sizeof(T) == 4));
  constexpr int N = JnBlock<h.tpr>::N;
  if constexpr (BWD)
    hipLaunchKernelGGL((k_join_bwd<T, h.ept, h.tpr, POST, GATE>), dim3(grid), dim3(N), 0, s, a);
  else
    hipLaunchKernelGGL((k_join_fwd<T, h.ept, h.tpr, POST, GATE>), dim3(grid), dim3(N), 0, s, a);
}

template <typename T, bool BWD, bool POST, int GATE>
static void jn_launch(hipStream_t s, int grid, const JoinArgs& a) {
  if (a.D <= 512) jn_go<T, BWD, POST, GATE, 512>(s, grid, a);
  else if (a.D <= 1024) jn_go<T, BWD, POST, GATE, 1024>(s, grid, a);
  else if (a.D <= 2048) jn_go<T, BWD, POST, GATE, 2048>(s, grid, a);
  else if (a.D <= 4096) jn_go<T, BWD, POST, GATE, 4096>(s, grid, a);
  else jn_go<T, BWD, POST, GATE, JN_MAXD>(s, grid, a);
}

template <typename T, bool BWD>
static void jn_pick(hipStream_t s, int grid, const JoinArgs& a) {
  const bool post = a.pw != nullptr;
  if (post && a.gate_kind == 2) jn_launch<T, BWD, true, 2>(s, grid, a);
  else if (post && a.gate_kind == 1) jn_launch<T, BWD, true, 1>(s, grid, a);
  else if (post) jn_launch<T, BWD, true, 0>(s, grid, a);
  else if (a.gate_kind == 2) jn_launch<T, BWD, false, 2>(s, grid, a);
  else if (a.gate_kind == 1) jn_launch<T, BWD, false, 1>(s, grid, a);
  else jn_launch<T, BWD, false, 0>(s, grid, a);
}

// Blocks of a group.  Backward 2048 waves: what the registers of most forms let
// be on the chip at once (two a SIMD); more would only write more parts.  Rows of
// at most 512 without Post leave room for three to five a SIMD, which 4096 waves
// use at 256 elements (196608 rows: 294 us with 2048, 184 with 4096) and not at
// 512 (98304 rows: 117 and 125; with Post 118 and 125).  Forward 4096 waves: each
// reads the weights once (49152 rows of 768: 62 us with 8192, 58 with 4096).
// Rows of 256 lanes with Post wait at more barriers and want 8192 (8192 rows of
// 4096: 59 us with 4096, 55 with 8192; 16384 of 1536: 54 and 48), without Post
// or with 512 lanes they do not (16384 of 2048: 53 and 54; 4096 of 8192 with
// Post: 61 and 65).
static int64_t jn_blocks(int64_t groups, int64_t rows, int64_t D, bool lean, bool post,
                         bool backward) {
  const JnShape h = jn_shape(D, lean && backward);
  const int64_t rpb = h.tpr < 128 ? 256 / h.tpr : 1;
  const int64_t waves = h.tpr < 128 ? 4 : h.tpr / 64;
  const int64_t most = (backward ? 2048 : post && h.tpr == 256 ? 8192 : 4096) / waves / groups;
  int64_t nb = (rows + rpb - 1) / rpb;
  if (nb > most) nb = most;
  return nb < 1 ? 1 : nb;
}

extern "C" int64_t ps_join_blocks(int64_t groups, int64_t rows, int64_t D, int post,
                                  int bf16) {
  return jn_blocks(groups, rows, D, post || !bf16, post, true);
}

static int jn_check(const JoinArgs& a, int64_t groups) {
  // a launch holds fewer than 2^32 threads, 512 a block at most
  if (a.D < 1 || a.D > JN_MAXD || groups * a.nb >= 1 << 23) return 9003;
  return 0;
}

// t: x, u, w, b, pw, pb, gate, y, h;  stats: my, ry, mu, ru
extern "C" int ps_join_fwd(void* stream, void* const* t, float* const* stats,
                           int bf16, int64_t groups, int64_t rows, int64_t D,
                           int layer, int gate_kind, int64_t gate_step,
                           float scale, float eps) {
  if (groups <= 0 || rows <= 0) return 0;
  JoinArgs a{};
  a.x = t[0]; a.u = t[1]; a.w = t[2]; a.b = t[3]; a.pw = t[4]; a.pb = t[5];
  a.gate = t[6]; a.y = t[7]; a.h = t[8];
  a.my = stats[0]; a.ry = stats[1]; a.mu = stats[2]; a.ru = stats[3];
  a.rows = rows; a.D = (int)D; a.layer = layer; a.gate_kind = gate_kind;
  a.gate_step = gate_step; a.scale = scale; a.eps = eps; a.invD = 1.0f / (float)D;
  a.nb = (int)jn_blocks(groups, rows, D, false, a.pw != nullptr, false);
  if (int e = jn_check(a, groups)) return e;
  const int grid = (int)(groups * a.nb);
  if (bf16) jn_pick<__hip_bfloat16, false>((hipStream_t)stream, grid, a);
  else jn_pick<float, false>((hipStream_t)stream, grid, a);
  return (int)hipGetLastError();
}

// t: u, w, pw, pb, gate, x, dy, dh, dx, du, dgate (whole tensor);
// sums: dw, db, dgate (vectors), dpw, dpb — null where not wanted.
extern "C" int ps_join_bwd(void* stream, void* const* t, float* const* stats,
                           void* const* sums, float* part, int bf16,
                           int64_t groups, int64_t rows, int64_t D, int layer,
                           int gate_kind, int64_t gate_step, float scale) {
  if (groups <= 0 || rows <= 0) return 0;
  JoinArgs a{};
  a.u = t[0]; a.w = t[1]; a.pw = t[2]; a.pb = t[3]; a.gate = t[4]; a.x = t[5];
  a.dy = t[6]; a.dh = t[7]; a.dx = t[8]; a.du = t[9]; a.dgate = t[10];
  a.my = stats[0]; a.ry = stats[1]; a.mu = stats[2]; a.ru = stats[3];
  a.part = part;
  a.rows = rows; a.D = (int)D; a.layer = layer; a.gate_kind = gate_kind;
  a.gate_step = gate_step; a.scale = scale; a.invD = 1.0f / (float)D;
  a.nb = (int)ps_join_blocks(groups, rows, D, a.pw != nullptr, bf16);
  if (int e = jn_check(a, groups)) return e;
  JoinSums q{};
  int* slot[5] = {&a.slot_w, &a.slot_b, &a.slot_g, &a.slot_pw, &a.slot_pb};
  for (int i = 0; i < 5; ++i) {
    *slot[i] = sums[i] ? a.slots : -1;
    if (sums[i]) q.out[a.slots++] = sums[i];
  }
  const int grid = (int)(groups * a.nb);
  hipStream_t s = (hipStream_t)stream;
  if (bf16) jn_pick<__hip_bfloat16, true>(s, grid, a);
  else jn_pick<float, true>(s, grid, a);
  if (int e = (int)hipGetLastError()) return e;
  if (a.slots == 0) return 0;
  q.part = part; q.slots = a.slots; q.slot_g = a.slot_g;
  q.groups = (int)groups; q.nb = a.nb; q.D = (int)D;
  const int gy = a.slots + (a.slot_g >= 0 && groups > 1 ? (int)groups - 1 : 0);
  // a grid has at most 65535 rows and here, with up to 256 columns of 1024
  // threads, fewer than 2^32 threads: more samples' gates take several launches
  constexpr int MOST = 1 << 13;
  for (; q.from < gy; q.from += MOST) {
    const dim3 sg((unsigned)((D + 31) / 32),
                  (unsigned)(gy - q.from < MOST ? gy - q.from : MOST));
    if (bf16) hipLaunchKernelGGL((k_join_sum<__hip_bfloat16>), sg, dim3(1024), 0, s, q);
    else hipLaunchKernelGGL((k_join_sum<float>), sg, dim3(1024), 0, s, q);
  }
  return (int)hipGetLastError();
}
