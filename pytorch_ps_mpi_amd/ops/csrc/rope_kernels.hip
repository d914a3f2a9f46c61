// rope_kernels.hip — rotary positions with several axes (gfx950 / MI355X).
//
// A head's first 2P elements are P pairs; each pair belongs to one axis (time,
// height, width) and turns by  position[axis] * freq[pair]:
//   (a, b) -> (a cos - b sin, a sin + b cos);   backward: the turn by -angle.
// Elements from 2P on pass through.
//
// The angle is taken in 64 bits as a number of revolutions, of which only the
// fraction goes on (a position of a million in 32 bits would be 0.06 rad off);
// it is computed once for a token and pair and used by all heads through LDS.
// Bound by HBM: q and k are read once and written once.  The frequencies
// travel in the kernel's arguments: no table lives on the device.  25216 tokens
// of 24 heads of 64, 155 MB: 35 us, 4.4 TB/s.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <cstdint>

#define RP_BLOCK 256
#define RP_MAXP 256
#define RP_TOK 4

struct RopeTensor {
  const void* x;
  void* y;            // contiguous [B, N, H, D]
  int64_t sB, sN, sH; // strides of x in elements
  int H;
};

struct RopeArgs {
  RopeTensor t[2];    // q, k
  const void* pos;
  int64_t pA, pB, pN; // strides of pos
  int pos64;
  int64_t rows;       // B * N
  int64_t first;      // first row of this launch
  int N, D, P;
  int start[4];       // first pair of axis 1, 2, 3 (P where there is none)
  float sign;         // -1: backward
  double rev[RP_MAXP];// revolutions for a position of 1
};

template <typename T> __device__ __forceinline__ float rp_f(T v) { return (float)v; }
template <> __device__ __forceinline__ float rp_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float rp_f(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T rp_t(float v) { return (T)v; }
template <> __device__ __forceinline__ __hip_bfloat16 rp_t(float v) { return __float2bfloat16(v); }
template <> __device__ __forceinline__ __half rp_t(float v) { return __float2half(v); }

// One way of rounding, whichever lane computes it.
template <typename T>
__device__ __forceinline__ void rp_turn(T& a, T& b, float x, float y, float2 k) {
#pragma clang fp contract(off)
  a = rp_t<T>(__builtin_fmaf(x, k.x, -(y * k.y)));
  b = rp_t<T>(__builtin_fmaf(x, k.y, y * k.x));
}

// 16 bytes at any address that is a multiple of two: odd numbers of pairs,
// strides and offsets are read as wide as others.
typedef uint32_t rp_u4 __attribute__((ext_vector_type(4)));
typedef rp_u4 rp_u4_any __attribute__((aligned(2)));
template <typename T> struct RpVec {
  static constexpr int N = 16 / sizeof(T);
  T v[N];
  // `n` elements, all of them in one access
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= N) {
      const rp_u4 u = *(const rp_u4_any*)p;
      __builtin_memcpy(v, &u, 16);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) v[j] = j < n ? p[j] : rp_t<T>(0.0f);
    }
  }
  __device__ __forceinline__ void store(T* p, int n) const {
    if (n >= N) {
      rp_u4 u;
      __builtin_memcpy(&u, v, 16);
      *(rp_u4_any*)p = u;
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (j < n) p[j] = v[j];
    }
  }
};

__device__ __forceinline__ void rp_angles(const RopeArgs& a, int64_t row0,
                                          int toks, float2* cs) {
  for (int i = threadIdx.x; i < toks * a.P; i += RP_BLOCK) {
    const int t = i / a.P, p = i - t * a.P;
    const int64_t row = row0 + t;
    const int64_t b = row / a.N, n = row - b * a.N;
    const int axis = (p >= a.start[0]) + (p >= a.start[1]) + (p >= a.start[2]);
    const int64_t at = axis * a.pA + b * a.pB + n * a.pN;
    const double pos = a.pos64 ? (double)((const int64_t*)a.pos)[at]
                               : (double)((const int32_t*)a.pos)[at];
    const double r = pos * a.rev[p];
    float s, c;
    sincospif((float)(2.0 * (r - rint(r))), &s, &c);
    cs[i] = make_float2(c, a.sign * s);
  }
}

// An item is a vector of V elements.  Half-split: item c holds pairs cV and on,
// that is two vectors P apart; behind them the items that pass through.
// Interleaved: elements cV and on, of which those before 2P turn.
//
// A range that is no multiple of V ends in a whole vector as well, moved back
// over its neighbour: both write the same values there, and inputs and outputs
// share no memory.  Single elements are for ranges shorter than a vector.
// 21518 tokens of 24 heads of 96, 25 interleaved pairs, 198 MB: 54 us, with the
// ends element by element 109.
// The first element of item i of a range of n.
template <int V> __device__ __forceinline__ int rp_at(int i, int n) {
  return n >= V ? min(i * V, n - V) : i * V;
}
template <typename T, bool INTER>
__global__ void __launch_bounds__(RP_BLOCK) k_rope(const RopeArgs a) {
  extern __shared__ float2 cs[];
  constexpr int V = RpVec<T>::N;
  const int64_t row0 = a.first + (int64_t)blockIdx.x * RP_TOK;
  const int toks = (int)min((int64_t)RP_TOK, a.rows - row0);
  rp_angles(a, row0, toks, cs);
  __syncthreads();
  const int P = a.P, D = a.D;
  const int turn = ((INTER ? D : P) + V - 1) / V;
  const int per = turn + (INTER ? 0 : (D - 2 * P + V - 1) / V);
  const int heads = a.t[0].H + a.t[1].H;
  const int total = toks * heads * per;
  for (int i = threadIdx.x; i < total; i += RP_BLOCK) {
    const int th = i / per, c = i - th * per;
    const int t = th / heads;
    int h = th - t * heads;
    const bool isk = h >= a.t[0].H;
    const RopeTensor& w = a.t[isk];
    if (isk) h -= a.t[0].H;
    const int64_t row = row0 + t;
    const int64_t b = row / a.N, n = row - b * a.N;
    const T* x = (const T*)w.x + b * w.sB + n * w.sN + h * w.sH;
    T* y = (T*)w.y + (row * w.H + h) * D;
    const float2* tc = cs + t * P;
    RpVec<T> u, v;
    if (c >= turn) {
      const int e = 2 * P + rp_at<V>(c - turn, D - 2 * P);
      u.load(x + e, D - e);
      u.store(y + e, D - e);
    } else if (INTER) {
      // moved back only by whole pairs
      const int e = D % 2 ? c * V : rp_at<V>(c, D);
      u.load(x + e, D - e);
#pragma unroll
      for (int j = 0; j < V; j += 2) {
        const int p = e / 2 + j / 2;
        const float2 k = tc[min(p, P - 1)];
        const float va = rp_f(u.v[j]), vb = rp_f(u.v[j + 1]);
        if (p < P) {
          rp_turn(u.v[j], u.v[j + 1], va, vb, k);
        }
      }
      u.store(y + e, D - e);
    } else {
      const int e = rp_at<V>(c, P);
      u.load(x + e, P - e);
      v.load(x + P + e, P - e);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float2 k = tc[min(e + j, P - 1)];
        const float va = rp_f(u.v[j]), vb = rp_f(v.v[j]);
        rp_turn(u.v[j], v.v[j], va, vb, k);
      }
      u.store(y + e, P - e);
      v.store(y + P + e, P - e);
    }
  }
}

template <typename T>
static void rp_launch(hipStream_t s, RopeArgs a, bool inter) {
  // a launch holds fewer than 2^32 threads: more rows take several
  constexpr int64_t MOST = 1 << 23;
  const size_t lds = (size_t)RP_TOK * a.P * sizeof(float2);
  for (a.first = 0; a.first < a.rows; a.first += MOST * RP_TOK) {
    const int64_t left = (a.rows - a.first + RP_TOK - 1) / RP_TOK;
    const dim3 grid((unsigned)(left < MOST ? left : MOST));
    if (inter)
      hipLaunchKernelGGL((k_rope<T, true>), grid, dim3(RP_BLOCK), lds, s, a);
    else
      hipLaunchKernelGGL((k_rope<T, false>), grid, dim3(RP_BLOCK), lds, s, a);
  }
}

// strides: q's B, N, H, k's B, N, H, pos's axis, B, N.  dtype: 0 bf16, 1 fp16,
// 2 fp32.  rev: revolutions a position for each of P pairs (host memory).
extern "C" int ps_rope(void* stream, const void* q, const void* k, void* yq,
                       void* yk, const void* pos, int pos64, int dtype,
                       const int64_t* strides, int64_t B, int64_t N, int H,
                       int KV, int D, int P, const int* start,
                       const double* rev, int inter, int backward) {
  const int64_t rows = B * N;
  if (rows <= 0) return 0;
  if (P < 1 || P > RP_MAXP || 2 * P > D ||
      N > 0x7fffffff ||
      (int64_t)RP_TOK * ((int64_t)H + KV) * D > 0x7fffffff)
    return 9003;
  RopeArgs a;
  a.t[0] = {q, yq, strides[0], strides[1], strides[2], H};
  a.t[1] = {k, yk, strides[3], strides[4], strides[5], KV};
  a.pos = pos;
  a.pA = strides[6]; a.pB = strides[7]; a.pN = strides[8];
  a.pos64 = pos64;
  a.rows = rows;
  a.N = (int)N; a.D = D; a.P = P;
  for (int i = 0; i < 3; ++i) a.start[i] = start[i];
  a.sign = backward ? -1.0f : 1.0f;
  for (int i = 0; i < P; ++i) a.rev[i] = rev[i];
  hipStream_t s = (hipStream_t)stream;
  if (dtype == 0) rp_launch<__hip_bfloat16>(s, a, inter);
  else if (dtype == 1) rp_launch<__half>(s, a, inter);
  else rp_launch<float>(s, a, inter);
  return (int)hipGetLastError();
}
