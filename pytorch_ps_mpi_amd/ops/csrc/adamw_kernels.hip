// adamw_kernels.hip — AdamW over a packed set of tensors (gfx950 / MI355X).
//
//   m = b1 m + (1-b1) g ;  v = b2 v + (1-b2) g^2
//   p = p (1 - lr wd decay[chunk]) - lr/bc1 * m / (sqrt(v)/sqrt(bc2) + eps)
//
// One launch updates every tensor of a packed buffer: tensors start at
// multiples of 256 elements, so what differs between them is one number for
// each chunk of 256.  A chunk is one wave, four neighbouring elements a lane.
//
// States are fp32, or 8 bits with one fp32 maximum for each chunk:
//   code k in 1..top stands for  max * 2^((k-top)/8),  0 for zero;
//   the second moment has top 255 (range 2^-31.75), the first has its sign in
//   bit 7 and top 127 (range 2^-15.75).
// A fixed rounding would freeze the averages: with b2 = 0.999 a step moves v
// by 0.1%, the codes are 9% apart.  So a value between two codes goes to the
// upper one with the probability that keeps its mean.  The 16 random bits come
// from a 32-bit mix of (element index, seed, step), the published integer hash
// lowbias32 with its constants and shifts: every rank and every bucketing rounds
// alike.  A second moment that is not zero keeps at least the lowest code, so
// that no denominator collapses to eps.  A state's chunk that holds an infinity
// or NaN gets the maximum NaN: all its values read as NaN.
//
// Bound by HBM: 30 bytes an element with fp32 states and a bf16 copy, 18 with
// 8-bit states.  124 M elements: 678 us (5.5 TB/s) and 489 us (4.6 TB/s).

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <cstdint>

#define AW_BLOCK 256
#define AW_CHUNK 256

struct AwArgs {
  float* p;
  void* out;            // model copy, or null
  const float* g;
  float* m32; float* v32;
  uint8_t* m8; uint8_t* v8;
  float* ms; float* vs;
  const float* decay;   // one factor for each chunk, or null
  int64_t n, offset;
  float step_size, lr_wd, beta1, rest1, beta2, rest2;  // rest = 1 - beta
  float inv_bc2_sqrt, eps, gscale;
  uint32_t key;
};

__device__ __forceinline__ uint32_t aw_mix(uint32_t h) {
  h ^= h >> 16; h *= 0x7feb352du;
  h ^= h >> 15; h *= 0x846ca68bu;
  return h ^ (h >> 16);
}

__device__ __forceinline__ float aw_wave_max(float v) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}

template <int TOP>
__device__ __forceinline__ float aw_decode(uint32_t c, float scale) {
  const uint32_t k = c & TOP;
  const float x = __builtin_amdgcn_exp2f((float)((int)k - TOP) * 0.125f);
  const float y = (k == 0 ? 0.0f : x) * scale;
  return c > TOP ? -y : y;
}

// Which code a value gets is decided in plain fp32 operations, each rounded
// once and none contracted, so that another implementation of them (one
// logarithm, one floor, one expm1) comes to the same codes bit for bit:
//   e = top + 8 log2(a / max), lo = floor(e),
//   up = expm1((e - lo) ln2/8) / (2^(1/8) - 1),  k = lo + (u < up).
// The quotient: a times the reciprocal, put right by its own remainder.
template <int TOP>
__device__ __noinline__ uint32_t aw_code_exact(float a, float s, float inv,
                                               uint32_t r16) {
#pragma clang fp contract(off)
  float r = a * inv;
  r = __builtin_fmaf(__builtin_fmaf(-r, s, a), inv, r);
  const float e = (float)TOP + 8.0f * __builtin_amdgcn_logf(r);
  const float lo = floorf(e);
  const float u = ((float)r16 + 0.5f) * (1.0f / 65536.0f);
  const float up = expm1f((e - lo) * 0.086643398f)   // ln2 / 8
                   * (1.0f / 0.090507733f);          // 2^(1/8) - 1
  float k = fminf(lo + (u < up ? 1.0f : 0.0f), (float)TOP);
  if (e < 1.0f) {  // under the lowest code
    if (TOP == 255) k = 1.0f;
    else k = u < __builtin_amdgcn_exp2f((e - 1.0f) * 0.125f) ? 1.0f : 0.0f;
  }
  return (uint32_t)k;
}

// The same code by a third of the instructions: quotient without its
// correction, exp2 in place of expm1.  That moves e by at most one rounding
// (2^-16) and up by 1.04 times that and 1.5e-6, 1.8e-5 together: where u is
// that near to up, e that near to a whole number or under the lowest code
// (about 1 of 10^4 values), the exact form decides.
template <int TOP>
__device__ __forceinline__ uint32_t aw_encode(float x, float s, float lift,
                                              float inv, bool lifted,
                                              uint32_t r16) {
  const float a = fabsf(x);
  const float e = fmaf(8.0f, __builtin_amdgcn_logf(a * inv), (float)TOP);
  const float lo = floorf(e);
  const float f = e - lo;
  const float t = __builtin_amdgcn_exp2f(f * 0.125f);
  // 65536 up - 0.5 against the 16 bits
  const float d = fmaf(t, 65536.0f * 11.0487795f,
                       -65536.0f * 11.0487795f - 0.5f) - (float)r16;
  uint32_t c = (uint32_t)fminf(lo + (d > 0.0f ? 1.0f : 0.0f), (float)TOP);
  const bool near = fabsf(d) < 1.4f || fabsf(f - 0.5f) > 0.49998f || e < 1.5f ||
                    lifted;
  if (!(a > 0.0f)) c = 0;
  else if (near) c = aw_code_exact<TOP>(a * lift, s, inv, r16);
  if (TOP == 127 && x < 0.0f && c) c |= 128u;
  return c;
}

// A maximum near fp32's smallest has no finite reciprocal: lift both sides.
__device__ __forceinline__ void aw_lift(float& s, float& lift, float& inv) {
  lift = s < 1e-30f ? 1.2676506e30f : 1.0f;  // 2^100
  s *= lift;
  inv = 1.0f / s;
}

__device__ __forceinline__ void aw_moments(const AwArgs& a, float g, float& m,
                                           float& v) {
#pragma clang fp contract(off)
  g *= a.gscale;
  m = a.beta1 * m + a.rest1 * g;
  v = a.beta2 * v + a.rest2 * g * g;
}

__device__ __forceinline__ float aw_param(const AwArgs& a, float p, float m,
                                          float v, float lwd) {
  p = fmaf(-lwd, p, p);
  // the square root instruction wants normal numbers
  const float r = v < 1e-30f
      ? __builtin_amdgcn_sqrtf(v * 1.2676506e30f) * 8.8817842e-16f
      : __builtin_amdgcn_sqrtf(v);
  const float d = fmaf(r, a.inv_bc2_sqrt, a.eps);
  return fmaf(-a.step_size, m * __builtin_amdgcn_rcpf(d), p);
}

// OUT: 0 none, 1 bf16, 2 f32.  VEC: 16-byte accesses; else element by element
// (a buffer that is not 16-byte aligned, and the last chunk of an odd length).
template <bool S8, int OUT, bool VEC>
__device__ __forceinline__ void aw_chunk(const AwArgs& a, int64_t c, int lane) {
  const int64_t i0 = c * AW_CHUNK + lane * 4;
  float p[4], g[4], m[4], v[4];
  float ms = 0, vs = 0;
  if (VEC) {
    *(float4*)p = *(const float4*)(a.p + i0);
    *(float4*)g = *(const float4*)(a.g + i0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = i0 + j < a.n;
      p[j] = in ? a.p[i0 + j] : 0.0f;
      g[j] = in ? a.g[i0 + j] : 0.0f;
    }
  }
  if (S8) {
    uint32_t mc = 0, vc = 0;
    if (VEC) {
      mc = *(const uint32_t*)(a.m8 + i0);
      vc = *(const uint32_t*)(a.v8 + i0);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j < a.n) {
          mc |= (uint32_t)a.m8[i0 + j] << (8 * j);
          vc |= (uint32_t)a.v8[i0 + j] << (8 * j);
        }
    }
    ms = a.ms[c];
    vs = a.vs[c];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = aw_decode<127>((mc >> (8 * j)) & 255u, ms);
      v[j] = aw_decode<255>((vc >> (8 * j)) & 255u, vs);
    }
  } else if (VEC) {
    *(float4*)m = *(const float4*)(a.m32 + i0);
    *(float4*)v = *(const float4*)(a.v32 + i0);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const bool in = i0 + j < a.n;
      m[j] = in ? a.m32[i0 + j] : 0.0f;
      v[j] = in ? a.v32[i0 + j] : 0.0f;
    }
  }
  const float lwd = a.decay ? a.lr_wd * a.decay[c] : a.lr_wd;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    aw_moments(a, g[j], m[j], v[j]);
    p[j] = aw_param(a, p[j], m[j], v[j], lwd);
  }
  if (VEC) {
    *(float4*)(a.p + i0) = *(float4*)p;
    if (OUT == 2) *(float4*)((float*)a.out + i0) = *(float4*)p;
    if (OUT == 1) {
      __hip_bfloat16 o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = __float2bfloat16(p[j]);
      *(uint2*)((__hip_bfloat16*)a.out + i0) = *(uint2*)o;
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < a.n) {
        a.p[i0 + j] = p[j];
        if (OUT == 2) ((float*)a.out)[i0 + j] = p[j];
        if (OUT == 1)
          ((__hip_bfloat16*)a.out)[i0 + j] = __float2bfloat16(p[j]);
      }
  }
  if (S8) {
    float am = 0, av = 0;
    bool mbad = false, vbad = false;  // one may overflow without the other
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (!VEC && i0 + j >= a.n) m[j] = v[j] = 0.0f;
      am = fmaxf(am, fabsf(m[j]));
      av = fmaxf(av, v[j]);
      mbad |= !(fabsf(m[j]) < INFINITY);
      vbad |= !(v[j] < INFINITY);
    }
    am = aw_wave_max(am);
    av = aw_wave_max(av);
    if (__any(mbad)) am = NAN;
    if (__any(vbad)) av = NAN;
    float mx = am, vx = av, ml, mi, vl, vi;
    aw_lift(mx, ml, mi);
    aw_lift(vx, vl, vi);
    const uint64_t e0 = (uint64_t)(a.offset + i0);
    uint32_t mc = 0, vc = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint64_t e = e0 + j;
      const uint32_t r = aw_mix((uint32_t)e ^ aw_mix(a.key + (uint32_t)(e >> 32)));
      mc |= aw_encode<127>(m[j], mx, ml, mi, ml > 1.0f, r & 0xffffu) << (8 * j);
      vc |= aw_encode<255>(v[j], vx, vl, vi, vl > 1.0f, r >> 16) << (8 * j);
    }
    if (VEC) {
      *(uint32_t*)(a.m8 + i0) = mc;
      *(uint32_t*)(a.v8 + i0) = vc;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (i0 + j < a.n) {
          a.m8[i0 + j] = (uint8_t)(mc >> (8 * j));
          a.v8[i0 + j] = (uint8_t)(vc >> (8 * j));
        }
    }
    if (lane == 0) {
      a.ms[c] = am;
      a.vs[c] = av;
    }
  } else if (VEC) {
    *(float4*)(a.m32 + i0) = *(float4*)m;
    *(float4*)(a.v32 + i0) = *(float4*)v;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i0 + j < a.n) {
        a.m32[i0 + j] = m[j];
        a.v32[i0 + j] = v[j];
      }
  }
}

template <bool S8, int OUT, bool VEC>
__global__ void __launch_bounds__(AW_BLOCK) k_fused_adamw(AwArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t chunks = (a.n + AW_CHUNK - 1) / AW_CHUNK;
  for (int64_t c = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6); c < chunks;
       c += (int64_t)gridDim.x * 4) {
    if (VEC && (c + 1) * AW_CHUNK <= a.n) aw_chunk<S8, OUT, true>(a, c, lane);
    else aw_chunk<S8, OUT, false>(a, c, lane);
  }
}

// 16 codes a lane: one 16-byte load.
template <int TOP, typename T>
__global__ void __launch_bounds__(AW_BLOCK)
k_state8_values(const uint8_t* __restrict__ codes,
                const float* __restrict__ scales, T* __restrict__ out,
                int64_t n, int vec) {
  const int64_t stride = (int64_t)gridDim.x * AW_BLOCK * 16;
  for (int64_t i = ((int64_t)blockIdx.x * AW_BLOCK + threadIdx.x) * 16; i < n;
       i += stride) {
    const float s = scales[i / AW_CHUNK];
    if (vec && i + 16 <= n) {
      const uint4 c4 = *(const uint4*)(codes + i);
      const uint32_t c[4] = {c4.x, c4.y, c4.z, c4.w};
      T o[16];
#pragma unroll
      for (int j = 0; j < 16; ++j)
        o[j] = (T)aw_decode<TOP>((c[j / 4] >> (8 * (j & 3))) & 255u, s);
#pragma unroll
      for (int j = 0; j < (int)sizeof(T); ++j)
        ((uint4*)(out + i))[j] = ((uint4*)o)[j];
    } else {
      for (int j = 0; j < 16 && i + j < n; ++j)
        out[i + j] = (T)aw_decode<TOP>(codes[i + j], s);
    }
  }
}

static inline bool aw_al(const void* p, uintptr_t to) {
  return ((uintptr_t)p & (to - 1)) == 0;
}

static inline int aw_grid(int64_t blocks) {
  // one pass a wave up to 2^20 blocks; longer buffers take the stride
  return (int)(blocks < 1 ? 1 : blocks > (1 << 20) ? (1 << 20) : blocks);
}

template <bool S8, bool VEC>
static void aw_launch(hipStream_t s, int grid, int out, const AwArgs& a) {
  if (out == 0)
    hipLaunchKernelGGL((k_fused_adamw<S8, 0, VEC>), dim3(grid), dim3(AW_BLOCK), 0, s, a);
  else if (out == 1)
    hipLaunchKernelGGL((k_fused_adamw<S8, 1, VEC>), dim3(grid), dim3(AW_BLOCK), 0, s, a);
  else
    hipLaunchKernelGGL((k_fused_adamw<S8, 2, VEC>), dim3(grid), dim3(AW_BLOCK), 0, s, a);
}

extern "C" int ps_fused_adamw(void* stream, float* p, void* out, int out_kind,
                              const float* g, void* m, void* v, float* ms,
                              float* vs, const float* decay, int64_t n,
                              int64_t offset, float step_size, float lr_wd,
                              double beta1, double beta2, float inv_bc2_sqrt,
                              float eps, float gscale, uint32_t key) {
  if (n <= 0) return 0;
  const bool s8 = ms != nullptr;
  // 1 - beta is taken in 64 bits: from a 32-bit 0.999 it is 1.3e-5 off
  AwArgs a{p, out, g, (float*)m, (float*)v, (uint8_t*)m, (uint8_t*)v, ms, vs,
           decay, n, offset, step_size, lr_wd, (float)beta1,
           (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2),
           inv_bc2_sqrt, eps, gscale, key};
  const bool vec = aw_al(p, 16) && aw_al(g, 16) && aw_al(m, s8 ? 4 : 16) &&
                   aw_al(v, s8 ? 4 : 16) &&
                   (out_kind == 0 || aw_al(out, out_kind == 1 ? 8 : 16));
  const int grid = aw_grid((n + 4 * AW_CHUNK - 1) / (4 * AW_CHUNK));
  hipStream_t s = (hipStream_t)stream;
  if (s8 && vec) aw_launch<true, true>(s, grid, out_kind, a);
  else if (s8) aw_launch<true, false>(s, grid, out_kind, a);
  else if (vec) aw_launch<false, true>(s, grid, out_kind, a);
  else aw_launch<false, false>(s, grid, out_kind, a);
  return (int)hipGetLastError();
}

extern "C" int ps_state8_values(void* stream, const uint8_t* codes,
                                const float* scales, void* out,
                                int out_is_bf16, int is_signed, int64_t n) {
  if (n <= 0) return 0;
  hipStream_t s = (hipStream_t)stream;
  const int grid = aw_grid((n + 16 * AW_BLOCK - 1) / (16 * AW_BLOCK));
  const int vec = aw_al(codes, 16) && aw_al(out, 16);
  if (out_is_bf16) {
    auto o = (__hip_bfloat16*)out;
    if (is_signed)
      hipLaunchKernelGGL((k_state8_values<127>), dim3(grid), dim3(AW_BLOCK), 0, s, codes, scales, o, n, vec);
    else
      hipLaunchKernelGGL((k_state8_values<255>), dim3(grid), dim3(AW_BLOCK), 0, s, codes, scales, o, n, vec);
  } else {
    auto o = (float*)out;
    if (is_signed)
      hipLaunchKernelGGL((k_state8_values<127>), dim3(grid), dim3(AW_BLOCK), 0, s, codes, scales, o, n, vec);
    else
      hipLaunchKernelGGL((k_state8_values<255>), dim3(grid), dim3(AW_BLOCK), 0, s, codes, scales, o, n, vec);
  }
  return (int)hipGetLastError();
}
