// window_attn_kernels.hip — causal attention with a sliding window and first
// tokens that stay visible, forward and backward (gfx950 / MI355X).
//
//   vis(i, j) = j <= i and (i - j < window or j < sinks), i, j < length
//   P = softmax over vis of scale * q.k ;  o = P v ;  rows past the length: 0
//   dV = P^T dO ; dP = dO V^T ; dS = P * (dP - rowsum(dO * O)) ;
//   dQ = scale * dS K ; dK = scale * dS^T Q
//
// q, k, v: bf16 of any strides with unit d stride, heads in groups that share
// keys and values.  D is 64 or 128.  Scores, statistics and sums in fp32, P and
// dS rounded to bf16 as operands of the matrix instructions.  rowsum(dO * O)
// takes O before its rounding (a second bf16 tensor holds the rest, written only
// where a gradient will be asked for): what all values share cancels in dS, an
// error of 2^-8 of it would not.  That costs the forward and dQ kernels 8 and 6 us
// at 8192 rows of 32 heads of 128; the error of dQ and dK against 64 bits, up to
// 4.0e-3 without it, is 2.4e-3 at all sizes tried.
//
// Layout.  mfma 32x32x16: operand rows (or columns) are lane % 32, its
// contraction index 8 * (lane / 32) + j; the result's column is lane % 32, its
// row 8 * (r / 4) + 4 * (lane / 32) + r % 4 for register r.  Scores are computed
// transposed to what owns them: a wave that owns 32 queries holds them as
// columns (S^T = K Q^T), one that owns 32 keys holds those as columns
// (S = Q K^T).  So statistics of a row are per-lane numbers (forward, dQ), and
// a result's registers 8s..8s+7 are, as they are, the operand of the next
// product for the contraction rows 16s + {0..3, 8..11} + 4 * (lane / 32): the
// other operand is read from LDS in that same order, by the transposing read.
// P and dS never go through LDS.
//
// Tiles of 64 rows stand in LDS row-major with their 16-byte granules swizzled
// (wa_swz) so that neither the row reads nor the transposing reads meet in a
// bank.  Tiles are double-buffered: the next one travels to LDS directly while
// this one is worked on; one barrier a tile.
//
// Four waves share a tile.  In the forward and dQ kernels they are up to four
// heads of a group (same rows, same keys) times neighbouring rows; in the dK/dV
// kernel four neighbouring strips of 32 keys, and the block walks all heads of
// the group, so that shared heads are summed in registers, without atomics.
//
// The first tokens are seen by all rows: their dK/dV would be one block's work
// of N rows among blocks of `window` rows.  The rows behind the window are
// shared out over further blocks; a last kernel adds their parts in fixed order.
//
// Bound by the matrix instructions and the softmax arithmetic between them.
// 8192 rows, 32 over 8 heads of 128, window 1024, 4 first tokens: forward 182
// us (710 TFLOP/s of visible work), dQ 222, dK/dV 350, their sums 5.  8 x 1024
// rows, 12 heads of 64, window 256: 28, 29, 42 and 4 us.

#include <hip/hip_runtime.h>
#include <hip/hip_bf16.h>
#include <cstdint>

typedef __attribute__((ext_vector_type(8))) __bf16 wa_bf8;
typedef __attribute__((ext_vector_type(2))) __bf16 wa_bf2;
typedef __attribute__((ext_vector_type(2))) float wa_f2;
typedef __attribute__((ext_vector_type(4))) short wa_s4;
typedef __attribute__((ext_vector_type(8))) short wa_s8;
typedef __attribute__((ext_vector_type(16))) float wa_f16;
typedef __attribute__((ext_vector_type(4))) uint32_t wa_u4;
typedef __attribute__((address_space(3))) wa_s4 wa_lds_s4;
typedef __attribute__((address_space(3))) void wa_lds;
typedef __attribute__((address_space(1))) const void wa_mem;

#define WA_BLOCK 256
#define WA_T 64           // rows of a tile
#define WA_KB 128         // keys of a dK/dV block
#define WA_MOST (1LL << 32)  // threads of a launch stay under this
// a call would put the accumulators into memory
#define WA_INLINE __attribute__((always_inline))
#define WA_LOG2E 1.4426950408889634f

struct WaTensor {
  const __bf16* p;
  int64_t sB, sH, sN;
};

struct WaArgs {
  WaTensor q, k, v, o, go;
  __bf16 *out, *dq, *dk, *dv;   // out, dq: [B,N,H,D]; dk, dv: [B,N,KV,D]
  __bf16* low;                  // what out's rounding left out, as out; or null
  float *lse, *delta;           // [B,H,N]; lse of base 2
  float* part;                  // dK, dV parts of the first tokens
  const int32_t* lengths;       // [B], or null
  int B, H, KV, N, window, sinks;
  int strips, slots;            // strips of 32 first tokens; blocks that share the rows
                                // behind the window of 128 of them
  int split;                    // blocks that share the rows of 128 keys
  float* splits;                // their sums, where there is more than one
  float scale;
};

template <int D>
__device__ __forceinline__ int wa_swz(int row) {
  return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3)
                  : ((row & 2) << 1) | ((row >> 2) & 3);
}

__device__ __forceinline__ wa_f16 wa_mfma(wa_bf8 a, wa_bf8 b, wa_f16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The order of a stretch of matrix instructions and the LDS reads that feed
// them: `ahead` reads first, then `each` a matrix instruction.  Left alone the
// compiler reads one operand and waits for it.
template <int MFMAS, int READS, int AHEAD, int EACH>
__device__ __forceinline__ void wa_feed() {
  constexpr int MFMA = 0x008, DS_READ = 0x100;
  __builtin_amdgcn_sched_group_barrier(DS_READ, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    if (AHEAD + i * EACH < READS) __builtin_amdgcn_sched_group_barrier(DS_READ, EACH, 0);
  }
}

// As wa_feed, with VALUS vector instructions behind each matrix instruction.
template <int MFMAS, int READS, int AHEAD, int EACH, int VALUS>
__device__ __forceinline__ void wa_mix() {
  constexpr int VALU = 0x002, MFMA = 0x008, DS_READ = 0x100;
  __builtin_amdgcn_sched_group_barrier(DS_READ, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < MFMAS; ++i) {
    __builtin_amdgcn_sched_group_barrier(MFMA, 1, 0);
    if (AHEAD + i * EACH < READS) __builtin_amdgcn_sched_group_barrier(DS_READ, EACH, 0);
    __builtin_amdgcn_sched_group_barrier(VALU, VALUS, 0);
  }
}

__device__ __forceinline__ float wa_exp2(float x) {
  return __builtin_amdgcn_exp2f(x);
}

// the other half wave's value joined to one's own
__device__ __forceinline__ float wa_other_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float wa_other_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

__device__ __forceinline__ uint32_t wa_pack(float a, float b) {
  const wa_bf2 v = __builtin_convertvector((wa_f2){a, b}, wa_bf2);
  return __builtin_bit_cast(uint32_t, v);
}

// registers 8s..8s+7 of a result as an operand
__device__ __forceinline__ wa_bf8 wa_operand(const wa_f16& f, int s) {
  wa_u4 u;
#pragma unroll
  for (int j = 0; j < 4; ++j) u[j] = wa_pack(f[8 * s + 2 * j], f[8 * s + 2 * j + 1]);
  return __builtin_bit_cast(wa_bf8, u);
}

// Operands of 16 columns of D for a row of the tensor, straight from memory.
template <int D>
__device__ __forceinline__ void wa_row(const __bf16* row, int half, wa_bf8* f) {
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk) f[kk] = *(const wa_bf8*)(row + kk * 16 + half * 8);
}

// A tile on its way from memory to LDS, without registers: each of NW waves
// moves pieces of 1 KB, lane i to the piece's 16 bytes number i; the swizzle is
// on the side of memory.  Whole tiles are addressed by a scalar base and a
// 32-bit offset a lane; in the last one rows past the length hold the last row
// again.  Those are multiplied like others and get the weight zero (a mask; in
// dK/dV a statistic of infinity), which only finite values let vanish.
template <int D, int NW>
struct WaMove {
  static constexpr int G = D / 8, R = 64 / G, CNT = WA_T / R / NW;
  int first;      // this lane's row in the wave's first piece
  int col;        // its elements of that row
  int64_t sN;
  uint32_t off;   // both, in bytes
  const __bf16* base;
  __device__ __forceinline__ WaMove(int lane, int wave) {
    first = wave * R + lane / G;
    // pieces NW apart have the same swizzle: it looks at a row modulo 16
    static_assert(NW * R % 16 == 0, "swizzle of a wave's pieces");
    col = ((lane % G) ^ wa_swz<D>(first)) * 8;
  }
  __device__ __forceinline__ void from(const __bf16* p, int64_t rows) {
    base = p;
    sN = rows;
    off = (uint32_t)((first * (uint32_t)rows + col) * 2);
  }
  __device__ __forceinline__ void go(int row0, int len, char* lds, int wave) const {
#pragma unroll
    for (int i = 0; i < CNT; ++i) {
      const char* at;
      if (row0 + WA_T <= len)
        at = (const char*)(base + (row0 + i * NW * R) * sN) + off;
      else
        at = (const char*)(base + min(row0 + first + i * NW * R, len - 1) * sN + col);
      __builtin_amdgcn_global_load_lds((wa_mem*)at, (wa_lds*)(lds + (i * NW + wave) * 1024), 16, 0, 0);
    }
  }
};

// Row operand: rows sub*32 + lane%32 of a tile, columns 16kk + 8*half ...
template <int D>
struct WaRows {
  int at[D / 16];
  __device__ __forceinline__ WaRows(int lane, int first = 0) {
    const int row = lane & 31, half = lane >> 5;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
      at[kk] = first + row * D * 2 + (((2 * kk + half) ^ wa_swz<D>(row)) * 16);
  }
  __device__ __forceinline__ wa_bf8 get(const char* tile, int sub, int kk) const {
    return *(const wa_bf8*)(tile + at[kk] + sub * 32 * D * 2);
  }
};

// Transposed operand: row is column 32dt + lane%32 of the tile, contraction
// over the tile's rows 16ks + {0..3, 8..11} + 4*half.
template <int D, int DT = D / 32>
struct WaCols {
  int at[2][DT];
  __device__ __forceinline__ WaCols(int lane, int dt0 = 0, int first = 0) {
    const int i = lane & 15, grp = lane >> 4, half = grp >> 1;
#pragma unroll
    for (int jj = 0; jj < 2; ++jj)
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        const int row = 8 * jj + 4 * half + (i >> 2);
        const int col = 32 * (dt0 + dt) + 16 * (grp & 1) + (i & 3) * 4;
        at[jj][dt] = first + row * D * 2 + ((col >> 3) ^ wa_swz<D>(row)) * 16 + (col & 7) * 2;
      }
  }
  __device__ __forceinline__ wa_bf8 get(const char* tile, int ks, int dt) const {
    const wa_s4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (wa_lds_s4*)(tile + at[0][dt] + ks * 16 * D * 2));
    const wa_s4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        (wa_lds_s4*)(tile + at[1][dt] + ks * 16 * D * 2));
    const wa_s8 s = __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    return __builtin_bit_cast(wa_bf8, s);
  }
};

// 8 neighbours of a transposed result's row, 16 bytes a lane: the half waves
// swap what they hold of them.
__device__ __forceinline__ wa_u4 wa_eight(const uint32_t* u) {
  auto a = __builtin_amdgcn_permlane32_swap(u[0], u[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(u[1], u[3], false, false);
  return (wa_u4){a[0], b[0], a[1], b[1]};
}

// Stores a transposed result (columns: 32 rows of the tensor, rows: D) times f;
// with `low` what the rounding left out as well.
template <int D>
__device__ __forceinline__ void wa_store(__bf16* row, const wa_f16* acc, float f,
                                         int half, bool write, __bf16* low = nullptr) {
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      uint32_t u[4], r[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float x = acc[dt][8 * p + 2 * j] * f, y = acc[dt][8 * p + 2 * j + 1] * f;
        u[j] = wa_pack(x, y);
        r[j] = wa_pack(x - __uint_as_float(u[j] << 16),
                       y - __uint_as_float(u[j] & 0xffff0000u));
      }
      const int at = 32 * dt + 16 * p + 8 * half;
      const wa_u4 w = wa_eight(u);
      if (write) *(wa_u4*)(row + at) = w;
      if (low) {
        const wa_u4 v = wa_eight(r);
        if (write) *(wa_u4*)(low + at) = v;
      }
    }
}

// ---------------------------------------------------------------------------
// where a block of the forward and dQ kernels works, and its tiles
// ---------------------------------------------------------------------------

struct WaPlace {
  int b, kv, head, row0, last, len;  // rows row0 .. last of this block
  int wrow;                          // this wave's first row
  int nsink, first, count;           // tiles: nsink from 0, the rest from first
  __device__ __forceinline__ int tile(int it) const {
    return it < nsink ? it : first + it - nsink;
  }
};

// All waves are here, and what they sent to LDS has arrived.
__device__ __forceinline__ void wa_sync() {
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
  __syncthreads();
}

__device__ __forceinline__ int wa_wave() {  // the same for all lanes: a scalar
  return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
}

__device__ __forceinline__ int wa_len(const WaArgs& a, int b) {
  return a.lengths ? max(0, min(a.lengths[b], a.N)) : a.N;
}

// Blocks go to the 8 XCDs in turn, each with an L2 of its own: give every XCD a
// stretch of neighbouring blocks, which read the same tiles.
__device__ __forceinline__ int wa_block(int n) {
  const int x = blockIdx.x & 7;
  return x * (n >> 3) + min(x, n & 7) + (blockIdx.x >> 3);
}

__device__ __forceinline__ WaPlace wa_place(const WaArgs& a, int gw) {
  WaPlace w;
  const int rw = 4 / gw, rows = 32 * rw, wave = wa_wave();
  const int blocks = (a.N + rows - 1) / rows, hb = a.H / gw;
  const int id = wa_block(gridDim.x), u = id / blocks;
  // last rows first: in a short sequence they have the most keys
  const int blk = blocks - 1 - (id - u * blocks);
  w.b = u / hb;
  const int h0 = (u - w.b * hb) * gw;
  w.head = h0 + wave % gw;
  w.kv = h0 / (a.H / a.KV);
  w.len = wa_len(a, w.b);
  w.row0 = blk * rows;
  w.last = min(w.row0 + rows, w.len) - 1;
  w.wrow = w.row0 + (wave / gw) * 32;
  w.first = max(0, w.row0 - a.window + 1) / WA_T;
  w.nsink = min((a.sinks + WA_T - 1) / WA_T, w.first);
  w.count = w.last < w.row0 ? 0 : w.nsink + w.last / WA_T + 1 - w.first;
  return w;
}

// Of rows r0..r0+31 and keys k0..k0+n-1: 0 none visible, 1 some, 2 all
__device__ __forceinline__ int wa_seen(const WaArgs& a, int r0, int k0, int n) {
  if (k0 > r0 + 31) return 0;
  if (k0 >= a.sinks && r0 - (k0 + n - 1) >= a.window) return 0;
  if (k0 + n - 1 <= r0 && (r0 + 31 - k0 < a.window || k0 + n <= a.sinks)) return 2;
  return 1;
}

// Whether element t of a lane is visible; d = row - key grows by `step` with t:
// 0 <= d < window is one unsigned comparison.
struct WaVis {
  int d0;         // row - key at t = 0
  uint32_t window;
  int sink;       // d is also visible from 0 to any size where t < sink
  bool any_sink;  // the same for all lanes
};
// keys run with t (forward, dQ): d = d0 - t
__device__ __forceinline__ bool wa_vis_key(const WaVis& v, int t) {
  bool ok = (uint32_t)(v.d0 - t) < v.window;
  if (v.any_sink) ok = ok || t < v.sink;
  return ok;
}
__device__ __forceinline__ WaVis wa_vis_of(const WaArgs& a, int row, int k0, int half) {
  WaVis v;
  v.d0 = row - k0 - 4 * half;
  v.window = (uint32_t)a.window;
  v.any_sink = k0 < a.sinks;
  v.sink = min(a.sinks - k0 - 4 * half, v.d0 + 1);
  return v;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

template <int D>
__global__ void __launch_bounds__(WA_BLOCK, 2) k_wa_fwd(const WaArgs a, int gw) {
  constexpr int TILE = WA_T * D * 2;  // bytes; two buffers of K and V
  __shared__ __attribute__((aligned(16))) char lds[4 * TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const WaPlace w = wa_place(a, gw);
  const int row = w.wrow + col;
  __bf16* out = a.out + (((int64_t)w.b * a.N + row) * a.H + w.head) * D;
  wa_f16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t) acc[t] = (wa_f16)(0.0f);
  if (w.count == 0) {  // rows past the length
    wa_store<D>(out, acc, 0.0f, half, row < a.N);
    return;
  }
  const __bf16* kb = a.k.p + w.b * a.k.sB + w.kv * a.k.sH;
  const __bf16* vb = a.v.p + w.b * a.v.sB + w.kv * a.v.sH;
  wa_bf8 qf[D / 16];
  wa_row<D>(a.q.p + w.b * a.q.sB + w.head * a.q.sH + min(row, w.len - 1) * a.q.sN, half, qf);
  const WaRows<D> rows(lane);
  const WaCols<D> cols(lane);
  // LDS: two buffers of K, two of V.  Keys are taken 32 at a time; while the
  // weights of one strip are computed, the next strip's scores run on the
  // matrix cores, so K is a strip ahead.
  char* const ldk = lds;
  char* const ldv = lds + 2 * TILE;
  const int wave = wa_wave();
  WaMove<D, 4> mk(lane, wave), mv(lane, wave);
  mk.from(kb, a.k.sN);
  mv.from(vb, a.v.sN);
  mk.go(w.tile(0) * WA_T, w.len, ldk, wave);
  mv.go(w.tile(0) * WA_T, w.len, ldv, wave);
  if (w.count > 1) mk.go(w.tile(1) * WA_T, w.len, ldk + TILE, wave);
  const float c = a.scale * WA_LOG2E;
  // This half wave's keys: the sum of the weights, for the statistic, and that of
  // the weights as they are rounded for their product.  The output is divided
  // by the latter: weights that add up to 1 leave a part that all values share
  // as it is, and in dP - rowsum(dO * O) it cancels.
  float m = -3.0e38f, l = 0.0f, lr = 0.0f;
  const wa_bf2 ones = {(__bf16)1.0f, (__bf16)1.0f};
  auto scores = [&](const char* tk, int sub, wa_f16& to) WA_INLINE {
    to = (wa_f16)(0.0f);
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) to = wa_mfma(rows.get(tk, sub, kk), qf[kk], to);
  };
  // scaled first: the products need no quieting before the comparisons
  auto highest = [&](wa_f16& s) WA_INLINE {
    float top = s[0];
#pragma unroll
    for (int r = 1; r < 15; r += 2) top = fmaxf(fmaxf(top, s[r]), s[r + 1]);
    return fmaxf(top, s[15]);
  };
  // the strip's weights and their product; then the next strip's scores
  auto strip = [&](wa_f16& s, int seen, int k0, const char* tv, int sub, wa_f16& next,
                   int seen_next, const char* tk, int sub_next) WA_INLINE {
    float top = -INFINITY;
    if (seen == 2 && seen_next) {
      scores(tk, sub_next, next);
      s *= c;
      top = highest(s);
      wa_mix<D / 16, D / 16, 4, 1, 3>();
    } else {
      if (seen_next) {
        scores(tk, sub_next, next);
        wa_feed<D / 16, D / 16, 4, 1>();
      }
      if (seen) {
        s *= c;
        if (seen == 1) {
          const WaVis vis = wa_vis_of(a, row, k0, half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!wa_vis_key(vis, 8 * (r / 4) + r % 4)) s[r] = -INFINITY;
        }
        top = highest(s);
      }
    }
    if (seen == 0) return;
    const float mn = fmaxf(m, wa_other_max(top));
    // weights may pass 1 by a factor of 2^8 before everything is rescaled
    if (__any(mn > m + 8.0f)) {
      const float f = wa_exp2(m - mn);
      l *= f;
      lr *= f;
#pragma unroll
      for (int t = 0; t < D / 32; ++t) acc[t] *= f;
      m = mn;
    }
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int r = 8 * ks; r < 8 * ks + 8; ++r) {
        s[r] = wa_exp2(s[r] - m);
        l += s[r];
      }
      const wa_bf8 p = wa_operand(s, ks);
#pragma unroll
      for (int j = 0; j < 8; j += 2)
        lr = __builtin_amdgcn_fdot2_f32_bf16((wa_bf2){p[j], p[j + 1]}, ones, lr, false);
#pragma unroll
      for (int t = 0; t < D / 32; ++t)
        acc[t] = wa_mfma(cols.get(tv, sub * 2 + ks, t), p, acc[t]);
    }
    wa_feed<D / 16, D / 8, 4, 2>();
  };
  wa_sync();
  wa_f16 s0, s1;
  int seen0 = wa_seen(a, w.wrow, w.tile(0) * WA_T, 32);
  if (seen0) {
    scores(ldk, 0, s0);
    wa_feed<D / 16, D / 16, 4, 1>();
  }
  // Nothing is read where the next tile arrives (`to`): the compiler need not
  // wait for it.
  auto first = [&](const char* __restrict__ tv, const char* __restrict__ tk,
                   char* __restrict__ to, bool more, int n0, int k0, int seen1) WA_INLINE {
    if (more) mv.go(n0, w.len, to, wave);
    strip(s0, seen0, k0, tv, 0, s1, seen1, tk, 1);
  };
  auto second = [&](const char* __restrict__ tv, const char* __restrict__ tk,
                    char* __restrict__ to, bool more, int n0, int k0, int seen1, int seen2) WA_INLINE {
    if (more) mk.go(n0, w.len, to, wave);
    strip(s1, seen1, k0, tv, 1, s0, seen2, tk, 0);
  };
  // o: 0 or TILE, where this tile stands
  auto step = [&](int it, int o) WA_INLINE {
    const int k0 = w.tile(it) * WA_T;
    const bool more = it + 1 < w.count, more2 = it + 2 < w.count;
    const int n0 = more ? w.tile(it + 1) * WA_T : 0;
    const int seen1 = wa_seen(a, w.wrow, k0 + 32, 32);
    const int seen2 = more ? wa_seen(a, w.wrow, n0, 32) : 0;
    if (it) wa_sync();
    first(ldv + o, ldk + o, ldv + (TILE - o), more, n0, k0, seen1);
    wa_sync();  // this tile's keys have been read
    second(ldv + o, ldk + (TILE - o), ldk + o, more2, more2 ? w.tile(it + 2) * WA_T : 0,
           k0 + 32, seen1, seen2);
    seen0 = seen2;
  };
  for (int it = 0; it < w.count; it += 2) {
    step(it, 0);
    if (it + 1 < w.count) step(it + 1, TILE);
  }
  l = wa_other_sum(l);
  lr = 1.0f / wa_other_sum(lr);
  const bool in = row < w.len;
  wa_store<D>(out, acc, lr, half, in, a.low ? a.low + (out - a.out) : nullptr);
  if (in) {
    if (half == 0) a.lse[((int64_t)w.b * a.H + w.head) * a.N + row] = m + __builtin_amdgcn_logf(l);
  } else if (row < a.N) {
    for (int e = half * 8; e < D; e += 16) *(wa_u4*)(out + e) = (wa_u4)(0u);
  }
}

// ---------------------------------------------------------------------------
// backward: dQ, and rowsum(dO * O) for the next kernel
// ---------------------------------------------------------------------------

template <int D>
__global__ void __launch_bounds__(WA_BLOCK, 2) k_wa_dq(const WaArgs a, int gw) {
  constexpr int TILE = WA_T * D * 2;  // bytes; two buffers of K and V
  __shared__ __attribute__((aligned(16))) char lds[4 * TILE];
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const WaPlace w = wa_place(a, gw);
  const int row = w.wrow + col;
  __bf16* out = a.dq + (((int64_t)w.b * a.N + row) * a.H + w.head) * D;
  wa_f16 acc[D / 32];
#pragma unroll
  for (int t = 0; t < D / 32; ++t) acc[t] = (wa_f16)(0.0f);
  if (w.count == 0) {
    wa_store<D>(out, acc, 0.0f, half, row < a.N);
    return;
  }
  const __bf16* kb = a.k.p + w.b * a.k.sB + w.kv * a.k.sH;
  const __bf16* vb = a.v.p + w.b * a.v.sB + w.kv * a.v.sH;
  const bool in = row < w.len;
  const int at = min(row, w.len - 1);
  wa_bf8 qf[D / 16], gf[D / 16];
  wa_row<D>(a.q.p + w.b * a.q.sB + w.head * a.q.sH + at * a.q.sN, half, qf);
  wa_row<D>(a.go.p + w.b * a.go.sB + w.head * a.go.sH + at * a.go.sN, half, gf);
  float delta = 0.0f;
  {
    const __bf16* orow = a.o.p + w.b * a.o.sB + w.head * a.o.sH + at * a.o.sN;
    const __bf16* lrow = a.low + (((int64_t)w.b * a.N + at) * a.H + w.head) * D;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      const wa_bf8 of = *(const wa_bf8*)(orow + kk * 16 + half * 8);
      const wa_bf8 lf = *(const wa_bf8*)(lrow + kk * 16 + half * 8);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        delta = fmaf((float)of[j] + (float)lf[j], (float)gf[kk][j], delta);
    }
    delta = wa_other_sum(delta);
  }
  const int64_t stat = ((int64_t)w.b * a.H + w.head) * a.N + at;
  const float lse = a.lse[stat];
  if (in && half == 0) a.delta[stat] = delta;
  const WaRows<D> rows(lane);
  const WaCols<D> cols(lane);
  const int wave = wa_wave();
  WaMove<D, 4> mk(lane, wave), mv(lane, wave);
  mk.from(kb, a.k.sN);
  mv.from(vb, a.v.sN);
  mk.go(w.tile(0) * WA_T, w.len, lds, wave);
  mv.go(w.tile(0) * WA_T, w.len, lds + TILE, wave);
  const float c = a.scale * WA_LOG2E;
  // nothing is read where the next tile arrives: the compiler need not wait
  auto step = [&](int it, char* __restrict__ mine, char* __restrict__ next) {
    char* tk = mine;
    char* tv = mine + TILE;
    const int k0 = w.tile(it) * WA_T;
    const bool more = it + 1 < w.count;
    const int n0 = more ? w.tile(it + 1) * WA_T : 0;
    wa_sync();
    if (more) {
      mk.go(n0, w.len, next, wave);
      mv.go(n0, w.len, next + TILE, wave);
    }
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int seen = wa_seen(a, w.wrow, k0 + sub * 32, 32);
      if (seen) {
        wa_f16 s = (wa_f16)(0.0f), p = (wa_f16)(0.0f);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) s = wa_mfma(rows.get(tk, sub, kk), qf[kk], s);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) p = wa_mfma(rows.get(tv, sub, kk), gf[kk], p);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = wa_exp2(fmaf(s[r], c, -lse));
        // the exponentials run beside dP's products
        wa_feed<D / 16, D / 16, 4, 1>();
        wa_mix<D / 16, D / 16, 4, 1, 4>();
        if (seen == 1) {
          const WaVis vis = wa_vis_of(a, row, k0 + sub * 32, half);
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (!wa_vis_key(vis, 8 * (r / 4) + r % 4)) s[r] = 0.0f;
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= p[r] - delta;
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          wa_bf8 f[D / 32];
#pragma unroll
          for (int t = 0; t < D / 32; ++t) f[t] = cols.get(tk, sub * 2 + ks, t);
          const wa_bf8 d = wa_operand(s, ks);
#pragma unroll
          for (int t = 0; t < D / 32; ++t) acc[t] = wa_mfma(f[t], d, acc[t]);
        }
        wa_feed<D / 16, D / 8, 4, 2>();
      }
    }
  };
  for (int it = 0; it < w.count; it += 2) {
    step(it, lds, lds + 2 * TILE);
    if (it + 1 < w.count) step(it + 1, lds + 2 * TILE, lds);
  }
  wa_store<D>(out, acc, a.scale, half, in);
  if (!in && row < a.N)
    for (int e = half * 8; e < D; e += 16) *(wa_u4*)(out + e) = (wa_u4)(0u);
}

// ---------------------------------------------------------------------------
// backward: dK and dV
// ---------------------------------------------------------------------------
// The first tile of rows that see none of keys k0..k0+127 by the window.  Where
// no blocks take the rest (slots = 0) there is none: no first tokens, or a
// window that covers the sequence.
__device__ __forceinline__ int wa_behind(const WaArgs& a, int k0, int len) {
  const int64_t end = (int64_t)k0 + WA_KB - 1 + a.window;
  return (int)((min(end, (int64_t)len) + WA_T - 1) / WA_T);
}

// fp32 sums [sequence and key head][strip][1 + slots][dK, dV][32][D]
template <int D>
__device__ __forceinline__ float* wa_part(const WaArgs& a, int u, int strip, int slot) {
  return a.part + (((int64_t)u * a.strips + strip) * (1 + a.slots) + slot) * 2 * 32 * D;
}
// fp32 sums [sequence and key head][128 keys][share][dK, dV][128][D]
template <int D>
__device__ __forceinline__ float* wa_split(const WaArgs& a, int u, int nkb, int kblk, int share) {
  return a.splits + (((int64_t)u * nkb + kblk) * a.split + share) * 2 * WA_KB * D;
}
template <int DT>
__device__ __forceinline__ void wa_store_part(float* row, const wa_f16* f, int half) {
#pragma unroll
  for (int t = 0; t < DT; ++t)
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const float4 v = {f[t][4 * r4], f[t][4 * r4 + 1], f[t][4 * r4 + 2], f[t][4 * r4 + 3]};
      *(float4*)(row + 32 * t + 8 * r4 + 4 * half) = v;
    }
}

// A block: 128 keys of a key head and the rows that see them by the window.
//
// PARTS 2: eight waves in pairs; wave w and w + 4 own the same 32 keys and lie
// on one SIMD.  Each computes P and dS of its half of the tile's rows, hands
// them over through LDS (as operands: each lane writes what the same lane of
// the other reads) and sums dK and dV over all rows for its half of D.  With
// full sums in one wave, and K and V in registers as well, D = 128 leaves one
// wave a SIMD: 738 us where pairs take 461 (8192 rows, 32 over 8 heads, window
// 1024; 350 with what came later, the rows behind the window included).  PARTS 1:
// a wave takes all rows and all of D; at three waves a SIMD it keeps 8 of its
// registers (32 bytes a lane) in scratch.

template <int D, int PARTS>
__global__ void __launch_bounds__(PARTS * WA_BLOCK, PARTS == 1 ? 3 : 2)
k_wa_dkv(const WaArgs a) {
  constexpr int NT = PARTS * WA_BLOCK;
  constexpr int TILE = WA_T * D * 2, BUF = 2 * TILE + 2 * WA_T * 4;
  constexpr int H2 = D / PARTS, DT = H2 / 32;  // this wave's part of D
  // two buffers of Q, dO and the rows' statistics; P and dS on their way
  __shared__ __attribute__((aligned(16))) char lds[2 * BUF + (PARTS - 1) * 8 * 4096];
  const int lane = threadIdx.x & 63, half = lane >> 5, col = lane & 31;
  const int wave = wa_wave(), part = PARTS == 1 ? 0 : wave >> 2;
  const int nkb = (a.N + WA_KB - 1) / WA_KB;
  const int main = a.B * a.KV * nkb * a.split;
  // behind: this block takes rows behind the window of first tokens
  const bool behind = (int)blockIdx.x >= main;
  const int shares = behind ? a.slots : a.split;
  const int at = behind ? (int)blockIdx.x - main : wa_block(main);
  const int id = at / shares, share = at - id * shares;
  const int nb = behind ? (a.strips + 3) / 4 : nkb;
  const int u = id / nb, k0 = (id - u * nb) * WA_KB;
  const int b = u / a.KV, kv = u - b * a.KV, G = a.H / a.KV;
  const int len = wa_len(a, b);
  // the rows, in tiles, of each head
  const int edge = wa_behind(a, k0, len), t0 = behind ? edge : k0 / WA_T;
  const int total = max((behind ? (len + WA_T - 1) / WA_T : edge) - t0, 0);
  // (head, tile) pairs: this block's share of them
  const int each = (total * G + shares - 1) / shares;
  const int it0 = min(share * each, total * G), it1 = min(it0 + each, total * G);
  const int wk = k0 + (wave & 3) * 32;   // this wave's first key
  const int key = wk + col;
  wa_f16 ak[DT], av[DT];
#pragma unroll
  for (int t = 0; t < DT; ++t) ak[t] = av[t] = (wa_f16)(0.0f);
  if (it0 < it1) {
    wa_bf8 kf[D / 16], vf[D / 16];
    const int kr = min(key, len - 1);
    wa_row<D>(a.k.p + b * a.k.sB + kv * a.k.sH + kr * a.k.sN, half, kf);
    wa_row<D>(a.v.p + b * a.v.sB + kv * a.v.sH + kr * a.v.sN, half, vf);
    // addresses of this wave's rows of the tile and of the other's
    const int own = part * 32 * D * 2, far = (part ^ (PARTS - 1)) * 32 * D * 2;
    const WaRows<D> rows(lane, own);
    const WaCols<D, DT> cols(lane, part * DT, own), others(lane, part * DT, far);
    WaMove<D, NT / 64> mq(lane, wave), mg(lane, wave);
    char* give = lds + 2 * BUF + wave * 4096 + lane * 16;
    char* take = lds + 2 * BUF + (wave ^ 4) * 4096 + lane * 16;
    float sl = 0.0f, sd = 0.0f;
    const float c = a.scale * WA_LOG2E;
    const bool sinkkey = key < a.sinks;
    int head = kv * G + it0 / total, tile = it0 % total;  // what travels next
    auto of_head = [&]() {
      mq.from(a.q.p + b * a.q.sB + head * a.q.sH, a.q.sN);
      mg.from(a.go.p + b * a.go.sB + head * a.go.sH, a.go.sN);
    };
    auto load = [&](char* to) {
      const int r0 = (t0 + tile) * WA_T;
      if (tile == 0) of_head();
      mq.go(r0, len, to, wave);
      mg.go(r0, len, to + TILE, wave);
      if (threadIdx.x < WA_T) {
        const int r = r0 + threadIdx.x;
        const int64_t i = ((int64_t)b * a.H + head) * a.N + min(r, len - 1);
        sl = r < len ? a.lse[i] : INFINITY;  // no weight for rows that are not
        sd = a.delta[i];
      }
      if (++tile == total) {
        tile = 0;
        ++head;
      }
    };
    auto keep = [&](char* to) {  // the rows' statistics
      if (threadIdx.x < WA_T) {
        ((float*)(to + 2 * TILE))[threadIdx.x] = sl;
        ((float*)(to + 2 * TILE))[WA_T + threadIdx.x] = sd;
      }
    };
    int at_tile = tile;
    of_head();
    load(lds);
    keep(lds);
    // nothing is read where the next tile arrives: the compiler need not wait
    auto step = [&](int it, char* __restrict__ buf, char* __restrict__ next) {
      char* tq = buf;
      char* tg = buf + TILE;
      float* stat = (float*)(buf + 2 * TILE);
      const int r0 = (t0 + at_tile) * WA_T;
      if (++at_tile == total) at_tile = 0;
      const bool more = it + 1 < it1;
      wa_sync();
      if (more) load(next);
      auto sum = [&](const WaCols<D, DT>& from, int ks, wa_bf8 pf, wa_bf8 df) {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
          av[t] = wa_mfma(from.get(tg, ks, t), pf, av[t]);
          ak[t] = wa_mfma(from.get(tq, ks, t), df, ak[t]);
        }
      };
#pragma unroll
      for (int mine = 0; mine < 2 / PARTS; ++mine) {
        const int sub = PARTS == 1 ? mine : part;
        const int seen = wa_seen(a, r0 + sub * 32, wk, 32);
        if (seen == 0) continue;
        const int in = PARTS == 1 ? mine : 0;  // `own` holds the rest
        wa_f16 s = (wa_f16)(0.0f), p = (wa_f16)(0.0f);
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          s = wa_mfma(rows.get(tq, in, kk), kf[kk], s);
        }
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          p = wa_mfma(rows.get(tg, in, kk), vf[kk], p);
        }
        wa_feed<D / 8, D / 8, 4, 1>();
        const int d0 = r0 + sub * 32 + 4 * half - key;  // row - key at t = 0
        const float* st = stat + sub * 32 + 4 * half;
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const float4 ls = *(const float4*)(st + 8 * r4);
          const float4 de = *(const float4*)(st + WA_T + 8 * r4);
          const float lj[4] = {ls.x, ls.y, ls.z, ls.w}, dj[4] = {de.x, de.y, de.z, de.w};
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float e = wa_exp2(fmaf(s[4 * r4 + j], c, -lj[j]));
            if (seen == 1) {
              const int d = d0 + 8 * r4 + j;
              if (!((uint32_t)d < (uint32_t)a.window || (sinkkey && d >= 0))) e = 0.0f;
            }
            s[4 * r4 + j] = e;
            p[4 * r4 + j] = e * (p[4 * r4 + j] - dj[j]);
          }
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
          const wa_bf8 pf = wa_operand(s, ks), df = wa_operand(p, ks);
          if (PARTS == 2) {
            *(wa_bf8*)(give + ks * 1024) = pf;
            *(wa_bf8*)(give + 2048 + ks * 1024) = df;
          }
          sum(cols, in * 2 + ks, pf, df);
        }
        wa_feed<4 * DT, 8 * DT, 4, 2>();
      }
      if (PARTS == 2) {
        wa_sync();
        if (wa_seen(a, r0 + (part ^ 1) * 32, wk, 32)) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
            sum(others, ks, *(const wa_bf8*)(take + ks * 1024),
                *(const wa_bf8*)(take + 2048 + ks * 1024));
          wa_feed<4 * DT, 8 * DT + 4, 8, 2>();
        }
      }
      if (more) keep(next);
    };
    for (int it = it0; it < it1; it += 2) {
      step(it, lds, lds + BUF);
      if (it + 1 < it1) step(it + 1, lds + BUF, lds);
    }
  }
  if (!behind && a.split > 1) {
    float* p = wa_split<D>(a, u, nkb, k0 / WA_KB, share) + (key - k0) * D + part * H2;
    wa_store_part<DT>(p, ak, half);
    wa_store_part<DT>(p + WA_KB * D, av, half);
    return;
  }
  const bool split = a.slots > 0 && key < a.sinks;
  if (split) {
    float* p = wa_part<D>(a, u, key / 32, behind ? 1 + share : 0) + (key % 32) * D + part * H2;
    wa_store_part<DT>(p, ak, half);
    wa_store_part<DT>(p + 32 * D, av, half);
  }
  if (behind) return;
  const bool write = key < a.N && !split;
  const int64_t off = (((int64_t)b * a.N + key) * a.KV + kv) * D + part * H2;
  wa_store<H2>(a.dk + off, ak, a.scale, half, write);
  wa_store<H2>(a.dv + off, av, 1.0f, half, write);
}

// dK and dV from parts, in fixed order.  The first blocks take a first token
// each, 1024 / D parts at a time; the others, where blocks shared the rows of
// 128 keys, 4096 / D of the remaining keys each.
template <int D>
__global__ void __launch_bounds__(1024) k_wa_sum(const WaArgs a, int per, int from) {
  constexpr int W = 1024 / D;
  __shared__ float lds[2][W][D];
  const int first = a.slots > 0 ? a.sinks : 0;  // keys with parts of strips
  const int id = from + blockIdx.x;  // `per` blocks a key head
  const int u = id / per, x = id - u * per;
  const int b = u / a.KV, kv = u - b * a.KV;
  const int nkb = (a.N + WA_KB - 1) / WA_KB;
  if (x >= first) {
    const int key = first + (x - first) * (4096 / D) + threadIdx.x / (D / 4);
    const int d = threadIdx.x % (D / 4) * 4;
    if (key >= a.N) return;
    const float* p = wa_split<D>(a, u, nkb, key / WA_KB, 0) + (key % WA_KB) * D + d;
    float4 k = {0, 0, 0, 0}, v = {0, 0, 0, 0};
    for (int s = 0; s < a.split; ++s, p += 2 * WA_KB * D) {
      const float4 x = *(const float4*)p, y = *(const float4*)(p + WA_KB * D);
      k.x += x.x; k.y += x.y; k.z += x.z; k.w += x.w;
      v.x += y.x; v.y += y.y; v.z += y.z; v.w += y.w;
    }
    const int64_t off = (((int64_t)b * a.N + key) * a.KV + kv) * D + d;
    const uint2 ok = {wa_pack(k.x * a.scale, k.y * a.scale), wa_pack(k.z * a.scale, k.w * a.scale)};
    const uint2 ov = {wa_pack(v.x, v.y), wa_pack(v.z, v.w)};
    *(uint2*)(a.dk + off) = ok;
    *(uint2*)(a.dv + off) = ov;
    return;
  }
  const int key = x, d = threadIdx.x % D, w = threadIdx.x / D;
  float sk = 0.0f, sv = 0.0f;
  // part 0 is the rows' by the window, unless those are shared out themselves
  for (int s = w + (a.split > 1); s <= a.slots; s += W) {
    const float* p = wa_part<D>(a, u, key / 32, s) + (key % 32) * D + d;
    sk += p[0];
    sv += p[32 * D];
  }
  if (a.split > 1)
    for (int s = w; s < a.split; s += W) {
      const float* p = wa_split<D>(a, u, nkb, key / WA_KB, s) + (key % WA_KB) * D + d;
      sk += p[0];
      sv += p[WA_KB * D];
    }
  lds[0][w][d] = sk;
  lds[1][w][d] = sv;
  __syncthreads();
  if (w == 0) {
#pragma unroll
    for (int i = 1; i < W; ++i) {
      sk += lds[0][i][d];
      sv += lds[1][i][d];
    }
    const int64_t off = (((int64_t)b * a.N + key) * a.KV + kv) * D + d;
    a.dk[off] = (__bf16)(sk * a.scale);
    a.dv[off] = (__bf16)sv;
  }
}

// ---------------------------------------------------------------------------

// Blocks that share the rows behind the window of 128 first tokens: at least
// four (head, tile) pairs each, 512 blocks in all.  0: there are no such rows.
static int wa_slots(int64_t U, int64_t G, int64_t N, int64_t window, int64_t sinks) {
  if (sinks <= 0 || N <= window) return 0;
  int64_t n = G * ((N - window + WA_T - 1) / WA_T) / 4;
  const int64_t most = 512 / (U * ((sinks + WA_KB - 1) / WA_KB));
  if (n > most) n = most;
  return (int)(n < 1 ? 1 : n);
}

// Blocks that share the rows of 128 keys where there are fewer of those than
// CUs: one round of blocks, with at least four (head, tile) pairs each.  6 sequences of
// 777, 8 over 2 heads of 128, window 100: 43 us in 84 blocks, 25 in 252.
static int wa_splits(int64_t U, int64_t G, int64_t N, int64_t window) {
  const int64_t blocks = U * ((N + WA_KB - 1) / WA_KB);
  const int64_t rows = window + WA_KB < N ? window + WA_KB : N;
  const int64_t most = G * ((rows + WA_T - 1) / WA_T) / 4;
  int64_t n = 256 / blocks;
  if (n > most) n = most;
  return (int)(n < 1 ? 1 : n);
}

static int64_t wa_slot_floats(int64_t U, int64_t D, int64_t sinks, int64_t slots) {
  return slots ? U * ((sinks + 31) / 32) * (1 + slots) * 2 * 32 * D : 0;
}

extern "C" int64_t ps_wa_part_floats(int64_t B, int64_t H, int64_t KV, int64_t N,
                                     int64_t D, int64_t window, int64_t sinks) {
  if (B <= 0 || KV <= 0 || N <= 0) return 0;
  const int64_t U = B * KV, G = H / KV;
  if (sinks > N) sinks = N;
  if (window > N) window = N;
  const int64_t split = wa_splits(U, G, N, window);
  return wa_slot_floats(U, D, sinks, wa_slots(U, G, N, window, sinks)) +
         (split > 1 ? U * ((N + WA_KB - 1) / WA_KB) * split * 2 * WA_KB * D : 0);
}

static int wa_fill(WaArgs& a, const int64_t* st, int64_t B, int64_t H, int64_t KV,
                   int64_t N, int64_t window, int64_t sinks, float scale,
                   const int32_t* lengths) {
  if (N > (1 << 30) || B * H > 0x7fffffff || N < 1 || KV < 1 || H % KV || window < 1 ||
      sinks < 0 || !(scale > 0.0f))
    return 9003;
  WaTensor* t[5] = {&a.q, &a.k, &a.v, &a.o, &a.go};
  for (int i = 0; i < 5; ++i) {
    t[i]->sB = st[3 * i]; t[i]->sH = st[3 * i + 1]; t[i]->sN = st[3 * i + 2];
  }
  a.B = (int)B; a.H = (int)H; a.KV = (int)KV; a.N = (int)N;
  a.window = (int)(window < N ? window : N);
  a.sinks = (int)(sinks < N ? sinks : N);
  a.strips = (a.sinks + 31) / 32;
  a.slots = wa_slots(B * KV, H / KV, N, a.window, a.sinks);
  a.split = wa_splits(B * KV, H / KV, N, a.window);
  a.scale = scale;
  a.lengths = lengths;
  return 0;
}

static int wa_heads_a_block(int64_t G) { return G % 4 == 0 ? 4 : G % 2 == 0 ? 2 : 1; }

static int64_t wa_row_grid(int64_t B, int64_t H, int64_t N, int gw) {
  const int64_t rows = 128 / gw;
  return B * (H / gw) * ((N + rows - 1) / rows);
}

// A launch holds fewer than 2^32 threads: more sums take several.
template <int D>
static void wa_sum(hipStream_t s, const WaArgs& a, int64_t sums) {
  constexpr int64_t MOST = 1 << 21;
  const int per = (int)(sums / ((int64_t)a.B * a.KV));
  for (int64_t from = 0; from < sums; from += MOST)
    hipLaunchKernelGGL((k_wa_sum<D>), dim3((unsigned)(sums - from < MOST ? sums - from : MOST)),
                       dim3(1024), 0, s, a, per, (int)from);
}

// st: strides (B, H, N) of q, k, v, o, go; o and low are written as [B, N, H, D]
extern "C" int ps_wa_fwd(void* stream, const void* q, const void* k, const void* v,
                         void* o, void* low, float* lse, const int32_t* lengths,
                         const int64_t* st, int64_t B, int64_t H, int64_t KV,
                         int64_t N, int64_t D, int64_t window, int64_t sinks,
                         float scale) {
  if (B <= 0 || N <= 0) return 0;
  WaArgs a{};
  if (int e = wa_fill(a, st, B, H, KV, N, window, sinks, scale, lengths)) return e;
  a.q.p = (const __bf16*)q; a.k.p = (const __bf16*)k; a.v.p = (const __bf16*)v;
  a.out = (__bf16*)o; a.low = (__bf16*)low; a.lse = lse;
  const int gw = wa_heads_a_block(H / KV);
  const int64_t grid = wa_row_grid(B, H, N, gw);
  if (grid >= WA_MOST / WA_BLOCK || (D != 64 && D != 128)) return 9003;
  hipStream_t s = (hipStream_t)stream;
  if (D == 64) hipLaunchKernelGGL((k_wa_fwd<64>), dim3((unsigned)grid), dim3(WA_BLOCK), 0, s, a, gw);
  else hipLaunchKernelGGL((k_wa_fwd<128>), dim3((unsigned)grid), dim3(WA_BLOCK), 0, s, a, gw);
  return (int)hipGetLastError();
}

extern "C" int ps_wa_bwd(void* stream, const void* q, const void* k, const void* v,
                         const void* o, const void* low, const void* go, float* lse,
                         float* delta, void* dq, void* dk, void* dv, float* part,
                         const int32_t* lengths, const int64_t* st, int64_t B,
                         int64_t H, int64_t KV, int64_t N, int64_t D,
                         int64_t window, int64_t sinks, float scale) {
  if (B <= 0 || N <= 0) return 0;
  WaArgs a{};
  if (int e = wa_fill(a, st, B, H, KV, N, window, sinks, scale, lengths)) return e;
  a.q.p = (const __bf16*)q; a.k.p = (const __bf16*)k; a.v.p = (const __bf16*)v;
  a.o.p = (const __bf16*)o; a.go.p = (const __bf16*)go; a.low = (__bf16*)low;
  a.lse = lse; a.delta = delta; a.part = part;
  a.dq = (__bf16*)dq; a.dk = (__bf16*)dk; a.dv = (__bf16*)dv;
  const int gw = wa_heads_a_block(H / KV);
  const int64_t grid = wa_row_grid(B, H, N, gw);
  a.splits = part + wa_slot_floats(B * KV, D, a.sinks, a.slots);
  const int64_t kgrid = B * KV * (((N + WA_KB - 1) / WA_KB) * a.split +
                                  (a.strips + 3) / 4 * a.slots);
  // blocks that add parts: see k_wa_sum
  const int64_t first = a.slots ? a.sinks : 0;
  const int64_t sums =
      B * KV * (first + (a.split > 1 ? (N - first + 4096 / D - 1) / (4096 / D) : 0));
  if (grid >= WA_MOST / WA_BLOCK || kgrid >= WA_MOST / (2 * WA_BLOCK) || sums > 0x7fffffff ||
      (D != 64 && D != 128))
    return 9003;
  hipStream_t s = (hipStream_t)stream;
  const dim3 rows((unsigned)grid), keys((unsigned)kgrid);
  if (D == 64) {
    hipLaunchKernelGGL((k_wa_dq<64>), rows, dim3(WA_BLOCK), 0, s, a, gw);
    // Pairs of waves where blocks do not fill the chip by themselves (16 key
    // heads of 2048, 256 blocks: 66 us against 102), else one wave for both (96
    // of 1024, 768 blocks: 31 us against 41).  The border lies between these
    // two; blocks for rows behind the window count as others.
    if (kgrid < 512)
      hipLaunchKernelGGL((k_wa_dkv<64, 2>), keys, dim3(2 * WA_BLOCK), 0, s, a);
    else
      hipLaunchKernelGGL((k_wa_dkv<64, 1>), keys, dim3(WA_BLOCK), 0, s, a);
    wa_sum<64>(s, a, sums);
  } else {
    hipLaunchKernelGGL((k_wa_dq<128>), rows, dim3(WA_BLOCK), 0, s, a, gw);
    hipLaunchKernelGGL((k_wa_dkv<128, 2>), keys, dim3(2 * WA_BLOCK), 0, s, a);
    wa_sum<128>(s, a, sums);
  }
  return (int)hipGetLastError();
}
