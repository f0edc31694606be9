// Matrix product with bias, activation and residual in its epilogue, and its gradients:
// dd_linear_fwd, dd_linear_bwd_data, dd_linear_bwd_weight, dd_linear_act_bwd.
//
//   y = act(z) + res,  z[m][n] = x_scale[m] w_scale[n] sum_k x[m][k] w[n][k] + bias[n]
//   dz = dy act'(z),  dx = dz w,  dw = dz^T x,  dbias = sum over rows of dz
//
// Operands bf16 or e4m3 (twice the rate, half the bytes), sums in fp32.  The 8-bit instruction adds eight consecutive
// products aligned at the largest and cuts what is below 2^-13 of it, then goes on in fp32: taken for its
// rate, because the operands themselves are rounded to 2^-4.  All three products are P Q^T with different storage orders: an operand is
// contraction-contiguous (KC) or row-contiguous (RC).
#include "block_core.h"
#include <type_traits>

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

// What happens to a finished sum on its way out.
struct Epi {
  void* y; long ldy; int ytype;
  const float* bias;
  int act;
  const void* res; long ldr;
  __bf16* z; long ldz;
  const float* xs; const float* wsc;
  int accumulate;
};

__device__ __forceinline__ float act_any(int act, float z) {
  switch (act) {
    case DD_ACT_ELU: return act_f<DD_ACT_ELU>(z);
    case DD_ACT_SILU: return act_f<DD_ACT_SILU>(z);
    case DD_ACT_GELU: return act_f<DD_ACT_GELU>(z);
    default: return z;
  }
}

// V consecutive outputs of row m from column n (any alignment).
template <int V>
__device__ __forceinline__ void finish(const Epi& e, long m, long n, float v[V]) {
  if (e.xs) {
    const float s = e.xs[m];
    float w[V];
    load_f32<V>(e.wsc + n, w);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = v[j] * s * w[j];
  }
  if (e.bias) {
    float b[V];
    load_f32<V>(e.bias + n, b);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += b[j];
  }
  // the pre-activation is kept in bf16 for the backward pass, half the bytes of fp32 (the derivative is read from it: by
  // itself that leaves dx and dw off by 6e-4 in the 2-norm, beside 1.7e-3 for dz's rounding and as much for their own)
  if (e.z) store_bf16<V>(e.z + m * e.ldz + n, v);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = act_any(e.act, v[j]);
  if (e.res) {
    float r[V];
    if (e.ytype == DD_F32) load_f32<V>((const float*)e.res + m * e.ldr + n, r);
    else load_bf16<V>((const __bf16*)e.res + m * e.ldr + n, r);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += r[j];
  }
  if (e.ytype == DD_F32) {
    float* p = (float*)e.y + m * e.ldy + n;
    if (e.accumulate) {
      float o[V];
      load_f32<V>(p, o);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += o[j];
    }
    store_f32<V>(p, v);
  } else {
    __bf16* p = (__bf16*)e.y + m * e.ldy + n;
    if (e.accumulate) {
      float o[V];
      load_bf16<V>(p, o);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += o[j];
    }
    store_bf16<V>(p, v);
  }
}

// The last columns of a row, fewer than eight; v in LDS.
__device__ __forceinline__ void finish_ragged(const Epi& e, long m, long n, long N, const float* v) {
#pragma unroll 1
  for (int j = 0; n + j < N; ++j) { float t[1] = {v[j]}; finish<1>(e, m, n + j, t); }
}

// An operand: R rows (of the output's rows or columns), contraction length K.
struct Mat { const void* p; long ld; int R; };
typedef unsigned u32x4u __attribute__((ext_vector_type(4), aligned(1)));   // 16 bytes at any address

// The first n (at least one, fewer than a chunk's) elements at p, zeros behind: 8 + 4 + 2 + 1 bytes, in flight
// together.
typedef int i32x4 __attribute__((ext_vector_type(4)));
template <int ES>
__device__ __forceinline__ i32x4 partial_chunk(const char* p, int n) {
  n = __builtin_amdgcn_readfirstlane(n) * ES;   // (the same for all rows)
  typedef unsigned u32x2 __attribute__((ext_vector_type(2), aligned(1)));
  typedef unsigned u32 __attribute__((aligned(1)));
  typedef unsigned short u16 __attribute__((aligned(1)));
  u32x2 a = {0, 0};
  unsigned b = 0, c = 0, d = 0;
  if (n & 8) a = *reinterpret_cast<const u32x2*>(p);
  if (n & 4) b = *reinterpret_cast<const u32*>(p + (n & 8));
  if (n & 2) c = *reinterpret_cast<const u16*>(p + (n & 12));
  if (ES == 1 && n & 1) d = *reinterpret_cast<const unsigned char*>(p + (n & 14));
  c |= d << 8 * (n & 2);
  const i32x4 low = n & 4 ? i32x4{(int)b, (int)c, 0, 0} : i32x4{(int)c, 0, 0, 0};
  return n & 8 ? i32x4{(int)a.x, (int)a.y, low.x, low.y} : low;
}

constexpr int ROWB = 128;         // bytes of the contraction per tile row
constexpr int LROW = ROWB + 16;   // LDS row: 16 bytes more, so that 16-byte reads of 8 rows fall on different banks

// General kernel: 64 x 64 tile, four waves of 32 x 32, operands staged through registers with bounds
// checks on every element that needs them: any size, order and alignment.
template <int ES, bool RC>
__device__ __forceinline__ void stage(const Mat& a, long r0, long k0, int K, char* sh) {
  constexpr int PER = 16 / ES, BK = ROWB / ES;
#pragma unroll
  for (int it = 0; it < 2; ++it) {
    const int ch = threadIdx.x + it * 256;
    if constexpr (!RC) {
      const int r = ch >> 3, kc = (ch & 7) * PER;
      i32x4 v = {0, 0, 0, 0};
      if (r0 + r < a.R) {
        const char* p = (const char*)a.p + ((r0 + r) * a.ld + k0 + kc) * ES;
        if (k0 + kc + PER <= K) __builtin_memcpy(&v, p, 16);
        else if (k0 + kc < K) v = partial_chunk<ES>(p, K % PER);
      }
      *reinterpret_cast<i32x4*>(sh + r * LROW + kc * ES) = v;
    } else {
      // 8 consecutive rows of one k, written one by one into their K-contiguous rows
      const int k = ch >> 3, rr = (ch & 7) * 8;
      unsigned short e[8] = {};
      if (k0 + k < K) {
        const unsigned short* p = (const unsigned short*)a.p + (k0 + k) * a.ld + r0 + rr;
        if (r0 + rr + 8 <= a.R) {
          __builtin_memcpy(e, p, 16);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (r0 + rr + j < a.R) e[j] = p[j];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) *reinterpret_cast<unsigned short*>(sh + (rr + j) * LROW + k * 2) = e[j];
      (void)BK;
    }
  }
}

template <int ES, bool P_RC, bool Q_RC>
__global__ void __launch_bounds__(256) k_linear_any(Mat P, Mat Q, int K, int kspan, float* slabs, Epi e) {
  __shared__ __attribute__((aligned(16))) char sh[2 * 64 * LROW];
  char* shp = sh;
  char* shq = sh + 64 * LROW;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const long m0 = (long)blockIdx.x * 64, n0 = (long)blockIdx.y * 64;
  const long kb = (long)blockIdx.z * kspan;
  const int kend = (int)min((long)K, kb + kspan);
  const int wm = (wave >> 1) * 32, wn = (wave & 1) * 32, r = lane & 31, half = lane >> 5;
  f32x16 acc = {};
  for (long k0 = kb; k0 < kend; k0 += ROWB / ES) {
    stage<ES, P_RC>(P, m0, k0, kend, shp);
    stage<ES, Q_RC>(Q, n0, k0, kend, shq);
    __syncthreads();
    // Q is the instruction's first operand: a lane then holds four consecutive columns of one row
    if constexpr (ES == 2) {
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const bf16x8 q = *reinterpret_cast<const bf16x8*>(shq + (wn + r) * LROW + s * 32 + half * 16);
        const bf16x8 p = *reinterpret_cast<const bf16x8*>(shp + (wm + r) * LROW + s * 32 + half * 16);
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(q, p, acc, 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        i32x8 q, p;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int o = s * 64 + half * 32 + h * 16;
          const uint4 a = *reinterpret_cast<const uint4*>(shq + (wn + r) * LROW + o);
          const uint4 b = *reinterpret_cast<const uint4*>(shp + (wm + r) * LROW + o);
          q[4 * h] = a.x; q[4 * h + 1] = a.y; q[4 * h + 2] = a.z; q[4 * h + 3] = a.w;
          p[4 * h] = b.x; p[4 * h + 1] = b.y; p[4 * h + 2] = b.z; p[4 * h + 3] = b.w;
        }
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(q, p, acc, 0, 0, 0, 127, 0, 127);
      }
    }
    __syncthreads();
  }
  // the 64 x 64 sums through LDS, so that a lane finishes eight consecutive columns
  float* out = reinterpret_cast<float*>(sh);
#pragma unroll
  for (int t = 0; t < 16; ++t) out[(wm + r) * 68 + wn + 8 * (t / 4) + 4 * half + t % 4] = acc[t];
  __syncthreads();
  for (int it = 0; it < 2; ++it) {
    const int ch = threadIdx.x + it * 256, mr = ch >> 3, nc = (ch & 7) * 8;
    const long m = m0 + mr, n = n0 + nc;
    if (m >= P.R) continue;
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = out[mr * 68 + nc + j];
    if (slabs) {
      float* p = slabs + ((long)blockIdx.z * P.R + m) * Q.R + n;
      for (int j = 0; j < 8; ++j)
        if (n + j < Q.R) p[j] = v[j];
    } else if (n + 8 <= Q.R) {
      finish<8>(e, m, n, v);
    } else {
      finish_ragged(e, m, n, Q.R, out + mr * 68 + nc);
    }
  }
}

// ---- tiled kernel --------------------------------------------------------------------------------
//
// BM x BN outputs per workgroup, WM x WN waves, 128 bytes of the contraction per step.  A step's tiles come
// from global memory straight into LDS (16 bytes per lane, no registers in between), two steps ahead for P (three tiles of it), one for Q (two): 160 KB at
// 256 x 256, the whole LDS, 104 at 192 x 128, 80 and two workgroups per CU at 128 x 128.
// Reads past an operand's end give zeros (buffer descriptor) - no bounds checks in the loop; rows may
// start at any address.
//
// LDS holds 16-byte chunks; which chunk of its row a slot holds is permuted by the row, on the GLOBAL
// address of the copy (the LDS side of a copy is fixed: base + lane * 16), so that the lanes of a read
// fall on different banks:
//   KC operand: tile [R][128 B], slot c of row r holds chunk c ^ ((r >> 1) & 7); a lane reads 16 bytes
//     (8 bf16 or 16 e4m3 of its row)
//   RC operand: tile [64 k][R], slot c of row k holds chunk c ^ rc_swizzle(k); read by the transposing LDS
//     load: 4 k of one row per lane, two loads for the 8 k an instruction wants
#define DD_LDS __attribute__((address_space(3)))
__device__ __forceinline__ int rc_swizzle(int k) { return ((k & 3) << 2) ^ ((k >> 2) & 2); }

// 16 bytes per lane from a buffer descriptor's range to LDS, lane after lane from offset `lds`; zeros past the range.
// Written as assembly so that the compiler does not wait for a copy in flight at every LDS read that it cannot
// tell apart from the copy's target; the waits that are needed are written out.  (m0 is reserved: the
// compiler keeps nothing in it.)
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ void copy16(const u32x4& rs, unsigned lds, int voff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" :: "s"(lds), "v"(voff), "s"(rs) : "memory");
}

template <int ES, bool RC, int R_, int NW>
struct TileCopy {
  static constexpr int N = R_ / 8 / NW, BK = ROWB / ES;   // copies per wave and step
  const char* base;      // tile's first byte of the next step
  long step;             // bytes from a step to the next
  unsigned size;         // bytes from base to the end of the tile's last row (KC) or of a whole step (RC)
  unsigned ldb, cols;    // RC: bytes of a row, of the tile's part of it and what is behind (in the contraction's last row)
  int voff[N];
  // KC: contraction elements in front of the lane's chunk (a single wave: in even and odd blocks of 8 rows;
  // an even number of waves: a wave's blocks are all even or all odd)
  int col[1 + NW % 2];
  // the tile at (r0, k0); `apart`: steps of 128 bytes (KC) from one copy to the next
  // ends: the last step is the operand's last.  (A copy takes whole 4-byte units up to the range's end: the last
  // element of an odd RC row is read with the next row's first, and in the last row it is left to mend_corner.)
  __device__ __forceinline__ void init(const Mat& a, long r0, long k0, int K, int wave, int lane, bool ends = true, int apart = 1) {
    base = (const char*)a.p + (RC ? k0 * a.ld + r0 : r0 * a.ld + k0) * ES;
    step = RC ? BK * a.ld * ES : ROWB * apart;
    ldb = (unsigned)(a.ld * ES);
    cols = (unsigned)((a.R - r0) * ES);
    if (!ends) cols += cols & 2;
    size = RC ? (BK - 1) * ldb + cols + (cols & 2) : (unsigned)min((long)R_, a.R - r0) * ldb - ldb + (unsigned)(K - k0) * ES;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = (i * NW + wave) * 64 + lane;
      if constexpr (RC) {
        const int k = id / (R_ / 8), c = (id % (R_ / 8)) ^ rc_swizzle(k);
        voff[i] = (int)(k * ldb) + c * 16;
      } else {
        const int r = id >> 3, c = (id & 7) ^ ((r >> 1) & 7);
        voff[i] = (int)(r * ldb) + c * 16;
      }
    }
#pragma unroll
    for (int i = 0; i < 1 + NW % 2; ++i) col[i] = ((lane & 7) ^ ((4 * ((i * NW + wave) & 1) + (lane >> 4)) & 7)) * (16 / ES);
  }
  // The copies of the next step into LDS offset `lds`; rest: contraction elements left (none: zeros).
  __device__ __forceinline__ u32x4 begin(int rest, int wave) {
    unsigned bytes = rest > 0 ? size : 0u;
    if (RC && rest <= BK) bytes = rest > 0 ? (unsigned)(rest - 1) * ldb + cols : 0u;
    const u32x4 rs = {(unsigned)(uintptr_t)base, (unsigned)((uintptr_t)base >> 32) & 0xffffu, bytes, 0x00020000u};
    if (!RC && rest > 0 && rest < BK)     // the last step of a ragged contraction: chunks that are not whole are
#pragma unroll                            // moved out of the descriptor's range (mend_tail writes the one that is cut)
      for (int i = 0; i < N; ++i) voff[i] = col[i % (1 + NW % 2)] + 16 / ES > rest ? 0x7fffffff : voff[i];
    base += step;
    if (!RC) size -= (unsigned)step;
    return rs;
  }
  __device__ __forceinline__ void one(const u32x4& rs, unsigned lds, int wave, int i) const {
    copy16(rs, lds + (i * NW + wave) * 1024, voff[i]);
  }
  __device__ __forceinline__ void issue(unsigned lds, int wave, int rest) {
    const u32x4 rs = begin(rest, wave);
#pragma unroll
    for (int i = 0; i < N; ++i) one(rs, lds, wave, i);
  }
};
// The chunk in which a KC operand's contraction ends (K is no multiple of a chunk), element by element into
// its place in the tile of the last step; `threads` threads, this one the thread-th, share the rows.
template <int ES, int R_>
__device__ __forceinline__ void mend_tail(const Mat& a, long r0, int K, int k0, char* tile, int thread, int threads) {
  constexpr int PER = 16 / ES;
  const int c = (K - k0) / PER, n = (K - k0) % PER;
  for (int r = thread; r < R_; r += threads) {
    i32x4 v = {0, 0, 0, 0};
    if (r0 + r < a.R) v = partial_chunk<ES>((const char*)a.p + ((r0 + r) * a.ld + k0 + c * PER) * ES, n);
    *reinterpret_cast<i32x4*>(tile + r * ROWB + ((c ^ ((r >> 1) & 7)) << 4)) = v;
  }
}
// The last element of an RC operand of odd row length, row k of the tile of the last step.
template <int R_>
__device__ __forceinline__ void mend_corner(const Mat& a, long r0, int K, int k, char* tile) {
  const int r = (int)(a.R - 1 - r0);
  const unsigned short v = reinterpret_cast<const unsigned short*>(a.p)[(K - 1) * a.ld + a.R - 1];
  *reinterpret_cast<unsigned short*>(tile + k * (R_ * 2) + (((r >> 3) ^ rc_swizzle(k)) << 4) + (r & 7) * 2) = v;
}
// Every copy of this wave but the LATER newest has landed, and then every wave's; reads issued before are
// complete.
template <int LATER = 0>
__device__ __forceinline__ void sync_copies() {
  static_assert(LATER < 16, "");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0070 | LATER);   // vmcnt LATER, lgkmcnt 0
  asm volatile("s_barrier" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
}

// The matrix instruction, by element size: rows of an operand block, accumulator, and the operand of rows
// r .. r + ROWS - 1 and contraction step s (32 bf16, 64 e4m3).  bf16 takes the 16 x 16 form: it needs more
// operands per product than 32 x 32 but moves half the accumulators, and under the chip's power cap that is
// clock (8192^3: 766 against 811 us).
template <int ES>
struct Inst;
template <>
struct Inst<2> {
  static constexpr int ROWS = 16;
  typedef f32x4 Acc;
  typedef bf16x8 Op;
};
template <>
struct Inst<1> {
  static constexpr int ROWS = 32;
  typedef f32x16 Acc;
  typedef i32x8 Op;
};
template <int ES, bool RC, int R_>
struct Frag;
template <int R_>
struct Frag<2, false, R_> {
  static __device__ __forceinline__ bf16x8 read(const char* sh, int r, int s, int lane) {
    const int row = r + (lane & 15), c = (4 * s + (lane >> 4)) ^ ((row >> 1) & 7);
    return *reinterpret_cast<const bf16x8*>(sh + row * ROWB + c * 16);
  }
};
template <int R_>
struct Frag<2, true, R_> {
  static __device__ __forceinline__ bf16x8 read(const char* sh, int r, int s, int lane) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    typedef short s16x8 __attribute__((ext_vector_type(8)));
    const int k = s * 32 + (lane >> 4) * 8 + ((lane & 15) >> 2), row = r + (lane & 3) * 4;
    const int at = k * (R_ * 2) + (((row >> 3) ^ rc_swizzle(k)) << 4) + (row & 4) * 2;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DD_LDS s16x4*)(sh + at));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((DD_LDS s16x4*)(sh + at + 4 * R_ * 2));   // k + 4: the same swizzle
    const s16x8 t = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
    return __builtin_bit_cast(bf16x8, t);
  }
};
template <int R_>
struct Frag<1, false, R_> {
  // (which 32 of the 64 elements a lane holds, and in which order, is free: both operands agree)
  static __device__ __forceinline__ i32x8 read(const char* sh, int r, int s, int lane) {
    const int row = r + (lane & 31), x = (row >> 1) & 7, c = 4 * s + 2 * (lane >> 5);
    const i32x4 a = *reinterpret_cast<const i32x4*>(sh + row * ROWB + ((c ^ x) << 4));
    const i32x4 b = *reinterpret_cast<const i32x4*>(sh + row * ROWB + (((c + 1) ^ x) << 4));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};
__device__ __forceinline__ f32x4 mma(bf16x8 q, bf16x8 p, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(q, p, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(i32x8 q, i32x8 p, f32x16 c) {
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(q, p, c, 0, 0, 0, 127, 0, 127);
}

// The largest divisor of n that is at most m.
constexpr int whole_part(int n, int m) { return m <= 0 ? 0 : m >= n ? n : n % m == 0 ? m : whole_part(n, m - 1); }

template <int ES, bool P_RC, bool Q_RC, int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN, BM * BN > 16384 ? 2 : 4) k_linear_tile(Mat P, Mat Q, int K, int kspan, int tm, int tn, float* slabs, Epi e) {
  typedef Inst<ES> I;
  constexpr int NW = WM * WN, MT = BM / WM / I::ROWS, NT = BN / WN / I::ROWS, UP = BM * ROWB, UQ = BN * ROWB;
  static_assert(BM % (WM * I::ROWS) == 0 && BN % (WN * I::ROWS) == 0, "the waves' instructions cover the tile");
  constexpr int STEPS = 2, BK = ROWB / ES, LDS = 3 * UP + 2 * UQ;
  __shared__ __attribute__((aligned(1024))) char sh[LDS];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Consecutive workgroups go to the eight XCDs in turn: each XCD gets a contiguous run of tiles, four
  // columns wide, so that its L2 serves the rows and weights that its 32 running tiles share
  // (4 x 8 tiles read 12 operand tiles per step, 2 x 16 would read 18).
  const int total = gridDim.x, q8 = total / 8, r8 = total % 8, xcd = blockIdx.x % 8;
  int id = xcd * q8 + min(xcd, r8) + blockIdx.x / 8;
  const int split = id / (tm * tn);
  id -= split * (tm * tn);
  const int band = id / (4 * tm), width = min(4, tn - 4 * band);
  id -= band * 4 * tm;
  const int nt = 4 * band + id % width, mt = id / width;
  const long m0 = (long)mt * BM, n0 = (long)nt * BN, kb = (long)split * kspan;
  const int kend = (int)min((long)K, kb + kspan), steps = (kend - (int)kb + BK - 1) / BK;
  const int wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);

  TileCopy<ES, P_RC, BM, NW> cp;
  TileCopy<ES, Q_RC, BN, NW> cq;
  cp.init(P, m0, kb, K, wave, lane, kend == K);
  cq.init(Q, n0, kb, K, wave, lane, kend == K);
  const unsigned lds = (unsigned)(uintptr_t)(DD_LDS char*)sh;
  typename I::Acc acc[MT][NT] = {};
  int rest_p = kend - (int)kb, rest_q = rest_p;   // of the step that is copied next
  // A group: one contraction step of the instruction, all of the wave's rows, or half of them where two register
  // sets of all would not fit.
  constexpr int H = MT % 2 || (ES == 2 && MT <= 4) ? 1 : 2, MH = MT / H, GROUPS = STEPS * H;
  typename I::Op p[2][MH], q[2][NT];
  // one of a group's NT + MH operands
  auto read1 = [&](int at_p, int at_q, int g, int k) {
    if (k < NT) {
      if (g % H == 0) q[(g / H) & 1][k] = Frag<ES, Q_RC, BN>::read(sh + at_q, wn + I::ROWS * k, g / H, lane);
    } else {
      p[g & 1][k - NT] = Frag<ES, P_RC, BM>::read(sh + at_p, wm + I::ROWS * (k - NT + (g % H) * MH), g / H, lane);
    }
  };
  // The waves meet once a step, before its last group: step t + 1 has landed, step t's tiles are free but for
  // the last group's operands, which are in registers.  Behind the instructions of that group and of the
  // next one the copies of Q (step t + 2) and P (t + 3) are issued - a few behind each row of instructions: in
  // one go they would hold the waves up while the address unit works through them.  Operands are read one
  // group ahead, across the barrier too, so that the matrix unit has work while the waves meet.
  // (a contraction that ends inside a chunk, an odd RC row: the last step's tiles are mended once they have landed)
  const bool odd_p = P_RC && P.R % 2 != 0 && m0 + BM >= P.R, odd_q = Q_RC && Q.R % 2 != 0 && n0 + BN >= Q.R;
  const bool part = K % (16 / ES) != 0, cut = kend == K && ((part && !(P_RC && Q_RC)) || odd_p || odd_q);
  auto mend = [&](int at_p, int at_q) {
    const int k0 = (int)kb + (steps - 1) * BK;
    if constexpr (!P_RC) { if (part) mend_tail<ES, BM>(P, m0, K, k0, sh + at_p, threadIdx.x, NW * 64); }
    else if (odd_p && threadIdx.x == 0) mend_corner<BM>(P, m0, K, K - 1 - k0, sh + at_p);
    if constexpr (!Q_RC) { if (part) mend_tail<ES, BN>(Q, n0, K, k0, sh + at_q, threadIdx.x, NW * 64); }
    else if (odd_q && threadIdx.x == 0) mend_corner<BN>(Q, n0, K, K - 1 - k0, sh + at_q);
    sync_copies();
  };
  int p0 = 0, p1 = UP, p2 = 2 * UP, q0 = 3 * UP, q1 = 3 * UP + UQ;
  cp.issue(lds + p0, wave, rest_p); rest_p -= BK;
  cq.issue(lds + q0, wave, rest_q); rest_q -= BK;
  cp.issue(lds + p1, wave, rest_p); rest_p -= BK;
  sync_copies<TileCopy<ES, P_RC, BM, NW>::N>();
  if (cut && steps == 1) mend(p0, q0);
  cq.issue(lds + q1, wave, rest_q); rest_q -= BK;
#pragma unroll
  for (int k = 0; k < NT + MH; ++k) read1(p0, q0, 0, k);
  for (int t = 0; t < steps; ++t) {
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + 1 == GROUPS) {
        sync_copies<TileCopy<ES, P_RC, BM, NW>::N>();
        if (cut && t + 2 == steps) mend(p1, q1);
      }
      u32x4 rs;
      if (g == GROUPS - 1) { rs = cq.begin(rest_q, wave); rest_q -= BK; }
      if (g == 0) { rs = cp.begin(rest_p, wave); rest_p -= BK; }
#pragma unroll
      for (int i = 0; i < MH; ++i) {
#pragma unroll
        for (int k = i * (NT + MH) / MH; k < (i + 1) * (NT + MH) / MH; ++k)
          read1(g + 1 < GROUPS ? p0 : p1, g + 1 < GROUPS ? q0 : q1, g + 1 < GROUPS ? g + 1 : 0, k);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < NT; ++j)
          acc[i + (g % H) * MH][j] = mma(q[(g / H) & 1][j], p[g & 1][i], acc[i + (g % H) * MH][j]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int k = 0; k < cp.N; ++k)
          if (g == 0 && k >= i * cp.N / MH && k < (i + 1) * cp.N / MH) cp.one(rs, lds + p2, wave, k);
#pragma unroll
        for (int k = 0; k < cq.N; ++k)
          if (g == GROUPS - 1 && k >= i * cq.N / MH && k < (i + 1) * cq.N / MH) cq.one(rs, lds + q0, wave, k);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int tp = p0, tq = q0;
    p0 = p1; p1 = p2; p2 = tp;
    q0 = q1; q1 = tq;
  }
  sync_copies();

  // Sixteen rows at a time through the wave's own LDS (Q was the instruction's first operand: a lane holds four
  // consecutive columns of one row); LPR lanes finish a row, 8 columns each, RI rows per lane.  The residual's
  // tile - the part of it that these lanes finish - comes into the wave's LDS in bursts as large as that is, like the
  // tiles before it: requested sixteen rows at a time it cost a memory latency each (37500 x 2048 x 1024 with a
  // residual 222 us against 184).  Only the writes to LDS know which accumulators they take; the rest of the
  // loop stays rolled, because copies of three activations would not fit the instruction cache.
  constexpr int W = BN / WN, LPR = W / 8, RPI = 64 / LPR, RI = 16 / RPI, ROWS = I::ROWS, WROWS = BM / WM, HALVES = WROWS / 16;
  // Rows of an exchange, an accumulator block's where the wave's LDS holds them beside the residual; bytes of the two;
  // sixteens of rows in a burst of the residual (a divisor of the wave's, so that bursts end with the rows).
  constexpr int XR = LDS / NW - ROWS * W * 4 >= 4096 ? ROWS : 16, OUT = XR * W * 4, RES = LDS / NW - OUT;
  constexpr int BURST2 = whole_part(HALVES, RES / (16 * W * 2)), BURST4 = whole_part(HALVES, RES / (16 * W * 4));
  static_assert(RI * RPI == 16, "sixteen rows are whole rows of every lane");
  static_assert(BURST4 > 0, "the residual's LDS");
  char* mine = sh + wave * (OUT + RES);
  float* out = reinterpret_cast<float*>(mine);
  // 16-byte chunk c of row r, permuted by the row so that the writes of 16 rows fall on different banks
  auto at = [&](int r, int c) { return out + r * W + ((c ^ (r & (W / 4 - 1))) << 2); };
  // The lane's 8 columns end where the row ends and overlap its neighbour's (the same values twice) rather than being
  // cut: element by element they took longer than the product (111 x 2391 x 577 with a residual: 25 us against 13).
  // Fewer than 8 columns of the wave's: none is full.
  const int cols = (int)min((long)W, Q.R - (n0 + wn));
  int nc = (lane % LPR) * 8;
  const bool shifted = cols >= 8 && nc < cols && nc + 8 > cols;
  if (shifted) nc = cols - 8;
  const bool full = nc + 8 <= cols;
  const long n = n0 + wn + nc, mrow = m0 + wm + lane / LPR;
  const int es = e.ytype == DD_F32 ? 4 : 2, burst = e.ytype == DD_F32 ? BURST4 : BURST2;
  auto fetch = [&](int i) {   // the residual's rows 16 i .. 16 (i + burst) - 1 of the wave
    const int rows = (int)min((long)burst * 16, P.R - (m0 + wm + 16 * i));
    const unsigned ldb = (unsigned)(e.ldr * es);
    const char* base = (const char*)e.res + ((m0 + wm + 16 * i) * e.ldr + n0 + wn) * es;
    // an odd row's last bf16 is half of a 4-byte unit: read whole, except at the end of the matrix (below)
    const unsigned width = cols * es + (m0 + wm + 16 * i + rows < P.R ? cols * es & 2 : 0);
    const u32x4 rs = {(unsigned)(uintptr_t)base, (unsigned)((uintptr_t)base >> 32) & 0xffffu,
                      rows > 0 && cols > 0 ? (rows - 1) * ldb + width : 0u, 0x00020000u};
    const unsigned to = lds + wave * (OUT + RES) + OUT, step = 1024 / (W * es) * ldb,
                   v = es == 4 ? lane / (W / 4) * ldb + lane % (W / 4) * 16 : lane / (W / 8) * ldb + lane % (W / 8) * 16;
#pragma unroll 1
    for (int k = 0; k < burst * 16 * W * es / 1024; ++k) copy16(rs, to + k * 1024, (int)(v + k * step));
  };
  // the sums of sixteen rows: lane's RI rows of 8 columns
  const int lr = lane / LPR;
  float v[RI][8];
  auto exchange = [&](int i) {
    constexpr int PER = ROWS / 16;   // sixteens of an accumulator block
    // (a bit, not i / PER == k: the compiler would index the accumulators by i, in memory)
    const unsigned which = 1u << i / PER;
    int l = lane, c = nc;
    asm volatile("" : "+v"(c));   // these addresses are computed here, not kept across the loop
    if constexpr (BM * BN <= 16384) asm volatile("" : "+v"(l));   // (nor these: 128 registers)
    const int lr = l / LPR + (XR == 32 ? i % 2 * 16 : 0);
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < MT; ++k)
      if (which >> k & 1 && (XR == 32 ? i % 2 == 0 : PER == 1 || (l % 32) / 16 == i % PER))
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int g = 0; g < PER * PER; ++g) {   // 16 x 16: one run of four columns, 32 x 32: four, 8 apart
            const f32x4 t = {acc[k][j][4 * g], acc[k][j][4 * g + 1], acc[k][j][4 * g + 2], acc[k][j][4 * g + 3]};
            *reinterpret_cast<f32x4*>(at(l % XR, (ROWS * j + 8 * g) / 4 + l / ROWS)) = t;
          }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int k = 0; k < RI; ++k)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const f32x4 t = *reinterpret_cast<const f32x4*>(at(lr + RPI * k, lane % LPR * 2 + h));
#pragma unroll
        for (int j = 0; j < 4; ++j) v[k][4 * h + j] = t[j];
      }
    if (cols % 8 != 0 && cols >= 8 && cols < W) {   // (wave-uniform)
      if (shifted)
#pragma unroll
        for (int k = 0; k < RI; ++k)
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] = at(lr + RPI * k, (c + j) / 4)[(c + j) & 3];
    }
  };
  if (slabs) {
    float* slab = slabs + ((long)split * P.R + mrow) * Q.R + n;
#pragma unroll 1
    for (int i = 0; i < HALVES; ++i) {
      exchange(i);
#pragma unroll
      for (int k = 0; k < RI; ++k) {
        if (mrow + 16 * i + RPI * k >= P.R) continue;
        float* to = slab + (long)(16 * i + RPI * k) * Q.R;
        if (full) {
          store_f32<8>(to, v[k]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (nc + j < cols) to[j] = v[k][j];
        }
      }
    }
    return;
  }
  float bias[8] = {}, col[8], xs[(WROWS + 63) / 64];
  if (full && e.bias) load_f32<8>(e.bias + n, bias);
  if (e.xs) {
    if (full) load_f32<8>(e.wsc + n, col);
#pragma unroll
    for (int k = 0; k < (WROWS + 63) / 64; ++k) xs[k] = e.xs[min(m0 + wm + 64 * k + lane, (long)P.R - 1)];
  }
  const int left = (int)min((long)WROWS, P.R - mrow);   // rows from the lane's first one on
  const float corner = shifted && e.res && es == 2 ? (float)((const __bf16*)e.res)[min(mrow + left - 1, (long)P.R - 1) * e.ldr + n + 7] : 0.f;
#pragma unroll 1
  for (int i = 0; i < HALVES; ++i) {
    if (e.res && i % burst == 0) fetch(i);
    exchange(i);
    if (e.xs) {
      if (i % 4 == 0 && i > 0) xs[0] = xs[(WROWS - 1) / 64];
#pragma unroll
      for (int k = 0; k < RI; ++k) {
        const float s = __shfl(xs[0], (16 * i + RPI * k + lr) & 63);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] = fma_(v[k][j] * s, col[j], bias[j]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < RI; ++k)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[k][j] += bias[j];
    }
    if (e.res && i % burst == 0) {
      __builtin_amdgcn_s_waitcnt(0x0f70);   // the burst has landed
      asm volatile("" ::: "memory");
    }
    if (full) {
      if (e.z) {
        __bf16* to = e.z + (mrow + 16 * i) * e.ldz + n;
#pragma unroll
        for (int k = 0; k < RI; ++k)
          if (16 * i + RPI * k < left) store_bf16<8>(to + RPI * k * e.ldz, v[k]);
      }
#define DD_ACT_CASE(A_)                          \
  case A_:                                       \
    _Pragma("unroll") for (int k = 0; k < RI; ++k) { \
      _Pragma("unroll") for (int j = 0; j < 8; ++j) v[k][j] = act_f<A_>(v[k][j]); \
      __builtin_amdgcn_sched_barrier(0);         \
    }                                            \
    break;
      switch (e.act) { DD_ACT_CASE(DD_ACT_ELU) DD_ACT_CASE(DD_ACT_SILU) DD_ACT_CASE(DD_ACT_GELU) }
#undef DD_ACT_CASE
      if (e.res) {
        const char* r = mine + OUT + ((16 * (i % burst) + lr) * W + nc) * es;
#pragma unroll
        for (int k = 0; k < RI; ++k) {
          float t[8];
          if (e.ytype == DD_F32) load_f32<8>((const float*)r + RPI * k * W, t);
          else load_bf16<8>((const __bf16*)r + RPI * k * W, t);
          if (shifted && es == 2 && 16 * i + RPI * k == left - 1) t[7] = corner;
#pragma unroll
          for (int j = 0; j < 8; ++j) v[k][j] += t[j];
        }
      }
      if (e.ytype == DD_F32) {
        float* to = (float*)e.y + (mrow + 16 * i) * e.ldy + n;
#pragma unroll
        for (int k = 0; k < RI; ++k, to += RPI * e.ldy) {
          if (16 * i + RPI * k >= left) continue;
          if (e.accumulate) {
            float o[8];
            load_f32<8>(to, o);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] += o[j];
          }
          store_f32<8>(to, v[k]);
        }
      } else {
        __bf16* to = (__bf16*)e.y + (mrow + 16 * i) * e.ldy + n;
#pragma unroll
        for (int k = 0; k < RI; ++k, to += RPI * e.ldy) {
          if (16 * i + RPI * k >= left) continue;
          if (e.accumulate) {
            float o[8];
            load_bf16<8>(to, o);
#pragma unroll
            for (int j = 0; j < 8; ++j) v[k][j] += o[j];
          }
          store_bf16<8>(to, v[k]);
        }
      }
    }
    if (cols > 0 && cols < 8)
      for (int k = lane; k < 16 * 8; k += 64) {
        const int r = k / 8, j = k % 8;
        const long m = m0 + wm + 16 * i + r;
        if (j >= cols || m >= P.R) continue;
        float t[1] = {at(r + (XR == 32 ? i % 2 * 16 : 0), j / 4)[j & 3]};
        finish<1>(e, m, n0 + wn + j, t);
      }
    // (the reads of this burst are complete before the next one overwrites it)
    if (e.res && (i + 1) % burst == 0) {
      __builtin_amdgcn_s_waitcnt(0xc07f);
      asm volatile("" ::: "memory");
    }
  }
}

// ---- few rows: single steps of serving -----------------------------------------------------------
//
// At most 128 rows, so the weights are read once and that read is the time.  A workgroup owns 16 weight
// rows; its waves take turns along the contraction, 128 bytes of every row at a time, each with two LDS
// buffers of its own: no barrier, the next turn's copies are in flight while 16 x 16 instructions work on
// this one's.  At the end the waves add up in LDS: one launch, no partial sums in memory.  (Operands straight
// into registers would have 16 different rows in every quarter of a load: 18 bytes per clock and CU instead of
// 60; 32 x 1024 x 4096 bf16 13 us.)
template <int ES, int MB, int WV>
__global__ void __launch_bounds__(64 * WV) k_linear_few(Mat P, Mat Q, int K, Epi e) {
  constexpr int BK = ROWB / ES, TURN = (16 + 16 * MB) * ROWB, COPIES = 2 + 2 * MB;
  __shared__ __attribute__((aligned(1024))) char sh[WV * 2 * TURN];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4, swz = (row >> 1) & 7;
  const long n0 = (long)blockIdx.x * 16;
  const int steps = (K + BK - 1) / BK, turns = wave < steps ? (steps - wave + WV - 1) / WV : 0;
  char* mine = sh + wave * 2 * TURN;
  const unsigned lds = (unsigned)(uintptr_t)(DD_LDS char*)mine;
  TileCopy<ES, false, 16, 1> cq;
  TileCopy<ES, false, 16 * MB, 1> cp;
  int rest = K - wave * BK;
  cq.init(Q, n0, (long)wave * BK, K, 0, lane, true, WV);
  cp.init(P, 0, (long)wave * BK, K, 0, lane, true, WV);
  auto copy = [&](int buf) {
    cq.issue(lds + buf * TURN, 0, rest);
    cp.issue(lds + buf * TURN + 16 * ROWB, 0, rest);
    rest -= WV * BK;
  };
  f32x4 acc[MB] = {};
  copy(0);
  copy(1);
  for (int t = 0; t < turns; ++t) {
    char* a = mine + (t & 1) * TURN;
    __builtin_amdgcn_s_waitcnt(0x0f70 | (COPIES & 15) | (COPIES >> 4) << 14);   // vmcnt: all but the next turn's copies have landed
    asm volatile("" ::: "memory");
    const int k0 = (wave + t * WV) * BK;
    if (K % (16 / ES) != 0 && k0 + BK > K) {        // the contraction ends inside a chunk
      mend_tail<ES, 16>(Q, n0, K, k0, a, lane, 64);
      mend_tail<ES, 16 * MB>(P, 0, K, k0, a + 16 * ROWB, lane, 64);
      __builtin_amdgcn_s_waitcnt(0xc07f);           // lgkmcnt 0
      asm volatile("" ::: "memory");
    }
    auto chunk = [&](int r, int c) { return *reinterpret_cast<const i32x4*>(a + (r + row) * ROWB + ((c ^ swz) << 4)); };
    i32x4 q[2], x[MB][2];
    // bf16: chunks g, 4 + g for the two instructions; e4m3: any two that both operands agree on
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      q[j] = chunk(0, 4 * j + g);
#pragma unroll
      for (int b = 0; b < MB; ++b) x[b][j] = chunk(16 + 16 * b, 4 * j + g);
    }
    __builtin_amdgcn_s_waitcnt(0xc07f);             // read before the buffer is copied into again
    asm volatile("" ::: "memory");
    copy(t & 1);
#pragma unroll
    for (int b = 0; b < MB; ++b) {
      if constexpr (ES == 2) {
#pragma unroll
        for (int j = 0; j < 2; ++j)
          acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, q[j]), __builtin_bit_cast(bf16x8, x[b][j]), acc[b], 0, 0, 0);
      } else {
        const i32x8 w8 = __builtin_shufflevector(q[0], q[1], 0, 1, 2, 3, 4, 5, 6, 7);
        const i32x8 x8 = __builtin_shufflevector(x[b][0], x[b][1], 0, 1, 2, 3, 4, 5, 6, 7);
        acc[b] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w8, x8, acc[b], 0, 0, 0, 127, 0, 127);
      }
    }
  }
  sync_copies();   // (the copies behind the end wrote zeros)
  // a lane holds columns 4 g .. + 3 of row lane & 15
  float* out = reinterpret_cast<float*>(sh);
  static_assert(WV * MB * 16 * 17 * 4 <= WV * 2 * TURN, "the sums fit the copies' LDS");
#pragma unroll
  for (int b = 0; b < MB; ++b)
#pragma unroll
    for (int j = 0; j < 4; ++j) out[((wave * MB + b) * 16 + row) * 17 + 4 * g + j] = acc[b][j];
  __syncthreads();
  for (int i = threadIdx.x; i < MB * 256; i += 64 * WV) {
    const int m = i >> 4, c = i & 15;
    if (m < P.R && n0 + c < Q.R) {
      float v[1] = {out[m * 17 + c]};
#pragma unroll
      for (int w = 1; w < WV; ++w) v[0] += out[(w * MB * 16 + m) * 17 + c];
      finish<1>(e, m, n0 + c, v);
    }
  }
}

// Sum of the partial results of a split contraction, slabs ascending, and the epilogue: V columns of a row per
// thread, eight slabs' loads in flight.  Eight columns where that leaves every CU threads; one where the
// output is small or its rows ragged (64 x 71 of 60 slabs 6 us, of 16 by eight columns 11).
template <int V>
__global__ void __launch_bounds__(256) k_linear_finish(const float* slabs, int S, long M, long N, unsigned chunks, Epi e) {
  const unsigned i = blockIdx.x * 256 + threadIdx.x, r = i / chunks;
  const long m = r, n = (long)(i - r * chunks) * V, at = m * N + n;
  if (m >= M) return;
  float v[V], t[V];
  load_f32<V>(slabs + at, v);
#pragma unroll 8
  for (int s = 1; s < S; ++s) {
    load_f32<V>(slabs + s * M * N + at, t);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] += t[j];
  }
  finish<V>(e, m, n, v);
}
inline int sum_slabs(const char* who, const float* slabs, int S, long M, long N, const Epi& e, hipStream_t st) {
  DD_REQUIRE(M * N < (1l << 32) - 256, "dd_linear: a split product of 2^32 outputs");
  const unsigned per = N % 8 == 0 && M * N >= 8 * 65536 ? 8 : 1, grid = (unsigned)((M * N / per + 255) / 256);
  if (per == 8) k_linear_finish<8><<<grid, 256, 0, st>>>(slabs, S, M, N, (unsigned)(N / 8), e);
  else k_linear_finish<1><<<grid, 256, 0, st>>>(slabs, S, M, N, (unsigned)N, e);
  DD_CHECK_LAUNCH(who);
  return 0;
}

// Splits of a contraction: none where the tiles alone fill the chip.
inline int pick_splits(long tiles, int ktiles, size_t slab_bytes, size_t ws_bytes) {
  if (tiles >= 256 || ktiles < 8) return 1;
  long s = min(512 / tiles, (long)ktiles / 4);
  while (s > 1 && slab_bytes * (size_t)s > ws_bytes) --s;
  return (int)max(s, 1l);
}

// Can the tiled kernel's copies read this operand?  Offsets within a tile stay below 2^31.
inline bool tileable(const Mat& a, bool rc, int es) { return (long)(rc ? 64 : 256) * a.ld * es < (1l << 30); }

// The tile shapes: how many tiles run at once on the chip, and what a step of 128 contraction bytes, the
// rest of a tile (start, epilogue), an activation and one more tensor in the epilogue (residual, pre-activation) take
// then, in microseconds (fitted to products of 2500 to 37500 rows).
// 256 x 256 is the fastest per output (1430 against 1140 TFLOP/s of 128 x 128, 8192^3); the small ones fill the
// chip with fewer rows and waste less in a last round (2500 x 2048 x 1536: 192 x 128 22, 128 x 128 26, 256 x 256
// 36 us; 2500 x 1024 x 1024: 13.5, 12.4, 21).  192 rows are for P by rows: the transposing reads' swizzle
// wants a power of two.
struct TileShape { int rows, cols, slots; float step, rest, act, tensor; };
constexpr TileShape SHAPES[] = {
    {256, 256, 256, 1.38f, 10.f, 4.5f, 5.5f}, {128, 128, 512, 0.96f, 4.5f, 1.2f, 1.5f}, {192, 128, 256, 0.62f, 6.5f, 1.5f, 2.5f}};

inline float epilogue_cost(const TileShape& t, const Epi& e) {
  return (e.act != DD_ACT_NONE ? t.act : 0.f) + ((e.res != nullptr) + (e.z != nullptr)) * t.tensor;
}
struct Plan { int shape, splits; float us; };
inline Plan plan_product(long M, long N, int ksteps, size_t slab_room, int shapes, const Epi& e) {
  Plan best{0, 1, 1e30f};
  for (int i = 0; i < shapes; ++i) {
    TileShape t = SHAPES[i];
    t.rest += epilogue_cost(t, e);
    const long tiles = ((M + t.rows - 1) / t.rows) * ((N + t.cols - 1) / t.cols);
    for (int s = 1; s <= 64 && s <= max(1, ksteps / 4); s = s < 4 ? s + 1 : s * 2) {
      if (s > 1 && sizeof(float) * (size_t)(M * N) * s > slab_room) break;
      const long wgs = tiles * s, full = wgs / t.slots, left = wgs % t.slots;
      const float steps = (float)((ksteps + s - 1) / s);
      // a last round with a CU to itself is faster per step
      const float last = left == 0 ? 0.f : t.rest + steps * t.step * (left <= t.slots / 2 && t.slots > 256 ? 0.65f : 1.f);
      float us = full * (t.step * steps + t.rest) + last;
      if (s > 1) us += 6.f + (float)(M * N) * s * 8.f / 3.5e6f;   // partial sums out and in, one more launch
      if (us < best.us) best = {i, s, us};
    }
  }
  return best;
}

template <int ES, bool P_RC, bool Q_RC, int BM, int BN, int WM, int WN>
int tiled(const char* who, Mat P, Mat Q, int K, int splits, const Epi& e, float* slabs, hipStream_t st) {
  const int bk = ROWB / ES, tm = dd_ceil_div(P.R, BM), tn = dd_ceil_div(Q.R, BN), ksteps = dd_ceil_div(K, bk);
  const int kspan = dd_ceil_div(ksteps, splits) * bk, parts = dd_ceil_div(K, kspan);
  DD_REQUIRE((long)tm * tn * parts < (1l << 31), "dd_linear: too many tiles");
  k_linear_tile<ES, P_RC, Q_RC, BM, BN, WM, WN><<<(unsigned)((long)tm * tn * parts), 64 * WM * WN, 0, st>>>(
      P, Q, K, kspan, tm, tn, parts > 1 ? slabs : nullptr, e);
  DD_CHECK_LAUNCH(who);
  return parts > 1 ? sum_slabs(who, slabs, parts, P.R, Q.R, e, st) : 0;
}

template <int ES, bool P_RC, bool Q_RC>
int planned(const char* who, const Mat& P, const Mat& Q, int K, const Plan& plan, const Epi& e, float* slabs, hipStream_t st) {
  if constexpr (!P_RC)
    if (plan.shape == 2) {   // (48 rows a wave are three of the 16 x 16 instruction's, but no whole number of 32)
      if constexpr (ES == 2) return tiled<ES, P_RC, Q_RC, 192, 128, 4, 2>(who, P, Q, K, plan.splits, e, slabs, st);
      else return tiled<ES, P_RC, Q_RC, 192, 128, 2, 4>(who, P, Q, K, plan.splits, e, slabs, st);
    }
  if (plan.shape == 1) return tiled<ES, P_RC, Q_RC, 128, 128, 4, 2>(who, P, Q, K, plan.splits, e, slabs, st);
  return tiled<ES, P_RC, Q_RC, 256, 256, 2, 4>(who, P, Q, K, plan.splits, e, slabs, st);
}
// Which kernels a product takes, all of it host logic: the launches follow it, and dd_linear_plan tells it.
struct Choice {
  enum Kernel { FEW, TILES, GENERAL } kernel;
  int few;           // FEW: sixteens of rows in the accumulators
  long cut;          // TILES: rows of a first launch (0: one launch does all)
  Plan head, rest;   // its plan, the other rows'
  int splits;        // GENERAL: of the contraction
};

// Tiles.  Where the last round of tiles would leave most of the chip idle, whole rounds take the first rows and a
// launch of its own, with a plan of its own, the rest (37500 x 1024 x 2048, 2.3 rounds: 149 -> 137 us, with a residual
// 167 -> 153, in e4m3 99 -> 92; dx of 37500 x 2048 x 1024 152 -> 137; dx of 5641 x 461 x 3597 43 -> 40).
inline void choose_rounds(Choice& c, const Mat& P, const Mat& Q, int ksteps, int shapes, const Epi& e, size_t room) {
  c.cut = 0;
  c.rest = plan_product(P.R, Q.R, ksteps, room, shapes, e);
  float best = 0.95f * c.rest.us;
  for (int i = 0; i < shapes; ++i) {
    const TileShape& t = SHAPES[i];
    const long tm = dd_ceil_div(P.R, t.rows), tn = dd_ceil_div(Q.R, t.cols), full = tm * tn / t.slots;
    const long rows = full * t.slots / tn * t.rows;   // of whole rounds
    if (full == 0 || rows == 0 || rows >= P.R) continue;
    const Plan rest = plan_product(P.R - rows, Q.R, ksteps, room, shapes, e);
    const float us = full * (t.step * ksteps + t.rest + epilogue_cost(t, e)) + rest.us + 2.f;
    if (us < best) { best = us; c.cut = rows; c.head = {i, 1, us}; c.rest = rest; }
  }
}

inline Choice choose(const Mat& P, const Mat& Q, int K, int es, bool p_rc, bool q_rc, const Epi& e, size_t room) {
  Choice c{};
  // Below 2^22 multiplications over a short contraction the general kernel's small tiles start and end sooner
  // (128 x 128 x 128 4.2 us against 5.4, 8 x 64 x 72 dw 4.4 against 5.1; 70 x 64 x 1000 8.5 either way).
  const bool small = (double)P.R * Q.R * K < 4194304.0 && (long)K * es < 8 * ROWB;
  const bool can_tile = K > 0 && tileable(P, p_rc, es) && tileable(Q, q_rc, es);
  // Few rows, as long as the weights' 16-row workgroups are a round or two of the chip: each reads all of x, and tiles
  // read it less often (8 x 16384 x 1024 7.3 us against 12.5 on tiles, 8 x 32768 x 1024 14.6 against 14.2; 64 x 8192
  // x 1024 7.6 and 11.5, 64 x 16384 x 1024 13.5 and 13.2; 128 x 4096 x 1024 7.7 and 11.5, 128 x 8192 x 1024 14.0 and 11.5;
  // long rows and 16 of x at most: the weights' read is all there is, 8 x 65536 x 4096 91 and 123).
  const unsigned grid = dd_ceil_div(Q.R, 16);
  const unsigned most = P.R <= 16 ? ((long)K * es >= 8192 ? 1u << 30 : 1024) : P.R <= 64 ? 512 : P.R <= 128 && !small ? 256 : 0;
  const int ksteps = dd_ceil_div(K, ROWB / es);
  if (!p_rc && !q_rc && grid <= most && can_tile) {
    c.kernel = Choice::FEW;
    c.few = P.R <= 16 ? 1 : P.R <= 32 ? 2 : P.R <= 64 ? 4 : 8;
  } else if (!small && can_tile && (!e.res || e.ldr < (1l << 20))) {
    c.kernel = Choice::TILES;
    choose_rounds(c, P, Q, ksteps, p_rc ? 2 : 3, e, room);
  } else {
    c.kernel = Choice::GENERAL;
    c.splits = pick_splits((long)dd_ceil_div(P.R, 64) * dd_ceil_div(Q.R, 64), ksteps, sizeof(float) * (size_t)P.R * Q.R, room);
  }
  return c;
}

template <int ES, bool P_RC, bool Q_RC>
int product(const char* who, Mat P, Mat Q, int K, const Epi& e, float* ws, size_t ws_bytes, hipStream_t st) {
  const Choice c = choose(P, Q, K, ES, P_RC, Q_RC, e, ws ? ws_bytes : 0);
  if (c.kernel == Choice::FEW) {
    if constexpr (!P_RC && !Q_RC) {
      const unsigned grid = dd_ceil_div(Q.R, 16);
      if (c.few == 1) k_linear_few<ES, 1, 8><<<grid, 512, 0, st>>>(P, Q, K, e);
      else if (c.few == 2) k_linear_few<ES, 2, 8><<<grid, 512, 0, st>>>(P, Q, K, e);
      else if (c.few == 4) k_linear_few<ES, 4, 4><<<grid, 256, 0, st>>>(P, Q, K, e);
      else k_linear_few<ES, 8, 4><<<grid, 256, 0, st>>>(P, Q, K, e);
      DD_CHECK_LAUNCH(who);
    }
    return 0;
  }
  if (c.kernel == Choice::TILES) {
    if (c.cut == 0) return planned<ES, P_RC, Q_RC>(who, P, Q, K, c.rest, e, ws, st);
    Mat p = P;
    p.R = (int)c.cut;
    if (const int rc = planned<ES, P_RC, Q_RC>(who, p, Q, K, c.head, e, ws, st)) return rc;
    p.p = (const char*)P.p + (P_RC ? c.cut : c.cut * P.ld) * ES;
    p.R = P.R - (int)c.cut;
    Epi f = e;
    const long es = e.ytype == DD_F32 ? 4 : 2;
    f.y = (char*)e.y + c.cut * e.ldy * es;
    if (e.res) f.res = (const char*)e.res + c.cut * e.ldr * es;
    if (e.z) f.z = e.z + c.cut * e.ldz;
    if (e.xs) f.xs = e.xs + c.cut;
    return planned<ES, P_RC, Q_RC>(who, p, Q, K, c.rest, f, ws, st);
  }
  const int bk = ROWB / ES, ktiles = dd_ceil_div(K, bk);
  const dim3 tiles(dd_ceil_div(P.R, 64), dd_ceil_div(Q.R, 64));
  DD_REQUIRE(tiles.y <= 65535, "dd_linear: more than 4194240 output columns");
  const int kspan = max(1, dd_ceil_div(ktiles, c.splits)) * bk, parts = max(1, dd_ceil_div(K, kspan));
  k_linear_any<ES, P_RC, Q_RC><<<dim3(tiles.x, tiles.y, parts), 256, 0, st>>>(P, Q, K, kspan, parts > 1 ? ws : nullptr, e);
  DD_CHECK_LAUNCH(who);
  return parts > 1 ? sum_slabs(who, ws, parts, P.R, Q.R, e, st) : 0;
}

// dz = dy act'(z), and the workgroup's share of dbias; without an activation dz IS dy and only the column
// sums are taken.  HBM-bound: a wave takes 512 columns of a row at a time (1 KB), or several rows of narrower
// matrices (`lanes` of it per row: 30237 x 64: 6 us against 14 with whole waves), four waves on different rows, four rows
// requested at a time.  Up to 256 rows a workgroup takes all rows of
// 64 columns and stores the sums itself, one launch less (110 x 2752 gelu 4.6 us against 6.8; 500 x 741 10 against
// 8.5).
// Columns c .. c + V - 1 of rows m0, m0 + step, ...; `seen` of them are counted by another lane.
template <int V, int ACT>
__device__ __forceinline__ void act_rows(const __bf16* dy, long ldy, const __bf16* z, long ldz, __bf16* dz, long lddz, long c,
                                         long m0, long m1, int step, int seen, float sum[V]) {
  constexpr int ROWS = 4;   // loaded together (dz may be dy or z: a store in between would hold the next loads up)
  for (long m = m0; m < m1; m += ROWS * step) {
    float d[ROWS][V], t[ROWS][V];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const long row = m + r * step < m1 ? m + r * step : m;
      load_bf16<V>(dy + row * ldy + c, d[r]);
      if constexpr (ACT != DD_ACT_NONE) load_bf16<V>(z + row * ldz + c, t[r]);
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      if (m + r * step >= m1) break;
      if constexpr (ACT != DD_ACT_NONE) {
#pragma unroll
        for (int j = 0; j < V; ++j) d[r][j] *= act_slope<ACT>(t[r][j]);
        // bf16: the two products that read dz take bf16 operands, as they take x and w (dx and dw are off by 1.7e-3 in
        // the 2-norm for it; a dz of two bf16 parts would be twice the products)
        store_bf16<V>(dz + (m + r * step) * lddz + c, d[r]);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += j < seen ? 0.f : d[r][j];
    }
  }
}
template <int ACT>
__global__ void __launch_bounds__(256) k_act_bwd(const __bf16* dy, long ldy, const __bf16* z, long ldz, __bf16* dz, long lddz,
                                                 float* parts, int M, int N, int rows_per, int lanes, void* dbias, int type,
                                                 int accumulate) {
  __shared__ float sh[4 * 512];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, apart = 64 / lanes;   // rows of a wave
  const long c = ((long)blockIdx.x * lanes + lane % lanes) * 8;
  const long m0 = (long)blockIdx.y * rows_per + wave * apart + lane / lanes, m1 = min((long)M, (blockIdx.y + 1l) * rows_per);
  float sum[8] = {};
  // A ragged row's last columns are those of a full vector that overlaps the lane before, in the same wave (another
  // workgroup might have written dz over dy there); only a wave's first lane takes them one by one.
  const int seen = c < N && c + 8 > N && lane % lanes != 0 ? (int)(c + 8 - N) : 0;
  if (c + 8 - seen <= N && c < N) {
    act_rows<8, ACT>(dy, ldy, z, ldz, dz, lddz, c - seen, m0, m1, 4 * apart, seen, sum);
  } else {
#pragma unroll 1
    for (int j = 0; c + j < N; ++j) {
      float t[1] = {0.f};
      act_rows<1, ACT>(dy, ldy, z, ldz, dz, lddz, c + j, m0, m1, 4 * apart, 0, t);
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] = k == j ? t[0] : sum[k];
    }
  }
  if (!parts && !dbias) return;
#pragma unroll
  for (int j = 0; j < 8; ++j)   // (8 - seen sums, from the lane's own first column)
    if (j >= seen) sh[threadIdx.x * 8 + j - seen] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 8 * lanes; i += 256) {   // waves and their rows in order
    const long col = (long)blockIdx.x * lanes * 8 + i;
    if (col >= N) continue;
    float t = sh[i];
#pragma unroll 4
    for (int r = 1; r < 4 * apart; ++r) t += sh[r * lanes * 8 + i];
    if (parts) parts[(long)blockIdx.y * N + col] = t;
    else if (type == DD_F32) { float* p = (float*)dbias + col; *p = accumulate ? *p + t : t; }
    else { __bf16* p = (__bf16*)dbias + col; *p = (__bf16)(accumulate ? (float)*p + t : t); }
  }
}

inline bool in_range(int M, int N, int K) {
  constexpr int MOST = 1 << 30;
  return M >= 0 && N > 0 && K > 0 && M <= MOST && N <= MOST && K <= MOST;
}

}  // namespace

extern "C" int dd_linear_fwd(const void* x, long ldx, const void* w, long ldw, int type, const float* x_scale,
                             const float* w_scale, const float* bias, int act, const void* res, long ldr, void* y, long ldy,
                             int y_type, void* z, long ldz, int M, int N, int K, float* ws, size_t ws_bytes, void* stream) {
  DD_REQUIRE(in_range(M, N, K), "dd_linear_fwd: M >= 0, N > 0 and K > 0 (2^30 at most) are needed");
  DD_REQUIRE(type == DD_BF16 || type == DD_E4M3, "dd_linear_fwd: x and w are bf16 or e4m3 (fp32: dd_gemm_f32)");
  DD_REQUIRE(y_type == DD_BF16 || y_type == DD_F32, "dd_linear_fwd: y is bf16 or fp32");
  DD_REQUIRE(act >= DD_ACT_NONE && act <= DD_ACT_GELU, "dd_linear_fwd: unknown activation");
  DD_REQUIRE((type == DD_E4M3) == (x_scale != nullptr) && (type == DD_E4M3) == (w_scale != nullptr),
             "dd_linear_fwd: x_scale and w_scale go with e4m3 operands, and only with them");
  if (M == 0) return 0;
  DD_REQUIRE(x && w && y, "dd_linear_fwd: null x, w or y");
  DD_REQUIRE(ldx >= K && ldw >= K && ldy >= N && (!res || ldr >= N) && (!z || ldz >= N), "dd_linear_fwd: a leading dimension is too small");
  const Mat P{x, ldx, M}, Q{w, ldw, N};
  Epi e{y, ldy, y_type, bias, act, res, ldr, (__bf16*)z, ldz, x_scale, w_scale, 0};
  if (type == DD_BF16) return product<2, false, false>("dd_linear_fwd", P, Q, K, e, ws, ws_bytes, (hipStream_t)stream);
  return product<1, false, false>("dd_linear_fwd", P, Q, K, e, ws, ws_bytes, (hipStream_t)stream);
}

// The operands of the three products as the entry points pass them on.
extern "C" int dd_linear_plan(int what, int type, int M, int N, int K, long ldp, long ldq, int act, long ldr, int z, size_t ws_bytes,
                              int* plan) {
  DD_REQUIRE(in_range(M, N, K) && M > 0, "dd_linear_plan: M, N, K > 0 (2^30 at most) are needed");
  DD_REQUIRE(type == DD_BF16 || type == DD_E4M3, "dd_linear_plan: bf16 or e4m3");
  DD_REQUIRE(what == 0 || ((what == 1 || what == 2) && type == DD_BF16), "dd_linear_plan: 0 forward, 1 data, 2 weight (bf16)");
  DD_REQUIRE(act >= DD_ACT_NONE && act <= DD_ACT_GELU && plan, "dd_linear_plan: unknown activation, or no plan");
  Epi e{};
  if (what == 0) {
    e.act = act;
    e.res = ldr ? plan : nullptr;   // (looked at, not read)
    e.ldr = ldr;
    e.z = z ? (__bf16*)plan : nullptr;
  }
  const Mat P{nullptr, ldp, what == 2 ? N : M}, Q{nullptr, ldq, what == 0 ? N : K};
  const Choice c = choose(P, Q, what == 0 ? K : what == 1 ? N : M, type == DD_BF16 ? 2 : 1, what == 2, what != 0, e, ws_bytes);
  for (int i = 0; i < 8; ++i) plan[i] = 0;
  plan[0] = c.kernel;
  if (c.kernel == Choice::FEW) plan[1] = 16 * c.few;
  if (c.kernel == Choice::GENERAL) plan[1] = c.splits;
  if (c.kernel == Choice::TILES) {
    const TileShape &h = SHAPES[c.head.shape], &r = SHAPES[c.rest.shape];
    plan[1] = r.rows; plan[2] = r.cols; plan[3] = c.rest.splits;
    if (c.cut) { plan[4] = (int)c.cut; plan[5] = h.rows; plan[6] = h.cols; plan[7] = c.head.splits; }
  }
  return 0;
}

extern "C" int dd_linear_bwd_data(const void* dz, long lddz, const void* w, long ldw, void* dx, long lddx, int x_type, int M,
                                  int N, int K, float* ws, size_t ws_bytes, void* stream) {
  DD_REQUIRE(in_range(M, N, K), "dd_linear_bwd_data: M >= 0, N > 0 and K > 0 (2^30 at most) are needed");
  DD_REQUIRE(x_type == DD_BF16 || x_type == DD_F32, "dd_linear_bwd_data: dx is bf16 or fp32");
  if (M == 0) return 0;
  DD_REQUIRE(dz && w && dx, "dd_linear_bwd_data: null pointer");
  DD_REQUIRE(lddz >= N && ldw >= K && lddx >= K, "dd_linear_bwd_data: a leading dimension is too small");
  const Mat P{dz, lddz, M}, Q{w, ldw, K};
  Epi e{dx, lddx, x_type};
  return product<2, false, true>("dd_linear_bwd_data", P, Q, N, e, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int dd_linear_bwd_weight(const void* dz, long lddz, const void* x, long ldx, void* dw, long lddw, int w_type,
                                    int accumulate, int M, int N, int K, float* ws, size_t ws_bytes, void* stream) {
  DD_REQUIRE(in_range(M, N, K), "dd_linear_bwd_weight: M >= 0, N > 0 and K > 0 (2^30 at most) are needed");
  DD_REQUIRE(w_type == DD_BF16 || w_type == DD_F32, "dd_linear_bwd_weight: dw is bf16 or fp32");
  if (M == 0 && accumulate) return 0;
  DD_REQUIRE(dw && (M == 0 || (dz && x)), "dd_linear_bwd_weight: null pointer");
  DD_REQUIRE(lddw >= K && (M == 0 || (lddz >= N && ldx >= K)), "dd_linear_bwd_weight: a leading dimension is too small");
  const Mat P{dz, lddz, N}, Q{x, ldx, K};
  Epi e{dw, lddw, w_type};
  e.accumulate = accumulate;
  return product<2, true, true>("dd_linear_bwd_weight", P, Q, M, e, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int dd_linear_act_bwd(const void* dy, long ldy, const void* z, long ldz, int act, void* dz, long lddz, void* dbias,
                                 int bias_type, int accumulate, int M, int N, float* ws, size_t ws_bytes, void* stream) {
  DD_REQUIRE(M >= 0 && N > 0, "dd_linear_act_bwd: M >= 0 and N > 0 are needed");
  DD_REQUIRE(act >= DD_ACT_NONE && act <= DD_ACT_GELU, "dd_linear_act_bwd: unknown activation");
  DD_REQUIRE(!dbias || bias_type == DD_F32 || bias_type == DD_BF16, "dd_linear_act_bwd: dbias is fp32 or bf16");
  const bool act_on = act != DD_ACT_NONE;
  if (!act_on && !dbias) return 0;
  if (M == 0 && (!dbias || accumulate)) return 0;
  DD_REQUIRE(M == 0 || (dy && ldy >= N), "dd_linear_act_bwd: dy is null or its leading dimension is below N");
  DD_REQUIRE(M == 0 || !act_on || (z && dz && ldz >= N && lddz >= N), "dd_linear_act_bwd: an activation needs z and dz");
  const hipStream_t st = (hipStream_t)stream;
  // 1024 workgroups, at least a row each for every row of lanes
  const bool whole = M <= 256;
  int lanes = whole ? 8 : 64;
  while (lanes > 1 && N <= 4 * lanes) lanes /= 2;
  const int cols = dd_ceil_div(N, 8 * lanes);
  const int rows_per = whole ? max(M, 1) : max(256 / lanes, dd_ceil_div(M, max(1, dd_ceil_div(1024, cols)))), n = dd_ceil_div(M, rows_per);
  DD_REQUIRE(n <= 65535, "dd_linear_act_bwd: too many rows");
  DD_REQUIRE(!dbias || ws_bytes / sizeof(float) >= (size_t)n * N, "dd_linear_act_bwd: the workspace is too small");
  if (M > 0) {
    const dim3 grid(cols, n);
#define DD_ACT_BWD(A_)                                                                                          \
  case A_:                                                                                                      \
    k_act_bwd<A_><<<grid, 256, 0, st>>>((const __bf16*)dy, ldy, (const __bf16*)z, ldz, (__bf16*)dz, lddz,       \
                                        dbias && !whole ? ws : nullptr, M, N, rows_per, lanes, dbias, bias_type,    \
                                        accumulate);                                                                \
    break;
    switch (act) { DD_ACT_BWD(DD_ACT_NONE) DD_ACT_BWD(DD_ACT_ELU) DD_ACT_BWD(DD_ACT_SILU) DD_ACT_BWD(DD_ACT_GELU) }
#undef DD_ACT_BWD
    DD_CHECK_LAUNCH("dd_linear_act_bwd");
  }
  if (dbias && !(whole && M > 0)) {
    k_part_sum<<<dd_ceil_div(N, 32), 1024, 0, st>>>(ws, n, N, dbias, bias_type, accumulate);
    DD_CHECK_LAUNCH("dd_linear_act_bwd(dbias)");
  }
  return 0;
}
