// Root-mean-square norm with the residual stream's addition, its backward pass, and rows quantised to
// e4m3 with a scale each: dd_rms_norm_fwd, dd_rms_norm_bwd, dd_quant_rows.
//
//   s = round(x + r)    y = s rstd gamma,  rstd = 1 / sqrt(mean(s^2) + eps)
//   ds = dres + rstd (dy gamma - n mean(dy gamma n)),  n = s rstd;   dgamma = sum over rows of dy n
//
// The norm reads the SUM AS IT IS STORED, so that the backward pass, which only has that, is the
// derivative of what the forward pass computed; all arithmetic is fp32.
//
// Bound: HBM.  A row's elements stay in registers from their load to the last store - each input is
// read once, each output written once - so a row belongs to a wave or a part of one, to four or to sixteen, in vectors
// of eight elements, up to four of them per lane.  Forward a wave takes rows up to 2048, four up to 8192.  The
// backward pass holds four rows' worth: a wave up to 1024, four up to 4096, with two vectors a lane (with four of them in
// fewer waves too few fit a CU: 20001 x 1542 101 us).  Sixteen waves take rows up to 32768, four vectors a lane past 16384.
// The last vector of a ragged row ends at the row's end and so overlaps the one before it: both lanes hold and store the
// same values there, the sums over a row count them once.  (Element by element, its loads came one round trip after
// the other: 20001 x 1542 bf16, backward, 141 us; now 60, at the 52 of its bytes.)
#include "block_core.h"

namespace {

struct RmsArgs {
  const void* x; long ldx; int xt;
  const void* r; long ldr; int rt;
  void* s; long lds;
  const float* gamma;
  void* y; long ldy; int yt;
  float* rstd; float* scale;
  int rows, C; float eps;
};

// Where vector i of lane l starts in a row of C, and how many of its elements belong to the vector before;
// `on`: there is such a vector.  Rows shorter than a vector are read element by element.
struct Place { int at, dup; bool on; };
__device__ __forceinline__ Place place(int i, int l, int stride, int C) {
  const int c = (l + stride * i) * 8;
  const int over = C >= 8 ? max(0, c + 8 - C) : 0;
  return {c - over, over, c < C};
}

template <typename T, int NC>
__device__ __forceinline__ void load_as(const T* p, int l, int stride, int C, float v[NC][8]) {
  if (C >= 8) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const Place q = place(i, l, stride, C);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      if (q.on) {
        if constexpr (sizeof(T) == 4) load_f32<8>(p + q.at, v[i]);
        else load_bf16<8>(p + q.at, v[i]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = i == 0 && l == 0 && j < C ? (float)p[j] : 0.f;
  }
}
template <int NC>
__device__ __forceinline__ void load_row(const void* base, int type, long off, int l, int stride, int C, float v[NC][8]) {
  if (type == DD_F32) load_as<float, NC>((const float*)base + off, l, stride, C, v);
  else load_as<__bf16, NC>((const __bf16*)base + off, l, stride, C, v);
}

template <int V>
__device__ __forceinline__ void store_as(void* base, int type, long at, const float* v) {
  if (type == DD_F32) store_f32<V>((float*)base + at, v);
  else if (type == DD_BF16) store_bf16<V>((__bf16*)base + at, v);
  else store_e4m3<V>((unsigned char*)base + at, v);
}
template <int NC>
__device__ __forceinline__ void store_row(void* base, int type, long off, int l, int stride, int C, const float v[NC][8]) {
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const Place q = place(i, l, stride, C);
    if (!q.on) continue;
    if (C >= 8) store_as<8>(base, type, off + q.at, v[i]);
    else
      for (int j = 0; j < C; ++j) store_as<1>(base, type, off + j, &v[i][j]);
  }
}

// Sum (MAX: maximum) over the lanes of a row: a part of a wave, one wave, or the whole workgroup.
template <bool MAX>
__device__ __forceinline__ float row_reduce(float v, int per, float* red) {
  if (per < 64) {
    for (int d = per / 2; d > 0; d /= 2) {
      const float o = __shfl_xor(v, d);
      v = MAX ? fmaxf(v, o) : v + o;
    }
    return v;
  }
  v = MAX ? wave_max(v) : wave_sum(v);
  if (per == 64) return v;
  // What this wave read is in registers before another wave stores it (s over res: vectors overlap).
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();   // the previous reduction's values have been read
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float t = red[0];
  for (int w = 1; w < per / 64; ++w) t = MAX ? fmaxf(t, red[w]) : t + red[w];
  return t;
}

template <int NC, bool NORM, int THREADS>
__global__ void __launch_bounds__(THREADS) k_rms_fwd(RmsArgs a, int per) {
  __shared__ float red[16];
  const int l = threadIdx.x % per;
  const long row = (long)blockIdx.x * (blockDim.x / per) + threadIdx.x / per;
  if (row >= a.rows) return;   // all lanes of a row; a row of several waves has its workgroup for itself
  float v[NC][8], t[NC][8];
  load_row<NC>(a.x, a.xt, row * a.ldx, l, per, a.C, v);
  if (a.r) {
    load_row<NC>(a.r, a.rt, row * a.ldr, l, per, a.C, t);
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] += t[i][j];
  }
  if constexpr (NORM) {
    if (a.s && a.rt == DD_BF16)
#pragma unroll
      for (int i = 0; i < NC; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = (float)(__bf16)v[i][j];
    float ss = 0.f;
    load_row<NC>(a.gamma, DD_F32, 0, l, per, a.C, t);
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int dup = place(i, l, per, a.C).dup;
#pragma unroll
      for (int j = 0; j < 8; ++j) ss += j >= dup ? v[i][j] * v[i][j] : 0.f;
    }
    const float rstd = 1.0f / sqrtf(row_reduce<false>(ss, per, red) / (float)a.C + a.eps);
    if (a.s) store_row<NC>(a.s, a.rt, row * a.lds, l, per, a.C, v);
    if (a.rstd && l == 0) a.rstd[row] = rstd;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] *= rstd * t[i][j];
  }
  if (a.yt == DD_E4M3) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, fabsf(v[i][j]));
    m = row_reduce<true>(m, per, red);
    // a row of zeros is stored as zeros with scale 1; one so small that 448 / m would overflow is brought up by an exact
    // power of two first (its scale may be subnormal, and is rounded as those are)
    const float up = m < 0x1p-100f ? 0x1p64f : 1.0f, inv = m > 0.f ? E4M3_MAX / (m * up) : 1.0f;
    if (l == 0) a.scale[row] = m > 0.f ? m / E4M3_MAX : 1.0f;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float t = v[i][j] * up * inv;   // at most 448 but for the roundings; a NaN stays one
        v[i][j] = t > E4M3_MAX ? E4M3_MAX : t < -E4M3_MAX ? -E4M3_MAX : t;
      }
  }
  store_row<NC>(a.y, a.yt, row * a.ldy, l, per, a.C, v);
}

struct RmsBwdArgs {
  const void* dy; long ldy; int yt;
  const void* s; long lds; int rt;
  const void* dres; long ldr;
  void* ds; long ldd;
  const float* rstd; const float* gamma;
  float* parts;   // [gridDim.x][C] or NULL
  int rows, C;
};

// A workgroup strides over the rows; every lane keeps its columns' share of dgamma in registers, the
// four waves of a workgroup are added in LDS, one partial row per workgroup goes to the workspace.
template <int NC, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 4 : NC == 1 ? 6 : 4) k_rms_bwd(RmsBwdArgs a, int per) {
  extern __shared__ float sh[];   // 16 reduction slots | (a wave or less per row) [rows][C] partial sums
  const int l = threadIdx.x % per, rpb = blockDim.x / per, slot = threadIdx.x / per;
  float g[NC][8], pg[NC][8] = {};
  load_row<NC>(a.gamma, DD_F32, 0, l, per, a.C, g);
  for (long row = (long)blockIdx.x * rpb + slot; row < a.rows; row += (long)gridDim.x * rpb) {
    float dy[NC][8], n[NC][8], dr[NC][8] = {};
    load_row<NC>(a.dy, a.yt, row * a.ldy, l, per, a.C, dy);
    load_row<NC>(a.s, a.rt, row * a.lds, l, per, a.C, n);
    if (a.dres) load_row<NC>(a.dres, a.rt, row * a.ldr, l, per, a.C, dr);
    const float rstd = a.rstd[row];
    float s1 = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int dup = place(i, l, per, a.C).dup;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[i][j] *= rstd;
        pg[i][j] += dy[i][j] * n[i][j];
        dy[i][j] *= g[i][j];
        s1 += j >= dup ? dy[i][j] * n[i][j] : 0.f;
      }
    }
    s1 = row_reduce<false>(s1, per, sh) / (float)a.C;
#pragma unroll
    for (int i = 0; i < NC; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) dy[i][j] = dr[i][j] + rstd * (dy[i][j] - n[i][j] * s1);
    store_row<NC>(a.ds, a.rt, row * a.ldd, l, per, a.C, dy);
  }
  if (!a.parts) return;
  float* out = a.parts + (long)blockIdx.x * a.C;
  if (per > 64) {
    store_row<NC>(out, DD_F32, 0, l, per, a.C, pg);
    return;
  }
  float* acc = sh + 16;
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    const Place q = place(i, l, per, a.C);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (q.on && q.at + j < a.C) acc[slot * a.C + q.at + j] = pg[i][j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < a.C; c += blockDim.x) {
    float t = acc[c];
    for (int w = 1; w < rpb; ++w) t += acc[w * a.C + c];
    out[c] = t;
  }
}

// Waves per row and vectors per lane; wpr 0: too wide.  The backward pass keeps four rows' worth of a lane's
// elements in registers: two vectors of a lane at most below 16384 columns.  The forward pass takes the shape
// that leaves the fewest lanes idle (16384 x 1088 to e4m3: 24 us with four waves a row, 17 with three vectors).
struct Shape { int wpr, nc; };
inline Shape row_shape(int C, bool forward) {
  Shape best{0, 0};
  for (int wpr = 1; wpr <= 16; wpr *= 4)
    for (int nc = 1; nc <= 4; ++nc) {
      if (C > 512 * wpr * nc || (wpr == 16 && nc == 3) || (!forward && nc > 2 && wpr < 16)) continue;
      if (!best.wpr || (forward && wpr * nc < best.wpr * best.nc)) best = {wpr, nc};
    }
  return best;
}

// Lanes of a row: all of its waves', or the power of two that holds a narrow row, several of which share a wave
// then (31849 x 64: forward 14.8 us with a wave each, 6.2 so; backward 17.1 and 11.3).
inline int row_lanes(const Shape& sh, int C) {
  int per = 64 * sh.wpr;
  while (per > 8 && C <= 4 * per) per /= 2;
  return per;
}

template <bool NORM>
int launch_fwd(const RmsArgs& a, hipStream_t st) {
  const Shape sh = row_shape(a.C, true);
  DD_REQUIRE(sh.wpr > 0, "dd_rms_norm_fwd / dd_quant_rows: more than 32768 columns");
  const int threads = sh.wpr == 16 ? 1024 : 256, per = row_lanes(sh, a.C), rpb = threads / per;
  const dim3 grid(dd_ceil_div(a.rows, rpb));
#define DD_RMS_FWD(N_, T_) \
  if (sh.nc == N_ && threads == T_) { k_rms_fwd<N_, NORM, T_><<<grid, T_, 0, st>>>(a, per); }
  DD_RMS_FWD(1, 256) DD_RMS_FWD(2, 256) DD_RMS_FWD(3, 256) DD_RMS_FWD(4, 256) DD_RMS_FWD(2, 1024) DD_RMS_FWD(4, 1024)
#undef DD_RMS_FWD
  DD_CHECK_LAUNCH(NORM ? "dd_rms_norm_fwd" : "dd_quant_rows");
  return 0;
}

inline bool real_type(int t) { return t == DD_F32 || t == DD_BF16; }

}  // namespace

extern "C" int dd_rms_norm_fwd(const void* x, long ldx, int x_type, const void* res, long ldr, int res_type,
                               void* s, long lds, const float* gamma, void* y, long ldy, int y_type,
                               float* rstd, float* scale, int rows, int C, float eps, void* stream) {
  DD_REQUIRE(rows >= 0 && C > 0, "dd_rms_norm_fwd: rows >= 0 and C > 0 are needed");
  DD_REQUIRE(real_type(x_type) && real_type(res_type), "dd_rms_norm_fwd: x and res are fp32 or bf16");
  DD_REQUIRE(real_type(y_type) || y_type == DD_E4M3, "dd_rms_norm_fwd: y is fp32, bf16 or e4m3");
  DD_REQUIRE((y_type == DD_E4M3) == (scale != nullptr), "dd_rms_norm_fwd: scale goes with an e4m3 y, and only with it");
  if (rows == 0) return 0;
  DD_REQUIRE(x && gamma && y, "dd_rms_norm_fwd: null x, gamma or y");
  DD_REQUIRE(ldx >= C && ldy >= C && (!res || ldr >= C) && (!s || lds >= C), "dd_rms_norm_fwd: a leading dimension below C");
  DD_REQUIRE(s || !res, "dd_rms_norm_fwd: res without s (the sum is what the next block and the backward pass read)");
  const RmsArgs a{x, ldx, x_type, res, ldr, res_type, s, lds, gamma, y, ldy, y_type, rstd, scale, rows, C, eps};
  return launch_fwd<true>(a, (hipStream_t)stream);
}

extern "C" int dd_quant_rows(const void* x, long ldx, int x_type, void* q, long ldq, float* scale, int rows, int C,
                             void* stream) {
  DD_REQUIRE(rows >= 0 && C > 0, "dd_quant_rows: rows >= 0 and C > 0 are needed");
  DD_REQUIRE(real_type(x_type), "dd_quant_rows: x is fp32 or bf16");
  if (rows == 0) return 0;
  DD_REQUIRE(x && q && scale, "dd_quant_rows: null pointer");
  DD_REQUIRE(ldx >= C && ldq >= C, "dd_quant_rows: a leading dimension below C");
  const RmsArgs a{x, ldx, x_type, nullptr, 0, DD_F32, nullptr, 0, nullptr, q, ldq, DD_E4M3, nullptr, scale, rows, C, 0.f};
  return launch_fwd<false>(a, (hipStream_t)stream);
}

extern "C" int dd_rms_norm_bwd(const void* dy, long ldy, int y_type, const void* s, long lds, int res_type,
                               const float* rstd, const float* gamma, const void* dres, long ldr, void* ds, long ldd,
                               float* dgamma, int accumulate, int rows, int C, float* ws, size_t ws_bytes, void* stream) {
  DD_REQUIRE(rows >= 0 && C > 0, "dd_rms_norm_bwd: rows >= 0 and C > 0 are needed");
  DD_REQUIRE(real_type(y_type) && real_type(res_type), "dd_rms_norm_bwd: dy and s are fp32 or bf16");
  const hipStream_t st = (hipStream_t)stream;
  if (rows == 0 && (!dgamma || accumulate)) return 0;
  DD_REQUIRE(rows == 0 || (dy && s && rstd && gamma && ds), "dd_rms_norm_bwd: null pointer");
  DD_REQUIRE(rows == 0 || (ldy >= C && lds >= C && ldd >= C && (!dres || ldr >= C)), "dd_rms_norm_bwd: a leading dimension below C");
  const Shape sh = row_shape(C, false);
  DD_REQUIRE(sh.wpr > 0, "dd_rms_norm_bwd: more than 32768 columns");
  const int threads = sh.wpr == 16 ? 1024 : 256, per = row_lanes(sh, C), rpb = threads / per;
  // as many workgroups as are resident at once (more leave a ragged last round: 20001 x 1542 with 768, 1024,
  // 1536 workgroups 90, 76, 63 us; 20000 x 1024, two vectors a lane, 59, 60, 66)
  const int grid = min(dd_ceil_div(rows, rpb), threads == 1024 ? 256 : sh.nc == 1 ? 1536 : 768);
  DD_REQUIRE(!dgamma || ws_bytes / sizeof(float) >= (size_t)grid * C, "dd_rms_norm_bwd: the workspace is too small");
  if (grid > 0) {
    const RmsBwdArgs a{dy, ldy, y_type, s, lds, res_type, dres, ldr, ds, ldd, rstd, gamma, dgamma ? ws : nullptr, rows, C};
    const size_t lds_bytes = (16 + (per <= 64 && dgamma ? (size_t)rpb * C : 0)) * sizeof(float);
#define DD_RMS_BWD(N_, T_) \
  if (sh.nc == N_ && threads == T_) { k_rms_bwd<N_, T_><<<grid, T_, lds_bytes, st>>>(a, per); }
    DD_RMS_BWD(1, 256) DD_RMS_BWD(2, 256) DD_RMS_BWD(1, 1024) DD_RMS_BWD(2, 1024) DD_RMS_BWD(4, 1024)
#undef DD_RMS_BWD
    DD_CHECK_LAUNCH("dd_rms_norm_bwd");
  }
  if (dgamma) {
    k_part_sum<<<dd_ceil_div(C, 32), 1024, 0, st>>>(ws, grid, C, dgamma, DD_F32, accumulate);
    DD_CHECK_LAUNCH("dd_rms_norm_bwd(dgamma)");
  }
  return 0;
}
