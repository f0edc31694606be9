// Gated recurrence that is linear in its state, all time steps of a batch of sequences as one scan,
// and its backward pass: dd_gated_scan_fwd, dd_gated_scan_bwd.
//
//   v = u + shift;  a = sigmoid(-v), 0 where the sequence starts anew;  b = gate * phi(c),
//   gate = sigmoid(v) (the blend of a GRU cell) or sigmoid(i);  h[t] = a[t] h[t-1] + b[t]
//   backward: G[t] = a[t] (dh[t] + G[t+1]) runs the same scan from the end, G[T] = dhT, dh0 = G[0]
//
// A step is the map x -> A x + B; maps compose associatively, so a workgroup's waves take consecutive
// runs of STEPS time steps of the same channels, compose their run, exchange the pairs in LDS and then
// run their steps from the state that reaches them: a step's operands are read once and its a, b stay
// in registers.  Few sequences with many steps: the time axis is split over workgroups as well, whose
// pairs a first launch puts into the workspace.
//
// A restart is A == 0 EXACTLY and cuts whatever came before, non-finite values too (0 * NaN would
// not); every other factor is kept at or above FLT_MIN, so that a product that underflows does not look
// like a restart and a NaN in the state is not lost.  State, pairs and all arithmetic are fp32.
#include "block_core.h"
#include <float.h>

namespace {

constexpr int STEPS = 8;   // time steps of one wave between two exchanges

struct ScanArgs {
  const void* u; long ldu;
  const void* c; long ldc;
  const void* i; long ldi;          // input gate, NULL: sigmoid(v)
  const float* first; long fstride; // NULL: no restarts
  const float* x0;                  // h0 (forward), dhT (backward); NULL: zeros
  float* xT;                        // hT, dh0; NULL: not wanted
  void* h; long ldh;                // forward: out; backward: the stored states
  const float* h0;                  // backward: the initial state
  const void* dh; long lddh;
  void* du; long lddu; void* dc; long lddc; void* di; long lddi;
  float2* pairs;                    // [B][splits][D] of a split time axis
  int B, T, D, groups, splits, span;
  float shift; int tanh_c;
};

template <typename E, int VC>
__device__ __forceinline__ void ld(const void* p, long off, float v[VC]) {
  if constexpr (sizeof(E) == 4) load_f32<VC>((const float*)p + off, v);
  else load_bf16<VC>((const __bf16*)p + off, v);
}
template <typename E, int VC>
__device__ __forceinline__ void st(void* p, long off, const float v[VC]) {
  if constexpr (sizeof(E) == 4) store_f32<VC>((float*)p + off, v);
  else store_bf16<VC>((__bf16*)p + off, v);
}

__device__ __forceinline__ float at_least_min(float a) { return a < FLT_MIN ? FLT_MIN : a; }
__device__ __forceinline__ float apply(float A, float B, float x) { return A == 0.f ? B : __builtin_fmaf(A, x, B); }
// (A2, B2) after (A1, B1), into (A1, B1)
__device__ __forceinline__ void compose(float& A1, float& B1, float A2, float B2) {
  B1 = apply(A2, B2, B1);
  A1 = (A1 == 0.f || A2 == 0.f) ? 0.f : at_least_min(A1 * A2);
}

// decay and gate of one element
__device__ __forceinline__ void gates(float v, bool restart, float& a, float& z) {
  float q;
  sigmoid2(v, z, q);
  a = restart ? 0.f : at_least_min(q);
}
__device__ __forceinline__ float sigmoid1(float x) { float p, q; sigmoid2(x, p, q); return p; }

// The pair of one element's step: forward b from the gates, backward a * dh.
template <typename E, int VC, bool GATE, bool BWD>
__device__ __forceinline__ void step_pair(const ScanArgs& p, long row, int d, bool restart, float a[VC], float b[VC]) {
  float u[VC], z[VC];
  ld<E, VC>(p.u, row * p.ldu + d, u);
#pragma unroll
  for (int j = 0; j < VC; ++j) gates(u[j] + p.shift, restart, a[j], z[j]);
  if constexpr (BWD) {
    ld<E, VC>(p.dh, row * p.lddh + d, b);
#pragma unroll
    for (int j = 0; j < VC; ++j) b[j] = a[j] * b[j];
  } else {
    float c[VC], i[VC];
    ld<E, VC>(p.c, row * p.ldc + d, c);
    if constexpr (GATE) ld<E, VC>(p.i, row * p.ldi + d, i);
#pragma unroll
    for (int j = 0; j < VC; ++j) b[j] = (GATE ? sigmoid1(i[j]) : z[j]) * (p.tanh_c ? tanh_f(c[j]) : c[j]);
  }
}

// First launch of a split time axis: the pairs of all splits but the last (in scan order), and in
// slot 0 the initial state as a restart, so that a state updated in place is read before it is written.
template <typename E, int VC, bool GATE, bool BWD>
__global__ void __launch_bounds__(256) k_scan_pairs(ScanArgs p) {
  __shared__ float2 sh[4][64 * VC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int k = blockIdx.x % (p.splits - 1), g = (blockIdx.x / (p.splits - 1)) % p.groups;
  const long b = blockIdx.x / (p.splits - 1) / p.groups;
  const int d = (g * 64 + lane) * VC;
  const bool live = d < p.D;
  const int len = p.span / 4;   // this wave's run, in scan order
  float A[VC], Bv[VC];
#pragma unroll
  for (int j = 0; j < VC; ++j) { A[j] = 1.f; Bv[j] = 0.f; }
  if (live)
#pragma unroll 4
    for (int s = 0; s < len; ++s) {
      const int o = k * p.span + wave * len + s;   // the last split is not here: o < T
      const int t = BWD ? p.T - 1 - o : o;
      const long row = b * p.T + t;
      float a[VC], bb[VC];
      step_pair<E, VC, GATE, BWD>(p, row, d, p.first && p.first[row * p.fstride] != 0.f, a, bb);
#pragma unroll
      for (int j = 0; j < VC; ++j) compose(A[j], Bv[j], a[j], bb[j]);
    }
#pragma unroll
  for (int j = 0; j < VC; ++j) sh[wave][lane * VC + j] = make_float2(A[j], Bv[j]);
  __syncthreads();
  if (wave == 0 && live)
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      for (int w = 1; w < 4; ++w) compose(A[j], Bv[j], sh[w][lane * VC + j].x, sh[w][lane * VC + j].y);
      float2* out = p.pairs + b * p.splits * p.D + d + j;
      out[(long)(k + 1) * p.D] = make_float2(A[j], Bv[j]);
      if (k == 0) out[0] = make_float2(0.f, p.x0 ? p.x0[b * p.D + d + j] : 0.f);
    }
}

// State at the start of split k of (b, d): the initial one, or the composed pairs of what precedes it.
template <int VC>
__device__ __forceinline__ void start_state(const ScanArgs& p, long b, int k, int d, float x[VC]) {
#pragma unroll
  for (int j = 0; j < VC; ++j) x[j] = 0.f;
  if (p.splits == 1) {
    if (p.x0) load_f32<VC>(p.x0 + b * p.D + d, x);
    return;
  }
  for (int s = 0; s <= k; ++s) {
    const float2* q = p.pairs + (b * p.splits + s) * p.D + d;
#pragma unroll
    for (int j = 0; j < VC; ++j) x[j] = apply(q[j].x, q[j].y, x[j]);
  }
}

// A wave's pair into LDS; returns the state that reaches this wave and moves `x` past all waves.
template <int VC>
__device__ __forceinline__ void exchange(float2 (*sh)[64 * VC], int wave, int waves, int lane, const float A[VC],
                                         const float B[VC], float x[VC], float in[VC]) {
  if (waves == 1) {
#pragma unroll
    for (int j = 0; j < VC; ++j) { in[j] = x[j]; x[j] = apply(A[j], B[j], x[j]); }
    return;
  }
#pragma unroll
  for (int j = 0; j < VC; ++j) sh[wave][lane * VC + j] = make_float2(A[j], B[j]);
  __syncthreads();
  for (int w = 0; w < waves; ++w)
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      if (w == wave) in[j] = x[j];
      const float2 q = sh[w][lane * VC + j];
      x[j] = apply(q.x, q.y, x[j]);
    }
}

template <typename E, int VC, bool GATE>
__global__ void __launch_bounds__(256) k_scan_fwd(ScanArgs p) {
  __shared__ float2 sh[2][4][64 * VC];   // two buffers: one barrier per exchange
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int k = blockIdx.x % p.splits, g = (blockIdx.x / p.splits) % p.groups;
  const long b = blockIdx.x / p.splits / p.groups;
  const int d = min((g * 64 + lane) * VC, p.D - VC);   // lanes past the last channel repeat it, and store nothing
  const bool live = (g * 64 + lane) * VC < p.D;
  const int end = min(p.T, (k + 1) * p.span);
  float x[VC];
  start_state<VC>(p, b, k, d, x);
  int buf = 0;
  for (int base = k * p.span; base < end; base += waves * STEPS, buf ^= 1) {
    float a[STEPS][VC], bb[STEPS][VC], A[VC], Bv[VC], in[VC];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int t = base + wave * STEPS + s;
      const long row = b * p.T + min(t, end - 1);
      step_pair<E, VC, GATE, false>(p, row, d, p.first && p.first[row * p.fstride] != 0.f, a[s], bb[s]);
#pragma unroll
      for (int j = 0; j < VC; ++j)
        if (t >= end) { a[s][j] = 1.f; bb[s][j] = 0.f; }
    }
#pragma unroll
    for (int j = 0; j < VC; ++j) { A[j] = a[0][j]; Bv[j] = bb[0][j]; }
#pragma unroll
    for (int s = 1; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < VC; ++j) compose(A[j], Bv[j], a[s][j], bb[s][j]);
    exchange<VC>(sh[buf], wave, waves, lane, A, Bv, x, in);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int t = base + wave * STEPS + s;
#pragma unroll
      for (int j = 0; j < VC; ++j) in[j] = apply(a[s][j], bb[s][j], in[j]);
      if (live && t < end) st<E, VC>(p.h, (b * p.T + t) * p.ldh + d, in);
    }
  }
  if (p.xT && live && k == p.splits - 1 && wave == 0) store_f32<VC>(p.xT + b * p.D + d, x);
}

template <typename E, int VC, bool GATE>
__global__ void __launch_bounds__(256) k_scan_bwd(ScanArgs p) {
  __shared__ float2 sh[2][4][64 * VC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int k = blockIdx.x % p.splits, g = (blockIdx.x / p.splits) % p.groups;
  const long b = blockIdx.x / p.splits / p.groups;
  const int d = min((g * 64 + lane) * VC, p.D - VC);
  const bool live = (g * 64 + lane) * VC < p.D;
  const int end = min(p.T, (k + 1) * p.span);   // in scan order: o = T - 1 - t
  float x[VC];
  start_state<VC>(p, b, k, d, x);
  int buf = 0;
  for (int base = k * p.span; base < end; base += waves * STEPS, buf ^= 1) {
    float u[STEPS][VC], dh[STEPS][VC], c[STEPS][VC], gi[STEPS][VC], hp[STEPS][VC], A[VC], Bv[VC], in[VC];
    bool restart[STEPS];
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int t = p.T - 1 - min(base + wave * STEPS + s, end - 1);
      const long row = b * p.T + t;
      ld<E, VC>(p.u, row * p.ldu + d, u[s]);
      ld<E, VC>(p.dh, row * p.lddh + d, dh[s]);
      ld<E, VC>(p.c, row * p.ldc + d, c[s]);
      if constexpr (GATE) ld<E, VC>(p.i, row * p.ldi + d, gi[s]);
      if (t > 0) {
        ld<E, VC>(p.h, (row - 1) * p.ldh + d, hp[s]);
      } else {
#pragma unroll
        for (int j = 0; j < VC; ++j) hp[s][j] = 0.f;
        if (p.h0) load_f32<VC>(p.h0 + b * p.D + d, hp[s]);
      }
      restart[s] = p.first && p.first[row * p.fstride] != 0.f;
    }
#pragma unroll
    for (int j = 0; j < VC; ++j) { A[j] = 1.f; Bv[j] = 0.f; }
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      if (base + wave * STEPS + s < end)
#pragma unroll
        for (int j = 0; j < VC; ++j) {
          float a, z;
          gates(u[s][j] + p.shift, restart[s], a, z);
          compose(A[j], Bv[j], a, a * dh[s][j]);
        }
    exchange<VC>(sh[buf], wave, waves, lane, A, Bv, x, in);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      const int o = base + wave * STEPS + s;
      if (o < end) {
        float du[VC], dc[VC], di[VC];
#pragma unroll
        for (int j = 0; j < VC; ++j) {
          float z, q;
          sigmoid2(u[s][j] + p.shift, z, q);
          const float a = restart[s] ? 0.f : at_least_min(q);
          const float gr = dh[s][j] + in[j];             // d loss / d h[t]
          in[j] = a == 0.f ? 0.f : a * gr;
          const float phi = p.tanh_c ? tanh_f(c[s][j]) : c[s][j];
          const float slope = p.tanh_c ? 1.f - phi * phi : 1.f;
          const float before = restart[s] ? 0.f : hp[s][j];
          if constexpr (GATE) {
            float w, wq;
            sigmoid2(gi[s][j], w, wq);
            du[j] = -gr * before * z * q;
            di[j] = gr * phi * w * wq;
            dc[j] = gr * w * slope;
          } else {
            du[j] = gr * (phi - before) * z * q;
            dc[j] = gr * z * slope;
          }
        }
        if (live) {
          const long row = b * p.T + p.T - 1 - o;
          st<E, VC>(p.du, row * p.lddu + d, du);
          st<E, VC>(p.dc, row * p.lddc + d, dc);
          if constexpr (GATE) st<E, VC>(p.di, row * p.lddi + d, di);
        }
      }
    }
  }
  if (p.xT && live && k == p.splits - 1 && wave == 0) store_f32<VC>(p.xT + b * p.D + d, x);
}

// Splits of the time axis: none where the channels alone give every CU a workgroup; else enough for
// four workgroups per CU, each at least two exchanges (64 steps) long.
inline void plan(ScanArgs& p) {
  const long wgs = (long)p.B * p.groups;
  p.splits = 1;
  p.span = p.T;
  if (wgs < 256 && p.T >= 128) {
    const long want = min((1024 + wgs - 1) / wgs, (long)p.T / 64);
    p.span = dd_ceil_div(dd_ceil_div(p.T, want), 32) * 32;
    p.splits = dd_ceil_div(p.T, p.span);
    if (p.splits == 1) p.span = p.T;
  }
}

template <typename E, int VC, bool GATE, bool BWD>
int launch(ScanArgs& p, float* ws, size_t ws_bytes, hipStream_t stream) {
  p.groups = dd_ceil_div(p.D, 64 * VC);
  plan(p);
  const long wgs = (long)p.B * p.groups * p.splits;
  DD_REQUIRE(wgs < (1l << 31), "dd_gated_scan: too many sequences");
  if (p.splits > 1) {
    DD_REQUIRE(ws_bytes >= sizeof(float2) * (size_t)p.B * p.splits * p.D, "dd_gated_scan: the workspace is too small");
    DD_REQUIRE((uintptr_t)ws % 8 == 0, "dd_gated_scan: the workspace is not 8-byte aligned");
    p.pairs = (float2*)ws;
    k_scan_pairs<E, VC, GATE, BWD><<<(unsigned)((long)p.B * p.groups * (p.splits - 1)), 256, 0, stream>>>(p);
    DD_CHECK_LAUNCH("dd_gated_scan(pairs)");
  }
  const int threads = p.T <= STEPS ? 64 : 256;
  if constexpr (BWD) k_scan_bwd<E, VC, GATE><<<(unsigned)wgs, threads, 0, stream>>>(p);
  else k_scan_fwd<E, VC, GATE><<<(unsigned)wgs, threads, 0, stream>>>(p);
  DD_CHECK_LAUNCH(BWD ? "dd_gated_scan_bwd" : "dd_gated_scan_fwd");
  return 0;
}

template <bool BWD>
int dispatch(ScanArgs& p, int type, float* ws, size_t ws_bytes, hipStream_t st) {
  const int w = 2 * dtype_size(type);
  const bool pair = p.D % 2 == 0 && rows_aligned(p.u, p.ldu, type, w) && rows_aligned(p.c, p.ldc, type, w) &&
                    rows_aligned(p.i, p.ldi, type, w) && rows_aligned(p.h, p.ldh, type, w) &&
                    rows_aligned(p.dh, p.lddh, type, w) && rows_aligned(p.du, p.lddu, type, w) &&
                    rows_aligned(p.dc, p.lddc, type, w) && rows_aligned(p.di, p.lddi, type, w) &&
                    rows_aligned(p.x0, 0, DD_F32, 8) && rows_aligned(p.xT, 0, DD_F32, 8) && rows_aligned(p.h0, 0, DD_F32, 8);
#define DD_SCAN(E_, VC_) \
  return p.i ? launch<E_, VC_, true, BWD>(p, ws, ws_bytes, st) : launch<E_, VC_, false, BWD>(p, ws, ws_bytes, st)
  if (type == DD_F32) { if (pair) DD_SCAN(float, 2); DD_SCAN(float, 1); }
  if (pair) DD_SCAN(__bf16, 2);
  DD_SCAN(__bf16, 1);
#undef DD_SCAN
}

}  // namespace

extern "C" int dd_gated_scan_fwd(const void* u, long ldu, const void* c, long ldc, const void* i, long ldi, int type,
                                 const float* first, long fstride, const float* h0, void* h, long ldh, float* hT,
                                 int B, int T, int D, float shift, int cand_tanh, float* ws, size_t ws_bytes, void* stream) {
  DD_REQUIRE(B >= 0 && T > 0 && D > 0 && T <= (1 << 30) && D <= (1 << 30), "dd_gated_scan_fwd: B >= 0, 0 < T, D <= 2^30 are needed");
  DD_REQUIRE(type == DD_F32 || type == DD_BF16, "dd_gated_scan_fwd: fp32 or bf16");
  if (B == 0) return 0;
  DD_REQUIRE(u && c && h, "dd_gated_scan_fwd: null u, c or h");
  DD_REQUIRE(ldu >= D && ldc >= D && ldh >= D && (!i || ldi >= D), "dd_gated_scan_fwd: a leading dimension below D");
  ScanArgs p{};
  p.u = u; p.ldu = ldu; p.c = c; p.ldc = ldc; p.i = i; p.ldi = ldi; p.first = first; p.fstride = fstride;
  p.x0 = h0; p.xT = hT; p.h = h; p.ldh = ldh; p.B = B; p.T = T; p.D = D; p.shift = shift; p.tanh_c = cand_tanh;
  return dispatch<false>(p, type, ws, ws_bytes, (hipStream_t)stream);
}

extern "C" int dd_gated_scan_bwd(const void* dh, long lddh, const void* u, long ldu, const void* c, long ldc, const void* i,
                                 long ldi, const void* h, long ldh, int type, const float* first, long fstride,
                                 const float* h0, const float* dhT, void* du, long lddu, void* dc, long lddc, void* di,
                                 long lddi, float* dh0, int B, int T, int D, float shift, int cand_tanh, float* ws,
                                 size_t ws_bytes, void* stream) {
  DD_REQUIRE(B >= 0 && T > 0 && D > 0 && T <= (1 << 30) && D <= (1 << 30), "dd_gated_scan_bwd: B >= 0, 0 < T, D <= 2^30 are needed");
  DD_REQUIRE(type == DD_F32 || type == DD_BF16, "dd_gated_scan_bwd: fp32 or bf16");
  if (B == 0) return 0;
  DD_REQUIRE(dh && u && c && h && du && dc, "dd_gated_scan_bwd: null pointer");
  DD_REQUIRE((i != nullptr) == (di != nullptr), "dd_gated_scan_bwd: di goes with i, and only with it");
  DD_REQUIRE(lddh >= D && ldu >= D && ldc >= D && ldh >= D && lddu >= D && lddc >= D && (!i || (ldi >= D && lddi >= D)),
             "dd_gated_scan_bwd: a leading dimension below D");
  ScanArgs p{};
  p.u = u; p.ldu = ldu; p.c = c; p.ldc = ldc; p.i = i; p.ldi = ldi; p.first = first; p.fstride = fstride;
  p.x0 = dhT; p.xT = dh0; p.h = const_cast<void*>(h); p.ldh = ldh; p.h0 = h0; p.dh = dh; p.lddh = lddh;
  p.du = du; p.lddu = lddu; p.dc = dc; p.lddc = lddc; p.di = di; p.lddi = lddi;
  p.B = B; p.T = T; p.D = D; p.shift = shift; p.tanh_c = cand_tanh;
  return dispatch<true>(p, type, ws, ws_bytes, (hipStream_t)stream);
}
