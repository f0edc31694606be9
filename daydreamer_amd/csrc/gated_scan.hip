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
// in registers.  Up to 64 steps are in flight at once, all loads issued before the first is used.  Few
// sequences with many steps: the time axis is split over workgroups as well, whose pairs a first launch
// puts into the workspace.
//
// Bound: HBM, with the vector unit close behind (two to three sigmoids and a tanh per element, a quarter
// of the rate each for exponential and reciprocal).  Hence: restarts are a property of a row, the same for
// all lanes, and are looked at once per run of steps - runs without one (nearly all) take plain
// multiply-adds; one exponential and one reciprocal give a sigmoid and its complement; and with bf16
// operands tanh near zero is two terms of its series, not six.
//
// A restart is A == 0 EXACTLY and cuts whatever came before, non-finite values too (0 * NaN would
// not); every other factor is kept at or above FLT_MIN, so that a product that underflows does not look
// like a restart and a NaN in the state is not lost.  The running state, pairs and all arithmetic are fp32; h is stored in
// the operands' type, half the bytes in bf16, and the backward pass reads the states before each step as stored: with bf16
// operands that leaves du off by 7e-4 in the 2-norm, by 1.6e-3 (h alone is its factor) with an input gate, beside 1.7e-3
// for its own rounding; fp32 operands have neither.
#include "block_core.h"
#include <float.h>

namespace {

constexpr int STEPS = 8;   // time steps of one wave between two exchanges
constexpr int WAVES = 8;   // waves of a workgroup at most

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
  int shared_lines;                 // rows are not aligned to cache lines
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

// A product of factors, FLT_MIN at least.  It may lose a NaN (max): by then that is in the pair's other half, where it stays.
__device__ __forceinline__ float at_least_min(float a) { return fmaxf(a, FLT_MIN); }
__device__ __forceinline__ float apply(float A, float B, float x) { return A == 0.f ? B : fma_(A, x, B); }
// (A2, B2) after (A1, B1), into (A1, B1)
__device__ __forceinline__ void compose(float& A1, float& B1, float A2, float B2) {
  B1 = apply(A2, B2, B1);
  A1 = (A1 == 0.f || A2 == 0.f) ? 0.f : at_least_min(A1 * A2);
}

// z = sigmoid(u + shift) and the decay q = 1 - z from E = e^-v, neither by a difference: a gate that is all but open
// keeps its decay, and du, to a few ulp of themselves.  E is held between 2^-125 and 2^125: E z is no infinity times
// zero, q is above FLT_MIN, and a NaN stays one (minimum and maximum keep it).  FUSED (bf16 operands): u + shift is not
// formed by itself, one instruction less; E is then off by |shift| 2^-24 for the rounding of shift's product.
template <bool FUSED>
__device__ __forceinline__ void gates(float u, float shift, float& z, float& q) {
  const float t = FUSED ? fma_(u, -1.44269504088896341f, shift * -1.44269504088896341f) : (u + shift) * -1.44269504088896341f;
  const float E = __builtin_amdgcn_exp2f(__builtin_elementwise_maximum(__builtin_elementwise_minimum(t, 125.f), -125.f));
  z = fast_rcp(1.0f + E);
  q = E * z;
}
// phi(c).  BRIEF (bf16 operands): two terms of tanh's series up to 1/16, where the next is 2^-19 of it, and the
// exponential beyond, good to 2^-18 there (4 x 4096 x 1024 forward: 40.4 us; 39.1 with the exponential alone, which
// is off by 5 % at 1e-6).
template <bool BRIEF>
__device__ __forceinline__ float phi_of(float c, int tanh_c) {
  if (!tanh_c) return c;
  if constexpr (BRIEF) {
    const float small = c * fma_(c * c, -1.f / 3, 1.f);
    const float large = fma_(-2.0f, fast_rcp(1.0f + __builtin_amdgcn_exp2f(c * 2.88539008177792681f)), 1.0f);
    return fabsf(c) < 0.0625f ? small : large;
  } else {
    return tanh_f(c);
  }
}
// ... and its slope 1 - phi^2 = 4 e r^2, e = e^-2|c|, r = 1 / (1 + e), not by a difference either.
template <bool BRIEF>
__device__ __forceinline__ void phi_slope(float c, int tanh_c, float& phi, float& slope) {
  phi = c;
  slope = 1.f;
  if (!tanh_c) return;
  const float e = fast_exp(-2.0f * fabsf(c)), r = fast_rcp(1.0f + e), er = e * r;
  slope = 4.0f * r * er;
  if constexpr (BRIEF) phi = fabsf(c) < 0.0625f ? c * fma_(c * c, -1.f / 3, 1.f) : copysignf(fma_(-2.0f, er, 1.0f), c);
  else phi = tanh_f(c);
}
__device__ __forceinline__ float sigmoid1(float x) { return fast_rcp(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504088896341f)); }

// Bit s: step o0 + s (in scan order, of `n`) of sequence b starts anew.  One load for the wave's run.
template <bool BWD>
__device__ __forceinline__ unsigned restarts(const ScanArgs& p, long b, int o0, int n, int lane) {
  if (!p.first) return 0;
  bool r = false;
  if (lane < n) r = p.first[(b * p.T + (BWD ? p.T - 1 - o0 - lane : o0 + lane)) * p.fstride] != 0.f;
  return (unsigned)__ballot(r);
}

// A run of up to STEPS steps in scan order (the last one repeated past n), restarts aside: z, q as in gates and
// b = gate phi(c) (forward) or dh (backward).
template <typename E, int VC, bool GATE, bool BWD>
__device__ __forceinline__ void run_pairs(const ScanArgs& p, long b, int o0, int n, int d, float z[STEPS][VC],
                                          float q[STEPS][VC], float bb[STEPS][VC]) {
  constexpr bool BRIEF = sizeof(E) == 2;
  float u[STEPS][VC], c[STEPS][VC], i[STEPS][VC];
#pragma unroll
  for (int s = 0; s < STEPS; ++s) {
    const int o = o0 + min(s, n - 1);
    const long row = b * p.T + (BWD ? p.T - 1 - o : o);
    ld<E, VC>(p.u, row * p.ldu + d, u[s]);
    if constexpr (BWD) {
      ld<E, VC>(p.dh, row * p.lddh + d, bb[s]);
    } else {
      ld<E, VC>(p.c, row * p.ldc + d, c[s]);
      if constexpr (GATE) ld<E, VC>(p.i, row * p.ldi + d, i[s]);
    }
  }
#pragma unroll
  for (int s = 0; s < STEPS; ++s)
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      gates<BRIEF>(u[s][j], p.shift, z[s][j], q[s][j]);
      if constexpr (!BWD) bb[s][j] = (GATE ? sigmoid1(i[s][j]) : z[s][j]) * phi_of<BRIEF>(c[s][j], p.tanh_c);
    }
}

// The run's composed pair.
template <int VC, bool BWD>
__device__ __forceinline__ void run_total(int n, unsigned cut, const float q[STEPS][VC], const float bb[STEPS][VC], float A[VC],
                                          float B[VC]) {
#pragma unroll
  for (int j = 0; j < VC; ++j) { A[j] = 1.f; B[j] = 0.f; }
  if (cut == 0 && n == STEPS) {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        const float a = q[s][j];
        B[j] = BWD ? a * (B[j] + bb[s][j]) : fma_(a, B[j], bb[s][j]);
        A[j] = at_least_min(A[j] * a);
      }
  } else {
#pragma unroll
    for (int s = 0; s < STEPS; ++s)
      if (s < n)
#pragma unroll
        for (int j = 0; j < VC; ++j) {
          const float a = cut >> s & 1 ? 0.f : q[s][j];
          compose(A[j], B[j], a, BWD ? (a == 0.f ? 0.f : a * bb[s][j]) : bb[s][j]);
        }
  }
}

// This workgroup's sequence, channels and split.  Rows that are not aligned to cache lines: neighbouring channels
// of the same steps share lines, so they are given to one XCD (consecutive workgroups go to the eight in turn)
// one after the other and meet in its L2; else the splits of the same channels come first (1 x 24368 x 2367 fp32
// 774 us backward the second way, 598 the first; 2 x 16385 x 512 144 and 151).
struct Work { int g, k; long b; };
__device__ __forceinline__ Work work_of(const ScanArgs& p, int splits) {
  unsigned id = blockIdx.x;
  if (!p.shared_lines) return {(int)(id / splits % p.groups), (int)(id % splits), (long)(id / splits / p.groups)};
  const unsigned q = gridDim.x / 8, r = gridDim.x % 8, xcd = id % 8;
  id = xcd * q + min(xcd, r) + id / 8;
  return {(int)(id % p.groups), (int)(id / p.groups % splits), (long)(id / p.groups / splits)};
}

// First launch of a split time axis: the pairs of all splits but the last (in scan order), and in
// slot 0 the initial state as a restart, so that a state updated in place is read before it is written.
template <typename E, int VC, bool GATE, bool BWD>
__global__ void __launch_bounds__(64 * WAVES) k_scan_pairs(ScanArgs p) {
  __shared__ float2 sh[WAVES][64 * VC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const Work w = work_of(p, p.splits - 1);
  const int k = w.k, g = w.g;
  const long b = w.b;
  const int d = min((g * 64 + lane) * VC, p.D - VC);
  const bool live = (g * 64 + lane) * VC < p.D;
  const int len = p.span / WAVES;   // this wave's steps, in scan order: a multiple of STEPS; the last split is not here
  float A[VC], Bv[VC];
#pragma unroll
  for (int j = 0; j < VC; ++j) { A[j] = 1.f; Bv[j] = 0.f; }
  for (int s = 0; s < len; s += STEPS) {
    const int o0 = k * p.span + wave * len + s;
    float z[STEPS][VC], q[STEPS][VC], bb[STEPS][VC], a2[VC], b2[VC];
    const unsigned cut = restarts<BWD>(p, b, o0, STEPS, lane);
    run_pairs<E, VC, GATE, BWD>(p, b, o0, STEPS, d, z, q, bb);
    run_total<VC, BWD>(STEPS, cut, q, bb, a2, b2);
#pragma unroll
    for (int j = 0; j < VC; ++j) compose(A[j], Bv[j], a2[j], b2[j]);
  }
#pragma unroll
  for (int j = 0; j < VC; ++j) sh[wave][lane * VC + j] = make_float2(A[j], Bv[j]);
  __syncthreads();
  if (wave == 0 && live)
#pragma unroll
    for (int j = 0; j < VC; ++j) {
      for (int o = 1; o < WAVES; ++o) compose(A[j], Bv[j], sh[o][lane * VC + j].x, sh[o][lane * VC + j].y);
      float2* out = p.pairs + b * p.splits * p.D + d + j;
      out[(long)(k + 1) * p.D] = make_float2(A[j], Bv[j]);
      if (k == 0) out[0] = make_float2(0.f, p.x0 ? p.x0[b * p.D + d + j] : 0.f);
    }
}

// State at the start of split k of (b, d): the initial one, or the composed pairs of what precedes it, an equal
// run of them per wave (64 of them one after the other took a wave 6 us).
template <int VC>
__device__ __forceinline__ void start_state(const ScanArgs& p, long b, int k, int d, float2 (*sh)[64 * VC], int wave, int waves,
                                            int lane, float x[VC]) {
#pragma unroll
  for (int j = 0; j < VC; ++j) x[j] = 0.f;
  if (p.splits == 1) {
    if (p.x0) load_f32<VC>(p.x0 + b * p.D + d, x);
    return;
  }
  float A[VC], B[VC];
#pragma unroll
  for (int j = 0; j < VC; ++j) { A[j] = 1.f; B[j] = 0.f; }
  const int per = (k + waves) / waves, from = wave * per, to = min(k + 1, from + per);
#pragma unroll 8
  for (int s = from; s < to; ++s) {
    const float2* q = p.pairs + (b * p.splits + s) * p.D + d;
#pragma unroll
    for (int j = 0; j < VC; ++j) compose(A[j], B[j], q[j].x, q[j].y);
  }
#pragma unroll
  for (int j = 0; j < VC; ++j) sh[wave][lane * VC + j] = make_float2(A[j], B[j]);
  __syncthreads();
  for (int w = 0; w < waves; ++w)
#pragma unroll
    for (int j = 0; j < VC; ++j) x[j] = apply(sh[w][lane * VC + j].x, sh[w][lane * VC + j].y, x[j]);
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
__global__ void __launch_bounds__(64 * WAVES) k_scan_fwd(ScanArgs p) {
  __shared__ float2 sh[2][WAVES][64 * VC];   // two buffers: one barrier per exchange
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const Work w = work_of(p, p.splits);
  const int k = w.k, g = w.g;
  const long b = w.b;
  const int d = min((g * 64 + lane) * VC, p.D - VC);   // lanes past the last channel repeat it, and store nothing
  const bool live = (g * 64 + lane) * VC < p.D;
  const int end = min(p.T, (k + 1) * p.span);
  float x[VC];
  start_state<VC>(p, b, k, d, sh[1], wave, waves, lane, x);   // (the first exchange takes sh[0])
  int buf = 0;
  for (int base = k * p.span; base < end; base += waves * STEPS, buf ^= 1) {
    const int o0 = base + wave * STEPS, n = min(STEPS, end - o0);   // n <= 0: a wave behind the end
    float z[STEPS][VC], q[STEPS][VC], bb[STEPS][VC], A[VC], Bv[VC], in[VC];
    const unsigned cut = restarts<false>(p, b, o0, n, lane);
#pragma unroll
    for (int j = 0; j < VC; ++j) { A[j] = 1.f; Bv[j] = 0.f; }
    if (n > 0) {
      run_pairs<E, VC, GATE, false>(p, b, o0, n, d, z, q, bb);
      run_total<VC, false>(n, cut, q, bb, A, Bv);
    }
    exchange<VC>(sh[buf], wave, waves, lane, A, Bv, x, in);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s >= n) break;
#pragma unroll
      for (int j = 0; j < VC; ++j) in[j] = cut >> s & 1 ? bb[s][j] : fma_(q[s][j], in[j], bb[s][j]);
      if (live) st<E, VC>(p.h, (b * p.T + o0 + s) * p.ldh + d, in);
    }
  }
  if (p.xT && live && k == p.splits - 1 && wave == 0) store_f32<VC>(p.xT + b * p.D + d, x);
}

template <typename E, int VC, bool GATE>
__global__ void __launch_bounds__(64 * WAVES) k_scan_bwd(ScanArgs p) {
  constexpr bool BRIEF = sizeof(E) == 2;
  __shared__ float2 sh[2][WAVES][64 * VC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
  const Work w = work_of(p, p.splits);
  const int k = w.k, g = w.g;
  const long b = w.b;
  const int d = min((g * 64 + lane) * VC, p.D - VC);
  const bool live = (g * 64 + lane) * VC < p.D;
  const int end = min(p.T, (k + 1) * p.span);   // in scan order: o = T - 1 - t
  float x[VC];
  start_state<VC>(p, b, k, d, sh[1], wave, waves, lane, x);   // (the first exchange takes sh[0])
  int buf = 0;
  for (int base = k * p.span; base < end; base += waves * STEPS, buf ^= 1) {
    const int o0 = base + wave * STEPS, n = min(STEPS, end - o0);
    float z[STEPS][VC], q[STEPS][VC], dh[STEPS][VC], c[STEPS][VC], gi[STEPS][VC], hp[STEPS][VC], A[VC], Bv[VC], in[VC];
    const unsigned cut = restarts<true>(p, b, o0, n, lane);
#pragma unroll
    for (int j = 0; j < VC; ++j) { A[j] = 1.f; Bv[j] = 0.f; }
    if (n > 0) {
#pragma unroll
      for (int s = 0; s < STEPS; ++s) {
        const long row = b * p.T + p.T - 1 - (o0 + min(s, n - 1));
        ld<E, VC>(p.c, row * p.ldc + d, c[s]);
        if constexpr (GATE) ld<E, VC>(p.i, row * p.ldi + d, gi[s]);
        ld<E, VC>(p.h, max(row - 1, 0l) * p.ldh + d, hp[s]);
      }
      if (o0 + n == p.T) {   // the run's last step is the sequence's first: its state before is h0
        float first[VC] = {};
        if (p.h0) load_f32<VC>(p.h0 + b * p.D + d, first);
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
          for (int j = 0; j < VC; ++j) hp[s][j] = s == n - 1 ? first[j] : hp[s][j];
      }
      run_pairs<E, VC, GATE, true>(p, b, o0, n, d, z, q, dh);
      run_total<VC, true>(n, cut, q, dh, A, Bv);
    }
    exchange<VC>(sh[buf], wave, waves, lane, A, Bv, x, in);
#pragma unroll
    for (int s = 0; s < STEPS; ++s) {
      if (s >= n) break;
      const bool restart = cut >> s & 1;
      float du[VC], dc[VC], di[VC];
#pragma unroll
      for (int j = 0; j < VC; ++j) {
        const float gr = dh[s][j] + in[j];             // d loss / d h[t]
        in[j] = restart ? 0.f : q[s][j] * gr;
        float phi, slope;
        phi_slope<BRIEF>(c[s][j], p.tanh_c, phi, slope);
        const float before = restart ? 0.f : hp[s][j];
        const float gz = gr * z[s][j];
        if constexpr (GATE) {
          float w, w1;
          gates<true>(gi[s][j], 0.f, w, w1);
          const float gw = gr * w;
          du[j] = -gz * q[s][j] * before;
          di[j] = gw * phi * w1;
          dc[j] = gw * slope;
        } else {
          du[j] = gz * q[s][j] * (phi - before);
          dc[j] = gz * slope;
        }
      }
      if (live) {
        const long row = b * p.T + p.T - 1 - o0 - s;
        st<E, VC>(p.du, row * p.lddu + d, du);
        st<E, VC>(p.dc, row * p.lddc + d, dc);
        if constexpr (GATE) st<E, VC>(p.di, row * p.lddi + d, di);
      }
    }
  }
  if (p.xT && live && k == p.splits - 1 && wave == 0) store_f32<VC>(p.xT + b * p.D + d, x);
}

// Splits of the time axis: none where the channels alone give every CU a workgroup; else enough for
// four workgroups per CU, each at least one exchange of all waves long (two: 3 x 966 x 2240 forward 37 us against
// 28; from 256 steps on: 162 take 9 us in one launch and 12 in two).
inline void plan(ScanArgs& p) {
  constexpr int PASS = WAVES * STEPS;
  const long wgs = (long)p.B * p.groups;
  p.splits = 1;
  p.span = p.T;
  if (wgs < 256 && p.T >= 4 * PASS) {
    const long want = min((1024 + wgs - 1) / wgs, (long)p.T / PASS);
    p.span = dd_ceil_div(dd_ceil_div(p.T, want), PASS) * PASS;
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
    k_scan_pairs<E, VC, GATE, BWD><<<(unsigned)((long)p.B * p.groups * (p.splits - 1)), 64 * WAVES, 0, stream>>>(p);
    DD_CHECK_LAUNCH("dd_gated_scan(pairs)");
  }
  const int threads = 64 * min(WAVES, dd_ceil_div(p.T, STEPS));
  if constexpr (BWD) k_scan_bwd<E, VC, GATE><<<(unsigned)wgs, threads, 0, stream>>>(p);
  else k_scan_fwd<E, VC, GATE><<<(unsigned)wgs, threads, 0, stream>>>(p);
  DD_CHECK_LAUNCH(BWD ? "dd_gated_scan_bwd" : "dd_gated_scan_fwd");
  return 0;
}

// Two channels per lane.  bf16 (256 bytes of a row per wave): where that leaves every CU a workgroup, or the time axis
// is split anyway (50 x 50 x 1024 backward: 11 us against 16 with one; 4 x 4096 x 1024 forward 48 against 53).
// fp32: long scans of rows that are not aligned to cache lines, a smaller part of which is then shared (1 x 24368
// x 2367 backward 510 us against 598; aligned rows 2 x 16385 x 512 lose 2%, 29 x 78 x 3392 a fifth).
template <bool BWD>
int dispatch(ScanArgs& p, int type, float* ws, size_t ws_bytes, hipStream_t st) {
#define DD_SCAN(E_, VC_) \
  return p.i ? launch<E_, VC_, true, BWD>(p, ws, ws_bytes, st) : launch<E_, VC_, false, BWD>(p, ws, ws_bytes, st)
  const long es = type == DD_F32 ? 4 : 2;
  auto aligned = [&](const void* q, long ld) { return !q || ((uintptr_t)q % 128 == 0 && (ld * es) % 128 == 0); };
  p.shared_lines = !(aligned(p.u, p.ldu) && aligned(p.c, p.ldc) && aligned(p.i, p.ldi) && aligned(p.h, p.ldh) &&
                     aligned(p.dh, p.lddh) && aligned(p.du, p.lddu) && aligned(p.dc, p.lddc) && aligned(p.di, p.lddi));
  // (an odd row's last lane takes its neighbour's second channel as well; a group of that lane alone would write
  // another workgroup's channel, which a state updated in place must not see)
  const bool pairs = p.D > 1 && p.D % 128 != 1;
  const long wgs = (long)p.B * dd_ceil_div(p.D, 128);
  if (type == DD_F32) {
    if (pairs && p.shared_lines && wgs * dd_ceil_div(p.T, WAVES * STEPS) >= 2048) DD_SCAN(float, 2);
    DD_SCAN(float, 1);
  }
  if (p.D % 2 == 0 && (wgs >= 256 || p.T >= 4 * WAVES * STEPS)) DD_SCAN(__bf16, 2);
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
