// norm.cu -- the norms around a block: residual add with a scale for the branch
// before a LayerNorm / RMS norm, and a norm per group of channels with a gate
// after a mixer, one kernel forward and two backward.
//
// Per row, with groups of n = D / G channels (fp32 throughout, tensors rounded
// once on the way out):
//   h = residual + scale * x            (h = x without a residual)
//   z = (h - mean) * r,  r = 1 / sqrt(mean((h - mean)^2) + eps)   (mean 0 for RMS)
//   y = (z * weight + bias) * silu(gate)
// Backward, da = dy * silu(gate), dz = da * weight, gh the gradient of h itself:
//   dh = r (dz - mean(dz) - z mean(dz z)) + gh    (without mean(dz) for RMS)
//   dx = scale * dh, dresidual = dh, dgate = dy * (z * weight + bias) * silu'(gate)
//   dweight = sum da z, dbias = sum da, dscale = sum dh x     (over rows)
//
// Memory bound on paper: the forward reads each input once and writes each output
// once, a group's values staying in its threads' registers between the two
// reductions; the backward reads the inputs again instead of z (and h is taken
// in fp32 from x and residual, not from its rounded copy), with mean and r from
// the forward. Sums over rows stay in the threads' registers while a CTA walks
// its rows, then go through shared memory to one partial row per CTA and, in
// order, to the result: the same bits on every run.
#include <utility>

#include "common.cuh"
#include "odd_rows.h"

namespace mgs {
namespace norm {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxGroup = 16384;  // 1024 threads of 16 values

struct Args {
  const void *x, *res, *gate, *w, *b, *s, *dy, *dh;
  void *y, *h, *dx, *dres, *dgate;
  float* stats;  // (rows * G, 3): mean, what it leaves, r
  float* part;   // (3, grid, D): sums over a CTA's rows of dweight, dbias, dscale
  long long ldx, ldres, ldgate, lddy, lddh;  // row strides of the inputs; outputs are dense
  long long rows;
  int D, G, n, tpg, gpc, rpc;  // threads to a group, groups and rows to a CTA
  int rms, w32;  // weights in fp32
  int staged;    // backward: the inputs that come through shared memory, a row ahead; 0: straight
  float eps;
};

// A thread's K vectors of VEC elements, tpg vectors apart, zeros from column n on:
// loaded in one go, a row ahead of their use, and widened then.
template <typename T, int VEC, int K>
struct Raw {
  static constexpr int kN = VEC == 1 ? 1 : VEC * (int)sizeof(T) / 16;
  std::conditional_t<VEC == 1, T, uint4> r[K][kN];
  __device__ __forceinline__ void load(const void* p, long long i, int t, int tpg, int n) {
    const T* q = static_cast<const T*>(p) + i + t * VEC;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const bool in = (k * tpg + t) * VEC < n;
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        if constexpr (VEC == 1)
          r[k][j] = in ? q[k * tpg] : from_f32<T>(0.f);
        else
          r[k][j] = in ? __ldg(reinterpret_cast<const uint4*>(q + k * tpg * VEC) + j) : make_uint4(0, 0, 0, 0);
      }
    }
  }
  __device__ __forceinline__ void get(float (&v)[K * VEC]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const T* e = reinterpret_cast<const T*>(r[k]);
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[k * VEC + j] = to_f32<T>(e[j]);
    }
  }
};
template <typename T, int VEC, int K>
__device__ __forceinline__ void ldrow(const void* p, long long i, int t, int tpg, int n, float (&v)[K * VEC]) {
  Raw<T, VEC, K> r;
  r.load(p, i, t, tpg, n);
  r.get(v);
}
template <typename T, int VEC, int K>
__device__ __forceinline__ void strow(void* p, long long i, int t, int tpg, int n, const float (&v)[K * VEC]) {
  T* q = static_cast<T*>(p) + i + t * VEC;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if ((k * tpg + t) * VEC >= n) break;
    if constexpr (VEC == 1) {
      q[k * tpg] = from_f32<T>(v[k]);
    } else {
      uint4 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int j = 0; j < VEC; ++j) e[j] = from_f32<T>(v[k * VEC + j]);
      *reinterpret_cast<uint4*>(q + k * tpg * VEC) = u;
    }
  }
}

// The same K vectors into 16-byte places of the thread's own in shared memory, `stride`
// apart: on their way without registers. Out of the row they become zeros.
template <typename T, int VEC, int K>
__device__ __forceinline__ void stage_row(uint4* to, int stride, const void* p, long long i, int t, int tpg, int n) {
  constexpr int kN = VEC * (int)sizeof(T) / 16;
  const T* q = static_cast<const T*>(p);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (k * tpg + t) * VEC;
    const T* from = c < n ? q + i + c : q;
#pragma unroll
    for (int j = 0; j < kN; ++j)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to + (k * kN + j) * stride)),
                   "l"(reinterpret_cast<const uint4*>(from) + (c < n ? j : 0)), "r"(c < n ? 16 : 0)
                   : "memory");
  }
}
template <typename T, int VEC, int K>
__device__ __forceinline__ void staged_row(const uint4* from, int stride, float (&v)[K * VEC]) {
  Raw<T, VEC, K> r;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < r.kN; ++j) r.r[k][j] = from[(k * r.kN + j) * stride];
  r.get(v);
}

// Sums over the tpg threads of a group: a segment of a warp, or whole warps
// that meet at a named barrier of the group's own. `buf` alternates, so that
// one barrier is enough for each sum. What the threads wrote to shared memory
// before is visible to the group after.
struct Reduce {
  float2 (*red)[32];
  int tpg, slot, buf;
  template <int W, bool TWO>
  __device__ __forceinline__ static void lanes(unsigned mask, float& a, float& b) {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) {
      a += __shfl_xor_sync(mask, a, o);
      if constexpr (TWO) b += __shfl_xor_sync(mask, b, o);
    }
  }
  template <bool TWO>
  __device__ __forceinline__ float2 go(float a, float b) {
    const int lane = threadIdx.x & 31;
    if (tpg == 8) {
      __syncwarp(0xffu << (lane & 24));
      lanes<8, TWO>(0xffu << (lane & 24), a, b);
    } else if (tpg == 16) {
      __syncwarp(0xffffu << (lane & 16));
      lanes<16, TWO>(0xffffu << (lane & 16), a, b);
    } else {
      __syncwarp();
      lanes<32, TWO>(0xffffffffu, a, b);
      if (tpg > 32) {
        const int nw = tpg / 32, w0 = slot * nw;
        if (lane == 0) red[buf][threadIdx.x >> 5] = make_float2(a, b);
        named_bar(1 + slot, tpg);
        const float2 f = lane < nw ? red[buf][w0 + lane] : make_float2(0.f, 0.f);
        a = f.x, b = f.y;
        if (nw <= 4)
          lanes<4, TWO>(0xffffffffu, a, b);
        else
          lanes<32, TWO>(0xffffffffu, a, b);
        a = __shfl_sync(0xffffffffu, a, 0);
        if constexpr (TWO) b = __shfl_sync(0xffffffffu, b, 0);
        buf ^= 1;
      }
    }
    return make_float2(a, b);
  }
  __device__ __forceinline__ float2 operator()(float a, float b) { return go<true>(a, b); }
  __device__ __forceinline__ float operator()(float a) { return go<false>(a, 0.f).x; }
};

// 1 / (1 + e^-x) in four instructions: denormals of the hardware's 2^x and 1 / x are
// flushed, which nothing sees next to the 1, or below 2^-126.
__device__ __forceinline__ float sigm(float x) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.44269504f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  return r;
}

// 1 / sqrt(v) to the last place, by a step of Newton's on the hardware's: the
// gradient takes differences of z * z and 1. The step of an infinite sum of squares
// (finite values past 2^64) would be inf * 0; fminf makes it 1, and the result 0.
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  return fmaf(0.5f * r, fminf(fmaf(-v * r, r, 1.f), 1.f), r);
}

// A mean of squares that cancellation took below zero; NaN stays (fmaxf drops it, and
// a row with a NaN came out finite but for that element).
__device__ __forceinline__ float at_least_zero(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, 0f00000000;" : "=f"(r) : "f"(v));
  return r;
}

// Where a thread stands: its group (of the row), row slot and first column.
struct Place {
  int slot, rs, g, t;
  bool on;
  __device__ explicit Place(const Args& p) {
    slot = (int)threadIdx.x / p.tpg;
    t = (int)threadIdx.x % p.tpg;
    rs = slot / p.gpc;
    g = blockIdx.y * p.gpc + slot % p.gpc;
    on = rs < p.rpc && g < p.G;
  }
};

// CTAs to an SM that the registers are held to: latency is hidden by rows under
// way, 1024 threads' worth forward and 768 backward.
constexpr int fwd_ctas(int threads) { return 1024 / threads; }
constexpr int bwd_ctas(int threads) { return threads == 256 ? 3 : 1; }
// Odd rows, a row ahead in registers as well: 80 registers, up to 128 backward.
constexpr int odd_fwd_ctas(int threads) { return threads == 256 ? 3 : threads == 384 ? 2 : 1; }
constexpr int odd_bwd_ctas(int threads) { return threads == 256 ? 2 : 1; }

// Values of the next row are on their way where 8 to a thread leave registers for them
// (16: 64 registers are full without; 8192 x 512 fp32 takes 23 us with, 15 without).
// 16384 x 2048 bf16 with a residual: 55 us, 4.9 TB/s; 65536 x 512 bf16 in 8 gated
// groups: 40 us, 5.0 TB/s, bound by the instructions of the gate (75% of the issue
// slots before the sums that only a mean needs were left out of RMS rows: 47 us).
template <typename E, typename W, int VEC, int K, int MAXT>
__global__ void __launch_bounds__(MAXT, fwd_ctas(MAXT)) fwd_kernel(const Args p) {
  constexpr int N = K * VEC;
  __shared__ float2 red[2][32];
  const Place at(p);
  if (!at.on) return;
  Reduce sum{red, p.tpg, at.slot, 0};
  const float inv_n = 1.f / (float)p.n;
  const int col = at.g * p.n;
  auto in = [&](int i) { return ((i / VEC) * p.tpg + at.t) * VEC < p.n; };
  const long long step = (long long)gridDim.x * p.rpc;
  Raw<E, VEC, K> rx, ra;  // x, and the residual or else the gate, of the next row where there is room
  constexpr bool kAhead = K == 1;  // 16 values to a thread leave no registers for it
  auto fetch = [&](long long row) {
    if (row >= p.rows) return;
    rx.load(p.x, row * p.ldx + col, at.t, p.tpg, p.n);
    if (p.res)
      ra.load(p.res, row * p.ldres + col, at.t, p.tpg, p.n);
    else if (p.gate)
      ra.load(p.gate, row * p.ldgate + col, at.t, p.tpg, p.n);
  };
  if (kAhead) fetch((long long)blockIdx.x * p.rpc + at.rs);
  float wk[kAhead ? N : 1];  // the weight, for all rows
  if constexpr (kAhead) ldrow<W, VEC, K>(p.w, col, at.t, p.tpg, p.n, wk);
  for (long long row = (long long)blockIdx.x * p.rpc + at.rs; row < p.rows; row += step) {
    float h[N], a[N], w[N];
    if constexpr (kAhead) {
      rx.get(h);
      ra.get(a);
      fetch(row + step);
    } else {
      ldrow<E, VEC, K>(p.x, row * p.ldx + col, at.t, p.tpg, p.n, h);
      if (p.res)
        ldrow<E, VEC, K>(p.res, row * p.ldres + col, at.t, p.tpg, p.n, a);
      else if (p.gate)
        ldrow<E, VEC, K>(p.gate, row * p.ldgate + col, at.t, p.tpg, p.n, a);
    }
    if (p.res) {
      if (p.s) {
        ldrow<W, VEC, K>(p.s, col, at.t, p.tpg, p.n, w);
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] = fmaf(w[i], h[i], a[i]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) h[i] += a[i];
      }
    }
    if (p.res && p.gate) ldrow<E, VEC, K>(p.gate, row * p.ldgate + col, at.t, p.tpg, p.n, a);
    const long long o = row * p.D + col;
    if (p.h) strow<E, VEC, K>(p.h, o, at.t, p.tpg, p.n, h);
    float mean = 0.f, rest = 0.f, sq = 0.f;
    if (p.rms) {
#pragma unroll
      for (int i = 0; i < N; ++i) sq = fmaf(h[i], h[i], sq);  // zeros from column n on
      sq = sum(sq) * inv_n;
    } else {
      // The fp32 mean is off by up to half a unit of its last place: what it leaves in the
      // differences, `rest`, is their own mean, and comes with the sum of their squares.
#pragma unroll
      for (int i = 0; i < N; ++i) mean += h[i];
      mean = sum(mean) * inv_n;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        h[i] = in(i) ? h[i] - mean : 0.f;
        sq = fmaf(h[i], h[i], sq);
        rest += h[i];
      }
      const float2 m = sum(sq, rest);
      rest = m.y * inv_n;
      sq = at_least_zero(fmaf(-rest, rest, m.x * inv_n));
    }
    const float r = inv_sqrt(sq + p.eps);
    if (p.stats && at.t == 0) {
      float* st = p.stats + (row * p.G + at.g) * 3;
      st[0] = mean, st[1] = rest, st[2] = r;
    }
    const float shift = -rest * r;
    if constexpr (!kAhead) ldrow<W, VEC, K>(p.w, col, at.t, p.tpg, p.n, w);
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = fmaf(h[i], r, shift) * (kAhead ? wk[i % (kAhead ? N : 1)] : w[i]);
    if (p.b) {
      ldrow<W, VEC, K>(p.b, col, at.t, p.tpg, p.n, w);
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] += w[i];
    }
    if (p.gate) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] *= a[i] * sigm(a[i]);
    }
    strow<E, VEC, K>(p.y, o, at.t, p.tpg, p.n, h);
  }
}

// GATE and SCALE: whether they are there, so that a call without them keeps no
// registers for them. The seven arrays leave no registers for a row ahead, so rows
// come through shared memory, the next on its way during this one, where the SM has
// room for two rows' inputs of all its CTAs: 16384 x 2048 bf16 with a residual takes
// 77 us so and 112 straight, 65536 x 512 in 8 gated groups 78 and 116 (0.34 GB, 4.3
// TB/s: 440 instructions to 8 elements of a warp's lanes, 69% of the issue slots),
// 8192 x 512 fp32 14.1 and 14.5.
template <typename E, typename W, int VEC, int K, int MAXT, bool GATE, bool SCALE>
__global__ void __launch_bounds__(MAXT, bwd_ctas(MAXT)) bwd_kernel(const Args p) {
  constexpr int N = K * VEC;
  __shared__ float2 red[2][32];
  extern __shared__ float cols[];
  const Place at(p);
  Reduce sum{red, p.tpg, at.slot, 0};
  const float inv_n = 1.f / (float)p.n;
  const int col = at.g * p.n;
  float gw[N], gb[N], gs[SCALE ? N : 1];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    gw[i] = gb[i] = 0.f;
    if constexpr (SCALE) gs[i] = 0.f;
  }
  const long long step = (long long)gridDim.x * p.rpc;
  const bool staged = VEC > 1 && p.staged;
  constexpr int kPieces = VEC > 1 ? K * VEC * (int)sizeof(E) / 16 : 1;  // of 16 bytes to an input
  const int NT = blockDim.x, i_gate = 2 + (p.res != nullptr), i_dh = i_gate + GATE;
  auto place = [&](int buf, int i) {
    return reinterpret_cast<uint4*>(cols) + ((buf * p.staged + i) * kPieces * NT + (int)threadIdx.x);
  };
  auto fetch = [&](long long row, int buf) {
    if constexpr (VEC > 1) {
      if (row < p.rows) {
        auto go = [&](int i, const void* t, long long ld) {
          stage_row<E, VEC, K>(place(buf, i), NT, t, row * ld + col, at.t, p.tpg, p.n);
        };
        go(0, p.x, p.ldx);
        go(1, p.dy, p.lddy);
        if (p.res) go(2, p.res, p.ldres);
        if constexpr (GATE) go(i_gate, p.gate, p.ldgate);
        if (p.dh) go(i_dh, p.dh, p.lddh);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  int buf = 0;
  auto take = [&](int i, const void* t, long long at_row, float (&v)[N]) {
    if constexpr (VEC > 1) {
      if (staged) return staged_row<E, VEC, K>(place(buf, i), NT, v);
    }
    ldrow<E, VEC, K>(t, at_row, at.t, p.tpg, p.n, v);
  };
  if (at.on) {
    if (staged) fetch((long long)blockIdx.x * p.rpc + at.rs, 0);
    for (long long row = (long long)blockIdx.x * p.rpc + at.rs; row < p.rows; row += step, buf ^= staged) {
      if (staged) {  // a thread reads what it copied itself
        fetch(row + step, buf ^ 1);
        asm volatile("cp.async.wait_group 1;" ::: "memory");
      }
      const float* st = p.stats + (row * p.G + at.g) * 3;
      const long long o = row * p.D + col;
      float x[N], d[N], z[N], w[N];
      take(0, p.x, row * p.ldx + col, x);
      take(1, p.dy, row * p.lddy + col, d);
      const float mean = st[0], r = st[2], shift = -st[1] * r;
      if (SCALE || p.res) {
        take(2, p.res, row * p.ldres + col, z);
        if constexpr (SCALE) {
          ldrow<W, VEC, K>(p.s, col, at.t, p.tpg, p.n, w);
#pragma unroll
          for (int i = 0; i < N; ++i) z[i] = fmaf(w[i], x[i], z[i]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) z[i] += x[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = x[i];
      }
      ldrow<W, VEC, K>(p.w, col, at.t, p.tpg, p.n, w);
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = fmaf(z[i] - mean, r, shift);
      if constexpr (GATE) {
        float g[N], b[N];
        take(i_gate, p.gate, row * p.ldgate + col, g);
        if (p.b) {
          ldrow<W, VEC, K>(p.b, col, at.t, p.tpg, p.n, b);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) b[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float sg = sigm(g[i]), u = g[i] * sg;
          b[i] = d[i] * fmaf(z[i], w[i], b[i]) * fmaf(-u, sg, sg + u);  // silu' = sg + u - u sg
          d[i] *= u;
        }
        strow<E, VEC, K>(p.dgate, o, at.t, p.tpg, p.n, b);
      }
      float s1 = 0.f, s2 = 0.f;  // columns past n have d = w = 0
      if (p.b) {
#pragma unroll
        for (int i = 0; i < N; ++i) gb[i] += d[i];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        gw[i] = fmaf(d[i], z[i], gw[i]);
        d[i] *= w[i];
        s2 = fmaf(d[i], z[i], s2);
      }
      if (p.rms) {
        s2 = sum(s2);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s1 += d[i];
        const float2 m = sum(s1, s2);
        s1 = m.x, s2 = m.y;
      }
      s1 *= inv_n, s2 *= -inv_n;  // differences first: they cancel in small groups
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = r * fmaf(z[i], s2, d[i] - s1);
      if (p.dh) {
        take(i_dh, p.dh, row * p.lddh + col, w);
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] += w[i];
      }
      if constexpr (SCALE) {
        strow<E, VEC, K>(p.dres, o, at.t, p.tpg, p.n, d);
        ldrow<W, VEC, K>(p.s, col, at.t, p.tpg, p.n, w);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          gs[i] = fmaf(d[i], x[i], gs[i]);
          d[i] *= w[i];
        }
      }
      strow<E, VEC, K>(p.dx, o, at.t, p.tpg, p.n, d);
    }
  }
  if (staged) asm volatile("cp.async.wait_group 0;" ::: "memory");  // cols takes the places
  // the CTA's rows: one partial row of each sum
  const int width = p.gpc * p.n;  // columns of this CTA
  for (int q = 0; q < 2 + SCALE; ++q) {
    if (q == 1 && !p.b) continue;
    __syncthreads();
    if (at.on) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int c = (k * p.tpg + at.t) * VEC;
        if (c >= p.n) continue;
        float* o = cols + (long long)at.rs * width + (at.slot % p.gpc) * p.n + c;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
          float v = q == 0 ? gw[k * VEC + i] : gb[k * VEC + i];
          if constexpr (SCALE)
            if (q == 2) v = gs[k * VEC + i];
          o[i] = v;
        }
      }
    }
    __syncthreads();
    const int first = blockIdx.y * width;
    for (int c = threadIdx.x; c < width && first + c < p.D; c += blockDim.x) {
      float a = 0.f;
      for (int i = 0; i < p.rpc; ++i) a += cols[i * width + c];
      p.part[((long long)q * gridDim.x + blockIdx.x) * p.D + first + c] = a;
    }
  }
}

// ------------------------------------------------------------ odd rows --
//
// Rows that do not start on 16 bytes (an odd D). Element by element they cost a
// memory instruction for every 32 elements of every tensor, which is what bounds
// them; but rows of all tensors lie the same way, so a thread takes the 16-byte
// vectors of memory, from the one that the group's first element is in, and only
// what goes by column -- weights in, their gradients' sums -- is shifted with the
// row: these are fp32 in shared memory, column c in plane c % V, so that a warp's
// access to one element of its vectors is to consecutive words. 4097 x 5001 fp16 with
// a residual and a scale, forward and backward: 202 us (0.33 GB), element by element
// 290. The planes' accesses, three or four to an element, and the barriers of rows of
// 5000 bound them: both take half the issue slots.

template <int V>
struct Planes {
  int len;  // every column that a thread's vectors can hold, and the vector before: zeros outside
  __host__ __device__ explicit Planes(int vectors) : len(vectors + 2) {}
  __host__ __device__ int size() const { return V * len; }
  __device__ __forceinline__ int at(int c) const {  // c >= -V
    return (c & (V - 1)) * len + ((c + V) / V);
  }
};

// Where a thread's K vectors lie in a row whose first element is `sh` past the
// aligned one: columns, the places in the planes, and whether all its vectors are
// inside the group (most threads') or need a look at each element.
template <int V, int K>
struct OddRow {
  int sh, n, t, tpg;
  int off[V];  // element i of vector 0, in the planes
  bool edge;
  __device__ __forceinline__ OddRow(const Planes<V>& pl, int sh_, int n_, int t_, int tpg_)
      : sh(sh_), n(n_), t(t_), tpg(tpg_) {
#pragma unroll
    for (int i = 0; i < V; ++i) off[i] = ((i - sh) & (V - 1)) * pl.len + ((i - sh + V) / V) + t;
    edge = t * V < sh || ((K - 1) * tpg + t + 1) * V > sh + n;
  }
  __device__ __forceinline__ int plane(int i) const { return off[i % V] + (i / V) * tpg; }
  __device__ __forceinline__ bool in(int i) const {
    return (unsigned)(((i / V) * tpg + t) * V + i % V - sh) < (unsigned)n;
  }
  // f(i) for the thread's elements inside the group, where zeros will not do
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    if (!edge) {
#pragma unroll
      for (int i = 0; i < K * V; ++i) f(i);
    } else {
#pragma unroll
      for (int i = 0; i < K * V; ++i)
        if (in(i)) f(i);
    }
  }
  // The vectors of one tensor whose group starts at element `start`: loaded whole,
  // the neighbours' elements in them too, where another row follows; and as values,
  // zeros outside the group.
  template <typename T>
  __device__ __forceinline__ static void load(const void* p, long long start, bool last, int sh, int n, int t,
                                              int tpg, uint4 (&raw)[K]) {
    const T* q = static_cast<const T*>(p) + (start - sh) + t * V;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int pos = (k * tpg + t) * V;
      raw[k] = make_uint4(0, 0, 0, 0);
      if (pos < sh + n) {
        if (odd::whole(pos, sh + n, V, last)) {
          raw[k] = __ldg(reinterpret_cast<const uint4*>(q + k * tpg * V));
        } else {
          T e[V];
#pragma unroll
          for (int i = 0; i < V; ++i) e[i] = pos + i < sh + n ? q[k * tpg * V + i] : from_f32<T>(0.f);
          raw[k] = *reinterpret_cast<const uint4*>(e);
        }
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ void get(const uint4 (&raw)[K], float (&v)[K * V]) const {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const T* e = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
      for (int i = 0; i < V; ++i) v[k * V + i] = to_f32<T>(e[i]);
    }
    if (edge) {
#pragma unroll
      for (int i = 0; i < K * V; ++i)
        if (!in(i)) v[i] = 0.f;
    }
  }
  template <typename T>
  __device__ __forceinline__ void store(void* p, long long start, const float (&v)[K * V]) const {
    T* q = static_cast<T*>(p) + (start - sh) + t * V;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = (k * tpg + t) * V - sh;
      uint4 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < V; ++i) e[i] = from_f32<T>(v[k * V + i]);
      if (c >= 0 && c + V <= n) {
        *reinterpret_cast<uint4*>(q + k * tpg * V) = u;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if ((unsigned)(c + i) < (unsigned)n) q[k * tpg * V + i] = e[i];
      }
    }
  }
};

// The CTA's groups' columns of a weight as planes, one group after the other.
template <typename E, int V>
__device__ __forceinline__ void stage_planes(float* o, const void* w, const Args& p, const Planes<V>& pl) {
  const int first = blockIdx.y * p.gpc;
  for (int i = threadIdx.x; i < p.gpc * pl.size(); i += blockDim.x) o[i] = 0.f;
  __syncthreads();
  for (int i = threadIdx.x; i < p.gpc * p.n; i += blockDim.x) {
    const int g = i / p.n, c = i % p.n;
    const long long e = (long long)(first + g) * p.n + c;
    if (first + g < p.G)
      o[g * pl.size() + pl.at(c)] = p.w32 ? static_cast<const float*>(w)[e] : to_f32<E>(static_cast<const E*>(w)[e]);
  }
}

template <typename E, int K, int MAXT>
__global__ void __launch_bounds__(MAXT, odd_fwd_ctas(MAXT)) fwd_odd_kernel(const Args p) {
  constexpr int V = 16 / (int)sizeof(E), N = K * V;
  __shared__ float2 red[2][32];
  extern __shared__ float cols[];
  const Planes<V> pl(K * p.tpg);
  const Place at(p);
  const int width = p.gpc * pl.size(), g0 = (at.slot % p.gpc) * pl.size();
  float *w = cols, *b = w + width, *sc = b + (p.b ? width : 0);
  stage_planes<E, V>(w, p.w, p, pl);
  if (p.b) stage_planes<E, V>(b, p.b, p, pl);
  if (p.s) stage_planes<E, V>(sc, p.s, p, pl);
  __syncthreads();
  if (!at.on) return;
  w += g0, b += g0, sc += g0;
  Reduce sum{red, p.tpg, at.slot, 0};
  const float inv_n = 1.f / (float)p.n;
  const int col = at.g * p.n;
  const long long step = (long long)gridDim.x * p.rpc;
  using R = OddRow<V, K>;
  auto shift = [&](long long row) { return (int)((row * p.ldx + col) & (V - 1)); };
  uint4 rx[K], ra[K];  // of the next row: x, and the residual or else the gate
  auto ahead = [&](long long row) {
    if (row >= p.rows) return;
    const bool last = row + 1 == p.rows;
    const int sh = shift(row);
    R::template load<E>(p.x, row * p.ldx + col, last, sh, p.n, at.t, p.tpg, rx);
    if (p.res)
      R::template load<E>(p.res, row * p.ldres + col, last, sh, p.n, at.t, p.tpg, ra);
    else if (p.gate)
      R::template load<E>(p.gate, row * p.ldgate + col, last, sh, p.n, at.t, p.tpg, ra);
  };
  ahead((long long)blockIdx.x * p.rpc + at.rs);
  for (long long row = (long long)blockIdx.x * p.rpc + at.rs; row < p.rows; row += step) {
    const R at_row(pl, shift(row), p.n, at.t, p.tpg);
    float h[N], a[N];
    at_row.template get<E>(rx, h);
    at_row.template get<E>(ra, a);
    ahead(row + step);
    if (p.s) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] = fmaf(sc[at_row.plane(i)], h[i], a[i]);
    } else if (p.res) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] += a[i];
    }
    if (p.res && p.gate) {
      uint4 rg[K];
      R::template load<E>(p.gate, row * p.ldgate + col, row + 1 == p.rows, at_row.sh, p.n, at.t, p.tpg, rg);
      at_row.template get<E>(rg, a);
    }
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) acc += h[i];
    const float mean = p.rms ? 0.f : sum(acc, 0.f).x * inv_n;
    float sq = 0.f, rs = 0.f;
    at_row.each([&](int i) {
      const float d = h[i] - mean;
      sq = fmaf(d, d, sq);
      rs += d;
    });
    const float2 m = sum(sq, rs);
    const float rest = p.rms ? 0.f : m.y * inv_n;
    const float r = inv_sqrt(at_least_zero(fmaf(-rest, rest, m.x * inv_n)) + p.eps);
    if (p.stats && at.t == 0) {
      float* st = p.stats + (row * p.G + at.g) * 3;
      st[0] = mean, st[1] = rest, st[2] = r;
    }
    const long long o = row * p.D + col;
    if (p.h) at_row.template store<E>(p.h, o, h);
#pragma unroll
    for (int i = 0; i < N; ++i) h[i] = ((h[i] - mean) - rest) * r * w[at_row.plane(i)];
    if (p.b) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] += b[at_row.plane(i)];
    }
    if (p.gate) {
#pragma unroll
      for (int i = 0; i < N; ++i) h[i] *= a[i] * sigm(a[i]);
    }
    at_row.template store<E>(p.y, o, h);
  }
}

template <typename E, int K, int MAXT, bool GATE, bool SCALE>
__global__ void __launch_bounds__(MAXT, odd_bwd_ctas(MAXT)) bwd_odd_kernel(const Args p) {
  constexpr int V = 16 / (int)sizeof(E), N = K * V;
  __shared__ float2 red[2][32];
  extern __shared__ float cols[];
  const Planes<V> pl(K * p.tpg);
  const Place at(p);
  const int width = p.gpc * pl.size(), g0 = (at.slot % p.gpc) * pl.size(), all = p.rpc * width;
  float *w = cols, *b = w + width, *sc = b + (p.b ? width : 0), *gw = sc + (SCALE ? width : 0);
  float *gb = gw + all, *gs = gb + (p.b ? all : 0);
  stage_planes<E, V>(w, p.w, p, pl);
  if (p.b) stage_planes<E, V>(b, p.b, p, pl);
  if (SCALE) stage_planes<E, V>(sc, p.s, p, pl);
  for (int i = threadIdx.x; i < all * (1 + (p.b ? 1 : 0) + SCALE); i += blockDim.x) gw[i] = 0.f;
  __syncthreads();
  if (at.on) {
    const float *ws = w + g0, *bs = b + g0, *ss = sc + g0;
    const int mine = at.rs * width + g0;
    Reduce sum{red, p.tpg, at.slot, 0};
    const float inv_n = 1.f / (float)p.n;
    const int col = at.g * p.n;
    const long long step = (long long)gridDim.x * p.rpc;
    using R = OddRow<V, K>;
    auto shift = [&](long long row) { return (int)((row * p.ldx + col) & (V - 1)); };
    uint4 rx[K], rd[K], ra[K], rh[K];  // of the next row: x, dy, the gate or else the residual, dh
    float stats[3];
    auto ahead = [&](long long row) {
      if (row >= p.rows) return;
      const bool last = row + 1 == p.rows;
      const int sh = shift(row);
      R::template load<E>(p.x, row * p.ldx + col, last, sh, p.n, at.t, p.tpg, rx);
      R::template load<E>(p.dy, row * p.lddy + col, last, sh, p.n, at.t, p.tpg, rd);
      if (GATE)
        R::template load<E>(p.gate, row * p.ldgate + col, last, sh, p.n, at.t, p.tpg, ra);
      else if (SCALE || p.res)
        R::template load<E>(p.res, row * p.ldres + col, last, sh, p.n, at.t, p.tpg, ra);
      if (p.dh) R::template load<E>(p.dh, row * p.lddh + col, last, sh, p.n, at.t, p.tpg, rh);
#pragma unroll
      for (int i = 0; i < 3; ++i) stats[i] = p.stats[(row * p.G + at.g) * 3 + i];
    };
    ahead((long long)blockIdx.x * p.rpc + at.rs);
    for (long long row = (long long)blockIdx.x * p.rpc + at.rs; row < p.rows; row += step) {
      const R at_row(pl, shift(row), p.n, at.t, p.tpg);
      const long long o = row * p.D + col;
      float x[N], d[N], z[N], g[GATE ? N : 1], hh[N];
      at_row.template get<E>(rx, x);
      at_row.template get<E>(rd, d);
      if constexpr (GATE)
        at_row.template get<E>(ra, g);
      else
        at_row.template get<E>(ra, z);
      uint4 keep[K];  // dh, until it is wanted
#pragma unroll
      for (int k = 0; k < K; ++k) keep[k] = rh[k];
      const float mean = stats[0], rest = stats[1], r = stats[2];
      ahead(row + step);
      if (SCALE || p.res) {
        if (GATE) {
          uint4 rr[K];
          R::template load<E>(p.res, row * p.ldres + col, row + 1 == p.rows, at_row.sh, p.n, at.t, p.tpg, rr);
          at_row.template get<E>(rr, z);
        }
        if constexpr (SCALE) {
#pragma unroll
          for (int i = 0; i < N; ++i) z[i] = fmaf(ss[at_row.plane(i)], x[i], z[i]);
        } else {
#pragma unroll
          for (int i = 0; i < N; ++i) z[i] += x[i];
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) z[i] = x[i];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = ((z[i] - mean) - rest) * r;
      if constexpr (GATE) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int e = at_row.plane(i);
          const float sg = sigm(g[i]), a = fmaf(z[i], ws[e], p.b ? bs[e] : 0.f), dd = d[i];
          d[i] = dd * g[i] * sg;
          g[i] = dd * a * sg * fmaf(g[i], 1.f - sg, 1.f);
        }
        at_row.template store<E>(p.dgate, o, g);
      }
      float s1 = 0.f, s2 = 0.f;
      float *gwr = gw + mine, *gbr = gb + mine, *gsr = gs + mine;
#pragma unroll
      for (int i = 0; i < N; ++i) {  // outside the group d and the weights are zeros
        const int e = at_row.plane(i);
        gwr[e] = fmaf(d[i], z[i], gwr[e]);
        if (p.b) gbr[e] += d[i];
        d[i] *= ws[e];
        s1 += d[i];
        s2 = fmaf(d[i], z[i], s2);
      }
      const float2 m = sum(s1, s2);
      const float m1 = p.rms ? 0.f : m.x * inv_n, m2 = m.y * inv_n;
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = r * (d[i] - m1 - z[i] * m2);
      if (p.dh) {
        at_row.template get<E>(keep, hh);
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] += hh[i];
      }
      if constexpr (SCALE) {
        at_row.template store<E>(p.dres, o, d);
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const int e = at_row.plane(i);
          gsr[e] = fmaf(d[i], x[i], gsr[e]);
          d[i] *= ss[e];
        }
      }
      at_row.template store<E>(p.dx, o, d);
    }
  }
  // the CTA's rows: one partial row of each sum
  __syncthreads();
  const int first = blockIdx.y * p.gpc;
  for (int q = 0; q < 2 + SCALE; ++q) {
    if (q == 1 && !p.b) continue;
    const float* s = q == 0 ? gw : q == 1 ? gb : gs;
    for (int i = threadIdx.x; i < p.gpc * p.n; i += blockDim.x) {
      const int g = i / p.n, c = i % p.n;
      if (first + g >= p.G) break;
      float a = 0.f;
      for (int k = 0; k < p.rpc; ++k) a += s[k * width + g * pl.size() + pl.at(c)];
      p.part[((long long)q * gridDim.x + blockIdx.x) * p.D + (first + g) * p.n + c] = a;
    }
  }
}

// Partial rows -> dweight, dbias, dscale (blockIdx.y), 32 columns to a CTA.
template <typename W>
__global__ void __launch_bounds__(1024) sum_kernel(const float* part, W* dw, W* db, W* ds, int n, int D) {
  __shared__ float s[32][33];
  W* out = blockIdx.y == 0 ? dw : blockIdx.y == 1 ? db : ds;
  if (!out) return;
  const int c = blockIdx.x * 32 + threadIdx.x;
  const float* q = part + (long long)blockIdx.y * n * D;
  float a = 0.f;
  if (c < D)
    for (int i = threadIdx.y; i < n; i += 32) a += q[(long long)i * D + c];
  s[threadIdx.y][threadIdx.x] = a;
  __syncthreads();
  a = s[threadIdx.x][threadIdx.y];  // column threadIdx.y, partial threadIdx.x
  for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
  const int col = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && col < D) out[col] = from_f32<W>(a);
}

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = 148;  // no device here: the sizes of a B200
  }
  return n;
}

enum Way { kElements, kVectors, kOdd };  // how rows are read

struct Plan {
  Way way;
  int vec, k, tpg, gpc, rpc, threads;
  unsigned gx, gy;
  size_t odd_smem;
};

// Threads to a group: as few as hold it at `values` each (a row's sums then need
// few steps, and more rows are under way), a part of a warp or whole warps;
// groups side by side in a CTA as they lie in a row. 16 values forward; 8
// backward, which keeps seven arrays of them in registers, while a CTA of 1024
// threads holds the group at that (odd rows, backward: 16 values took 235 us where 8
// take 125).
bool make_plan(Plan& pl, long long rows, int D, int G, int size, Way way, bool fwd, int weights) {
  const int n = D / G;
  if (n > kMaxGroup) return false;
  const bool vec = way != kElements, odd = way == kOdd;
  const int values = fwd || n > kMaxGroup / 2 ? 16 : 8;
  pl.way = way;
  pl.vec = vec ? 16 / size : 1;
  const int need = (n + (odd ? pl.vec - 1 : 0) + pl.vec - 1) / pl.vec, most = values / pl.vec;
  pl.k = 1;
  while (pl.k < most && pl.k * 8 < need) pl.k *= 2;
  if (!vec && pl.k < 4) pl.k = 4;
  const int t = (need + pl.k - 1) / pl.k;
  pl.tpg = t <= 8 ? 8 : t <= 16 ? 16 : (t + 31) / 32 * 32;
  pl.threads = pl.tpg > kThreads ? pl.tpg : kThreads;
  pl.gpc = pl.threads / pl.tpg < G ? pl.threads / pl.tpg : G;
  pl.rpc = pl.threads / (pl.tpg * pl.gpc);
  pl.gy = (unsigned)((G + pl.gpc - 1) / pl.gpc);
  if (odd) {  // planes of the weights, and backward of their gradients' sums
    const size_t planes = (size_t)pl.vec * (pl.k * pl.tpg + 2) * pl.gpc * sizeof(float);
    pl.odd_smem = planes * weights * (fwd ? 1 : 1 + pl.rpc);
    if (pl.odd_smem > 200 * 1024 || pl.threads > 1024 || n > (fwd ? kMaxGroup : kMaxGroup / 2) - 8) return false;
  }
  // a few CTAs to an SM, each walking rows
  int per_sm = fwd ? 1024 / pl.threads : pl.threads > 512 ? 1 : pl.threads > 256 ? 2 : 3;
  if (odd) per_sm = fwd ? (pl.threads > 384 ? 1 : pl.threads > 256 ? 2 : 3) : pl.threads > 256 ? 1 : 2;
  const long long most_x = ((long long)sm_count() * per_sm + pl.gy - 1) / pl.gy;
  const long long want = (rows + pl.rpc - 1) / pl.rpc;
  pl.gx = (unsigned)(want < most_x ? (want < 1 ? 1 : want) : most_x);
  return true;
}

// The kernels that make_plan's rules reach: the most values to a thread with any
// number of threads, fewer with the smallest groups only.
#define MGS_NORM_CASE(v, kk, maxt) \
  if (pl.vec == v && pl.k == kk && pl.threads <= maxt) return MGS_NORM_KERNEL(v, kk, maxt);
#define MGS_NORM_SIZES(v, kk) MGS_NORM_CASE(v, kk, 256) MGS_NORM_CASE(v, kk, 512) MGS_NORM_CASE(v, kk, 1024)

#define MGS_NORM_ODD(kk, maxt) \
  if (pl.k == kk && pl.threads <= maxt) return MGS_NORM_ODD_KERNEL(kk, maxt);
#define MGS_NORM_ODD_SIZES(kk, mid) \
  MGS_NORM_ODD(kk, 256) MGS_NORM_ODD(kk, mid) MGS_NORM_ODD(kk, 768) MGS_NORM_ODD(kk, 1024)

template <typename E, typename W, class F>
int by_plan_fwd(const Plan& pl, F&& f) {
  constexpr int V = 16 / (int)sizeof(E);
  if (pl.way == kOdd) {
#define MGS_NORM_ODD_KERNEL(kk, maxt) f(fwd_odd_kernel<E, kk, maxt>)
    MGS_NORM_ODD(1, 256)
    if constexpr (V == 4) {
      MGS_NORM_ODD(2, 256)
    }
    MGS_NORM_ODD_SIZES(16 / V, 384)
#undef MGS_NORM_ODD_KERNEL
    return MGS_UNSUPPORTED;
  }
#define MGS_NORM_KERNEL(v, kk, maxt) f(fwd_kernel<E, W, v, kk, maxt>)
  MGS_NORM_CASE(V, 1, 256)
  if constexpr (V == 4) {
    MGS_NORM_CASE(V, 2, 256)
  }
  MGS_NORM_SIZES(V, 16 / V)
  MGS_NORM_CASE(1, 4, 256)
  MGS_NORM_CASE(1, 8, 256)
  MGS_NORM_SIZES(1, 16)
#undef MGS_NORM_KERNEL
  return MGS_UNSUPPORTED;
}

template <typename E, typename W, bool GATE, bool SCALE, class F>
int by_plan_bwd(const Plan& pl, F&& f) {
  constexpr int V = 16 / (int)sizeof(E);
  if (pl.way == kOdd) {
#define MGS_NORM_ODD_KERNEL(kk, maxt) f(bwd_odd_kernel<E, kk, maxt, GATE, SCALE>)
    if constexpr (V == 4) {
      MGS_NORM_ODD(1, 256)
    }
    MGS_NORM_ODD_SIZES(8 / V, 512)
#undef MGS_NORM_ODD_KERNEL
    return MGS_UNSUPPORTED;
  }
#define MGS_NORM_KERNEL(v, kk, maxt) f(bwd_kernel<E, W, v, kk, maxt, GATE, SCALE>)
  if constexpr (V == 4) {
    MGS_NORM_CASE(V, 1, 256)
  }
  MGS_NORM_SIZES(V, 8 / V)
  MGS_NORM_CASE(V, 16 / V, 1024)
  MGS_NORM_CASE(1, 4, 256)
  MGS_NORM_SIZES(1, 8)
  MGS_NORM_CASE(1, 16, 1024)
#undef MGS_NORM_KERNEL
  return MGS_UNSUPPORTED;
}
#undef MGS_NORM_SIZES
#undef MGS_NORM_CASE
#undef MGS_NORM_ODD_SIZES
#undef MGS_NORM_ODD

template <class F>
int by_dtypes(int dtype, int wdtype, F&& f) {
  const bool same = dtype == wdtype;
  if (!same && wdtype != MGS_F32) return MGS_BAD_DTYPE;
  switch (dtype) {
    case MGS_F32: return f(float{}, float{});
    case MGS_BF16: return same ? f(__nv_bfloat16{}, __nv_bfloat16{}) : f(__nv_bfloat16{}, float{});
    case MGS_F16: return same ? f(__half{}, __half{}) : f(__half{}, float{});
    default: return MGS_BAD_DTYPE;
  }
}

bool shape_ok(int64_t rows, int64_t D, int groups) {
  return rows >= 0 && D >= 1 && D <= 0x3fffffff && groups >= 1 && D % groups == 0;
}

// How a call's rows can be read: whole 16-byte vectors everywhere (addresses, row
// strides, group starts); vectors of memory with the columns shifted from row to
// row, where that shift is the same for all tensors and nothing past their ends is
// read; or element by element.
Way way_of(const Args& a, int size, int wsize) {
  const int v = 16 / size;
  bool vec = a.n % v == 0 && (long long)a.n * wsize % 16 == 0, odd = true;
  for (const void* q : {a.x, a.res, a.gate, a.dy, a.dh, (const void*)a.y, (const void*)a.h, (const void*)a.dx,
                        (const void*)a.dres, (const void*)a.dgate})
    odd = odd && aligned(q, 16);
  vec = vec && odd;
  for (const void* q : {a.w, a.b, a.s}) vec = vec && aligned(q, 16);
  const long long out = a.D % v;  // of the dense outputs
  for (auto [q, ld] : {std::pair(a.x, a.ldx), std::pair(a.res, a.ldres), std::pair(a.gate, a.ldgate),
                       std::pair(a.dy, a.lddy), std::pair(a.dh, a.lddh)})
    if (q) {
      vec = vec && ld % v == 0;
      odd = odd && ld % v == out && (a.rows == 1 || odd::steps_far_enough(ld, v));
    }
  vec = vec && (out == 0 || a.rows == 1);
  return vec ? kVectors : odd ? kOdd : kElements;
}

// The plan of a call's way, or of single elements where that does not fit.
bool plan_call(Plan& pl, const Args& a, int size, int wsize, bool fwd) {
  const int weights = 1 + (a.b ? 1 : 0) + (a.s ? 1 : 0);
  return make_plan(pl, a.rows, a.D, a.G, size, way_of(a, size, wsize), fwd, weights) ||
         make_plan(pl, a.rows, a.D, a.G, size, kElements, fwd, weights);
}

void set_plan(Args& a, const Plan& pl) { a.tpg = pl.tpg, a.gpc = pl.gpc, a.rpc = pl.rpc; }

int launched() { return cudaGetLastError() == cudaSuccess ? MGS_OK : MGS_LAUNCH_FAILED; }

}  // namespace
}  // namespace norm
}  // namespace mgs

extern "C" {

size_t mgs_block_norm_workspace_size(int64_t rows, int64_t D, int groups, int dtype) {
  using namespace mgs::norm;
  const int size = mgs::dtype_size(dtype);
  if (!shape_ok(rows, D, groups) || size == 0) return 0;
  size_t most = 0;
  for (Way way : {kElements, kVectors, kOdd}) {
    Plan pl;
    if (!make_plan(pl, rows, (int)D, groups, size, way, false, 1)) {
      if (way == kOdd) continue;
      return 0;
    }
    const size_t n = 3 * (size_t)pl.gx * (size_t)D * sizeof(float);
    most = n > most ? n : most;
  }
  return most;
}

int mgs_block_norm_fwd(const void* x, const void* residual, const void* gate, const void* weight,
                       const void* bias, const void* scale, void* y, void* h, float* stats,
                       const int64_t* row_strides, int64_t rows, int64_t D, int groups, int rms,
                       float eps, int dtype, int weight_dtype, void* stream) {
  using namespace mgs::norm;
  if (!shape_ok(rows, D, groups) || (scale && !residual) || (residual && !h)) return MGS_BAD_SHAPE;
  return by_dtypes(dtype, weight_dtype, [&](auto e, auto wt) -> int {
    using E = decltype(e);
    using W = decltype(wt);
    if (rows == 0) return MGS_OK;
    Args a{};
    a.x = x, a.res = residual, a.gate = gate, a.w = weight, a.b = bias, a.s = scale, a.y = y;
    a.h = residual ? h : nullptr, a.stats = stats;
    a.ldx = row_strides[0], a.ldres = row_strides[1], a.ldgate = row_strides[2];
    a.rows = rows, a.D = (int)D, a.G = groups, a.n = (int)D / groups, a.rms = rms, a.eps = eps;
    a.w32 = std::is_same_v<W, float>;
    Plan pl;
    if (!plan_call(pl, a, sizeof(E), sizeof(W), true)) return MGS_UNSUPPORTED;
    if (pl.gy > 65535) return MGS_UNSUPPORTED;
    set_plan(a, pl);
    return by_plan_fwd<E, W>(pl, [&](auto fwd) -> int {
      const size_t smem = pl.way == kOdd ? pl.odd_smem : 0;
      if (smem > 40 * 1024)
        MGS_CUDA_OK(cudaFuncSetAttribute(fwd, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      fwd<<<dim3(pl.gx, pl.gy), pl.threads, smem, static_cast<cudaStream_t>(stream)>>>(a);
      return launched();
    });
  });
}

int mgs_block_norm_bwd(const void* x, const void* residual, const void* gate, const void* weight,
                       const void* bias, const void* scale, const float* stats, const void* dy,
                       const void* dh, void* dx, void* dresidual, void* dgate, void* dweight, void* dbias,
                       void* dscale, const int64_t* row_strides, int64_t rows, int64_t D, int groups,
                       int rms, int dtype, int weight_dtype, void* workspace, size_t workspace_bytes,
                       void* stream) {
  using namespace mgs::norm;
  if (!shape_ok(rows, D, groups) || (scale && (!residual || !dresidual || !dscale)) || (gate && !dgate) ||
      (bias && !dbias))
    return MGS_BAD_SHAPE;
  return by_dtypes(dtype, weight_dtype, [&](auto e, auto wt) -> int {
    using E = decltype(e);
    using W = decltype(wt);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
      for (void* q : {dweight, bias ? dbias : nullptr, scale ? dscale : nullptr})
        if (q) MGS_CUDA_OK(cudaMemsetAsync(q, 0, (size_t)D * sizeof(W), st));
      return MGS_OK;
    }
    Args a{};
    a.x = x, a.res = residual, a.gate = gate, a.w = weight, a.b = bias, a.s = scale;
    a.dy = dy, a.dh = dh, a.dx = dx, a.dres = dresidual, a.dgate = dgate;
    a.stats = const_cast<float*>(stats), a.part = static_cast<float*>(workspace);
    a.ldx = row_strides[0], a.ldres = row_strides[1], a.ldgate = row_strides[2], a.lddy = row_strides[3],
    a.lddh = row_strides[4];
    a.rows = rows, a.D = (int)D, a.G = groups, a.n = (int)D / groups, a.rms = rms;
    a.w32 = std::is_same_v<W, float>;
    Plan pl;
    if (!plan_call(pl, a, sizeof(E), sizeof(W), false)) return MGS_UNSUPPORTED;
    if (pl.gy > 65535) return MGS_UNSUPPORTED;
    if (workspace_bytes < 3 * (size_t)pl.gx * (size_t)D * sizeof(float)) return MGS_WORKSPACE_TOO_SMALL;
    set_plan(a, pl);
    auto launch = [&](auto bwd) -> int {
      size_t smem = pl.way == kOdd ? pl.odd_smem : (size_t)pl.rpc * pl.gpc * a.n * sizeof(float);
      if (pl.way == kVectors) {  // two rows' inputs, where the SM has room for its CTAs
        const int inputs = 2 + (residual != nullptr) + (gate != nullptr) + (dh != nullptr);
        const size_t places = (size_t)2 * inputs * pl.k * pl.vec * sizeof(E) * pl.threads;
        const int ctas = pl.threads > 512 ? 1 : pl.threads > 256 ? 2 : 3;
        if (ctas * (places + 2048) <= 224 * 1024) {
          a.staged = inputs;
          smem = smem > places ? smem : places;
        }
      }
      if (smem > 40 * 1024)
        MGS_CUDA_OK(cudaFuncSetAttribute(bwd, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
      bwd<<<dim3(pl.gx, pl.gy), pl.threads, smem, st>>>(a);
      return launched();
    };
    int r;
    if (gate)
      r = scale ? by_plan_bwd<E, W, true, true>(pl, launch) : by_plan_bwd<E, W, true, false>(pl, launch);
    else
      r = scale ? by_plan_bwd<E, W, false, true>(pl, launch) : by_plan_bwd<E, W, false, false>(pl, launch);
    if (r) return r;
    sum_kernel<W><<<dim3((unsigned)((D + 31) / 32), 3), dim3(32, 32), 0, st>>>(
        a.part, static_cast<W*>(dweight), bias ? static_cast<W*>(dbias) : nullptr,
        scale ? static_cast<W*>(dscale) : nullptr, (int)pl.gx, (int)D);
    return launched();
  });
}

}  // extern "C"
