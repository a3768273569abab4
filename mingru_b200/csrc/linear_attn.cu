// linear_attn.cu -- linear attention with a decay for each head, over whole
// sequences, on the tcgen05 tensor cores (forward and backward).
//
// Per (batch, head), with gamma_t = exp(log_gamma_t) <= 1:
//   S_t = gamma_t S_{t-1} + k_t v_t^T        (d_k x d_v, fp32)
//   y_t = S_t^T q_t
// In chunks of C = 128 tokens, c_i the inclusive sum of log_gamma inside the
// chunk, S the state that enters it, D_ij = exp(c_i - c_j) for j <= i, else 0:
//   y  = (D * Q K^T) V + diag(e^{c}) Q S
//   S' = e^{c_C} S + K^T diag(e^{c_C - c}) V
// and, with dS' the gradient of the state that leaves it:
//   dQ = (D * dy V^T) K   + diag(e^{c}) dy S^T
//   dK = (D * dy V^T)^T Q + diag(e^{c_C - c}) V dS'^T
//   dV = (D * Q K^T)^T dy + diag(e^{c_C - c}) K dS'
//   dS = e^{c_C} dS' + Q^T diag(e^{c}) dy
//   dlog_gamma_t = sum_{i >= t > j} R_ij + sum_{i >= t} q_i . dQ'_i
//                + sum_{j < t} k_j . dK'_j + e^{c_C} <S, dS'>
// with R = D * Q K^T * dy V^T and dQ', dK' the state parts of dQ and dK: every
// term is one whose span of decays holds token t.
//
// Decays. The sums are formed in base 2 and kept as ch + cl, ch a multiple of
// 2^-9 (exact sums and differences in fp32) and cl the small rest, so that
// exp(c_i - c_j) is as good for two tokens late in a chunk of strong decays
// as for the first two. A token's log2 decay is held to >= -128: 2^-128 is
// below what fp32 keeps, so the state is wiped exactly (log_gamma = -inf, the
// start of a packed document, included) and nothing becomes inf - inf.
//
// Operands. The tensor cores take bf16; a value is held as up to three bf16
// levels (x = h + m + l to 2^-24) and a product takes the level pairs (i, j)
// with i + j <= 2. bf16 inputs are exact in one level, fp16 in two, fp32 in
// three. What is computed here -- masked products, states, decayed rows -- is
// held in as many levels as the result needs: those that end in a 16-bit
// output as many as the inputs (the rounding is of the size of the output's),
// those that end in a state or in dlog_gamma, which are fp32, in three.
// Accumulators, states and sums are fp32 (TMEM and registers).
//
// Sequences are split into segments of whole chunks where there are fewer
// (batch, head) pairs than CTAs fit the GPU: state_kernel sums what a segment
// adds to the state, scan_kernel joins these along the sequence, and the main
// kernels then run all segments at once, chunk by chunk inside each.
//
// What bounds them (8 x 8 heads of 64, T = 8192, bf16, 0.54 GB for forward and
// backward: 84 us at copy speed; 430 are taken): neither DRAM (27 to 48% of its peak)
// nor the tensor pipe (22 to 26%) but the chain inside a chunk -- products, mask,
// products that use it, sums that read those -- of which an SM has two under way, and
// the instructions of masking, scaling and rounding (37 to 47% of the issue slots).
// So the work on this chain is what each choice below is about.
#include <type_traits>

#include "common.cuh"
#include "umma.cuh"

namespace mgs {
namespace lattn {
namespace {

using bf16 = __nv_bfloat16;
namespace um = umma;

constexpr int kC = 128;        // tokens of a chunk: the rows of an M = 128 accumulator
// A CTA has two or four warps for each quarter of the TMEM lanes: 256 threads where
// two or three CTAs share an SM, 512 where one has it. "Part" is a warp's share of
// an accumulator's columns, warp / 4.
constexpr float kMinLog2 = -128.f;
// Polls of an mbarrier before a wait gives up (each suspends for some 10 us: over a second).
constexpr long long kPolls = 1ll << 17;

template <typename E>
constexpr int kLevels = 1;
template <>
constexpr int kLevels<__half> = 2;
template <>
constexpr int kLevels<float> = 3;

// A (B, H, T, d) tensor: base and strides in elements (the last dimension is
// dense); vec: every row starts on 16 bytes and holds whole groups of 8, wide:
// on 32 bytes and whole groups of 32 bytes.
template <typename P>
struct Ten {
  P* p;
  long long sb, sh, st;
  int vec, wide;
  // outputs that are sums over blocks of the heads: fp32 rows of 64 (BH, T, 64)
  float* part;
  int mode;
};
constexpr int kAdd = 1, kKeep = 2;  // part holds earlier blocks' share; more blocks follow

template <typename E>
struct Args {
  CUtensorMap mQ, mK, mV, mdy, my, mdQ, mdK, mdV;  // bf16 with tma set
  int tma;                                         // every tensor has a map
  Ten<const E> Q, K, V, dy;
  Ten<E> y, dQ, dK, dV;
  const float* lg;
  long long lsb, lsh, lst;
  const float* H0;   // (B, H, dk, dv) or null: zeros
  float* HT;         // forward: (B, H, dk, dv)
  const float* dHT;  // (B, H, dk, dv) or null: zeros
  float* dH0;        // (B, H, dk, dv) or null: not wanted
  float* dlg;        // (B, H, T)
  float* saved;      // (BH, nchunks, D * D) states at the chunks' starts, or null: no backward
  float* seg;        // (BH, nsub, D * D) states at the parts' starts (backward: ends) (workspace)
  float* segl;       // (BH, nsub) log2 of each part's total decay (workspace)
  float* rows_R;     // (BH, T) a token's sum of R over the tokens before it in its chunk (workspace)
  float* state_q;    // (BH, T) q . the state part of its gradient (workspace)
  float* quarters;   // (BH, nchunks, 16) sums of R over quarters of rows (4) and of columns (workspace)
  long long T;
  int H, dk, dv, nchunks, m, nseg;  // m chunks to a segment
  int ms, r, nsub;                  // segments in r parts of ms chunks for the state sums, nsub in all
  long long BH;
  long long sbh;  // H0, H_T and their gradients: from one (batch, head) to the next,
  int sld;        // and from one row to the next
  int dlg_add;    // dlog_gamma holds earlier blocks' share
};

// ------------------------------------------------------------- tile loads --

// x[0..7] -> NL bf16 levels at element offset o of tiles `stride` elements apart.
template <int NL>
__device__ __forceinline__ void store_levels8(bf16* t, long long stride, int o, const float* x) {
  uint32_t w[NL][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float a = x[2 * i], b = x[2 * i + 1];
#pragma unroll
    for (int l = 0; l < NL; ++l) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
      w[l][i] = *reinterpret_cast<const uint32_t*>(&h);
      if (l + 1 < NL) {
        const float2 f = __bfloat1622float2(h);
        a -= f.x;
        b -= f.y;
      }
    }
  }
#pragma unroll
  for (int l = 0; l < NL; ++l)
    *reinterpret_cast<uint4*>(t + l * stride + o) = make_uint4(w[l][0], w[l][1], w[l][2], w[l][3]);
}

// Sum of the levels of 8 consecutive elements.
template <int NL>
__device__ __forceinline__ void load_levels8(const bf16* t, long long stride, int o, float* x) {
#pragma unroll
  for (int l = 0; l < NL; ++l) {
    const uint4 u = *reinterpret_cast<const uint4*>(t + l * stride + o);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[i]));
      x[2 * i] = l == 0 ? f.x : x[2 * i] + f.x;
      x[2 * i + 1] = l == 0 ? f.y : x[2 * i + 1] + f.y;
    }
  }
}

// Tiles are what the tensor maps' 128-byte swizzle makes of 64 columns: rows of
// 128 bytes, the 16-byte group g of row r at group g ^ (r % 8); wider tiles are
// such halves one after the other. Reading or writing a row with a lane for each
// row, or whole rows with eight lanes to a row, is free of bank conflicts.
template <int R>
__device__ __forceinline__ int sw(int r, int c) {
  return (c >> 6) * (R * 64) + r * 64 + ((((c >> 3) & 7) ^ (r & 7)) << 3) + (c & 7);
}

// A 128 x D tile in items of 16 bytes in memory order: thread t of NT has items t,
// t + NT, ..., which are the same columns of rows NT / 8 apart in each half.
template <int D, int NT>
struct Items {
  static constexpr int kN = kC * D / 8 / NT, kHalf = 1024 / NT;
  __device__ static int row(int i) { return (i % kHalf) * (NT / 8) + (threadIdx.x >> 3); }
  __device__ static int col(int i) {
    return (i / kHalf) * 64 + (((threadIdx.x & 7) ^ ((threadIdx.x >> 3) & 7)) << 3);
  }
  __device__ static int offset(int i) { return 8 * (i * NT + (int)threadIdx.x); }
};

// Rows [t0, t0 + n) of a head as bf16 levels in a tile, through registers; rows
// from n on and columns from d are zeros.
template <typename E, int D, int NT>
__device__ __forceinline__ void load_tile(bf16* tile, const Ten<const E>& x, long long b, long long h,
                                          long long t0, int n, int d) {
  using I = Items<D, NT>;
  constexpr int NL = kLevels<E>;
  const E* head = x.p + b * x.sb + h * x.sh + t0 * x.st;
#pragma unroll
  for (int i = 0; i < I::kN; ++i) {
    const int r = I::row(i), c = I::col(i);
    const E* s = head + r * x.st + c;
    float v[8];
    if (x.vec) {
      if (r < n && c < d) {
        constexpr int kN = 16 / (int)sizeof(E);
#pragma unroll
        for (int k = 0; k < 8; k += kN) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(s + k));
          const E* e = reinterpret_cast<const E*>(&u);
#pragma unroll
          for (int j = 0; j < kN; ++j) v[k + j] = to_f32<E>(e[j]);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = 0.f;
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = r < n && c + j < d ? to_f32<E>(s[j]) : 0.f;
    }
    store_levels8<NL>(tile, kC * D, I::offset(i), v);
  }
}

// The same rows into L2, ahead of their load.
template <typename E>
__device__ __forceinline__ void prefetch_rows(const Ten<const E>& x, long long b, long long h, long long t0,
                                              int n, int d) {
  const E* head = x.p + b * x.sb + h * x.sh + t0 * x.st;
  const int bytes = d * (int)sizeof(E), lines = (bytes + 127) / 128;
  for (int i = threadIdx.x; i < n * lines; i += (int)blockDim.x) {
    const char* a = reinterpret_cast<const char*>(head + (i / lines) * x.st) + (i % lines) * 128;
    asm volatile("prefetch.global.L2 [%0];" ::"l"(a));
  }
}

// bf16 tensors that a tensor map can describe (columns, time, head, batch) come
// and go by TMA, one thread issuing: rows and columns outside read as zeros and
// are not written.
template <int D>
__device__ __forceinline__ void tma_load(bf16* tile, const CUtensorMap* m, long long t0, int h, int b,
                                         uint64_t* bar) {
#pragma unroll
  for (int x = 0; x < D; x += 64)
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(smem_u32(tile + x * kC)),
        "l"(reinterpret_cast<uint64_t>(m)), "r"(x), "r"((int)t0), "r"(h), "r"(b), "r"(smem_u32(bar))
        : "memory");
}
template <int D>
__device__ __forceinline__ void tma_store(const CUtensorMap* m, long long t0, int h, int b, int d,
                                          const bf16* tile) {
#pragma unroll
  for (int x = 0; x < D; x += 64) {
    if (x >= d) break;
    asm volatile(
        "cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
            reinterpret_cast<uint64_t>(m)),
        "r"(x), "r"((int)t0), "r"(h), "r"(b), "r"(smem_u32(tile + x * kC))
        : "memory");
  }
  bulk_commit();
}
template <int D>
__device__ __forceinline__ void tma_prefetch(const CUtensorMap* m, long long t0, int h, int b, int d) {
#pragma unroll
  for (int x = 0; x < D; x += 64)
    if (x < d)
    asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(
                     reinterpret_cast<uint64_t>(m)),
                 "r"(x), "r"((int)t0), "r"(h), "r"(b)
                 : "memory");
}
constexpr int tile_bytes(int D) { return kC * D * 2; }

// 16 values of one row (columns c0.., c0 % 16 == 0) into a bf16 tile.
__device__ __forceinline__ void row16_to_tile(bf16* tile, int r, int c0, const float (&v)[16]) {
  store_levels8<1>(tile, 0, sw<kC>(r, c0), v);
  store_levels8<1>(tile, 0, sw<kC>(r, c0 + 8), v + 8);
}

// 16 values of row t (columns c0..) of a head's output, in whole 32-byte sectors
// where the rows allow it.
template <typename E>
__device__ __forceinline__ void store_row16(const Ten<E>& x, int b, int h, int H, long long t, long long T, int c0,
                                            int d, float (&v)[16]) {
  if (x.mode) {
    float4* o = reinterpret_cast<float4*>(x.part + (((long long)b * H + h) * T + t) * 64 + c0);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (x.mode & kAdd) {
        const float4 f = o[k];
        v[4 * k] += f.x, v[4 * k + 1] += f.y, v[4 * k + 2] += f.z, v[4 * k + 3] += f.w;
      }
      if (x.mode & kKeep) o[k] = make_float4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]);
    }
    if (x.mode & kKeep) return;
  }
  E* row = x.p + b * x.sb + h * x.sh + t * x.st;
  if (x.vec) {
    constexpr int kN = 32 / (int)sizeof(E);
#pragma unroll
    for (int k = 0; k < 16; k += kN) {
      uint32_t w[8];
      E* e = reinterpret_cast<E*>(w);
#pragma unroll
      for (int i = 0; i < kN; ++i) e[i] = from_f32<E>(v[k + i]);
      E* o = row + c0 + k;
      if (x.wide) {
        if (c0 + k < d)
          asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(o), "r"(w[0]), "r"(w[1]),
                       "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                       : "memory");
      } else {
        if (c0 + k < d) *reinterpret_cast<uint4*>(o) = make_uint4(w[0], w[1], w[2], w[3]);
        if (c0 + k + kN / 2 < d) *reinterpret_cast<uint4*>(o + kN / 2) = make_uint4(w[4], w[5], w[6], w[7]);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i)
      if (c0 + i < d) row[c0 + i] = from_f32<E>(v[i]);
  }
}

// ----------------------------------------------------------------- decays --

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A chunk's decays: inclusive sums of the log2 decays as ch + cl, and cf, a
// token's factor to the edge of its block of 16: 2^(c_last - c_t) (kStart:
// 2^(c_t - c_first)). For a whole block on one side of token i the factor
// between i and any t of it is one of i's to the block's edge times cf[t], both
// <= 1, so nothing is lost that the product would keep.
struct Decays {
  float ch[kC], cl[kC], cf[kC];
  __device__ __forceinline__ float to(float h, float l, int t) const { return ex2((h - ch[t]) + (l - cl[t])); }
  __device__ __forceinline__ float from(float h, float l, int t) const { return ex2((ch[t] - h) + (cl[t] - l)); }
};

// By one warp, four tokens to a lane. Tokens from n on add nothing. A token's log2
// decay is split into a multiple of 2^-9, whose sums fp32 holds exactly, and the
// rest, below 2^-10, whose sums stay below 1/8.
struct DecayWarp {
  float lg[4];
  __device__ __forceinline__ void load(const float* p, long long st, int n) {
    const int t0 = 4 * (threadIdx.x & 31);
#pragma unroll
    for (int i = 0; i < 4; ++i) lg[i] = t0 + i < n ? p[(t0 + i) * st] : 0.f;
  }
  template <bool kStart>
  __device__ __forceinline__ void table(Decays& o) const {
    constexpr float kLog2e = 1.44269502f, kLog2eLow = 1.92596299e-8f;  // their sum is log2(e) to 2^-49
    const int lane = threadIdx.x & 31;
    float h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float v = lg[i] * kLog2e;
      float rest = fmaf(lg[i], kLog2eLow, fmaf(lg[i], kLog2e, -v));
      if (v < kMinLog2) v = kMinLog2, rest = 0.f;
      h[i] = rintf(v * 512.f) * (1.f / 512.f);
      l[i] = (v - h[i]) + rest;
      if (i > 0) h[i] += h[i - 1], l[i] += l[i - 1];
    }
    float ih = h[3], il = l[3];
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const float x = __shfl_up_sync(0xffffffffu, ih, d), y = __shfl_up_sync(0xffffffffu, il, d);
      if (lane >= d) ih += x, il += y;
    }
    const float bh = ih - h[3], bl = il - l[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] += bh, l[i] += bl;
    const int edge = kStart ? lane & ~3 : lane | 3;
    const float eh = __shfl_sync(0xffffffffu, kStart ? h[0] : h[3], edge);
    const float el = __shfl_sync(0xffffffffu, kStart ? l[0] : l[3], edge);
    float4 ch, cl, cf;
    float *ph = &ch.x, *pl = &cl.x, *pf = &cf.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ph[i] = h[i], pl[i] = l[i];
      pf[i] = kStart ? ex2((h[i] - eh) + (l[i] - el)) : ex2((eh - h[i]) + (el - l[i]));
    }
    *reinterpret_cast<float4*>(o.ch + 4 * lane) = ch;
    *reinterpret_cast<float4*>(o.cl + 4 * lane) = cl;
    *reinterpret_cast<float4*>(o.cf + 4 * lane) = cf;
  }
};

// A sum as two fp32 numbers, the second what the first's roundings lost (Knuth).
struct Two {
  float s, e;
  __device__ __forceinline__ void add(float x) {
    const float t = s + x, b = t - s;
    e += (s - (t - b)) + (x - b);
    s = t;
  }
  __device__ __forceinline__ void add(const Two& o) {
    add(o.s);
    e += o.e;
  }
};

// ------------------------------------------------------------ MMA issuing --

// A tile of R rows as an operand: contraction over its columns (K-major) or
// over its rows (MN-major), as descriptors of the 128-byte swizzle (groups of
// eight rows 1024 bytes apart, halves of 64 columns R rows apart).
template <int R>
struct Op {
  uint64_t d;
  uint32_t level;  // from one level to the next, in 16-byte units
  bool mn;
  // k-th step of 16 along the contraction, in 16-byte units
  __device__ __forceinline__ uint32_t at(int k) const {
    return mn ? k * 128 : (k & 3) * 2 + (k >> 2) * (R * 8);
  }
};
template <int R>
__device__ __forceinline__ Op<R> operand(const bf16* t, bool mn, int level_elems) {
  return {um::desc(um::saddr(t), mn ? R * 128 : 16, 1024) | ((uint64_t)2 << 61),
          (uint32_t)(level_elems * 2 / 16), mn};
}
template <int D>
__device__ __forceinline__ Op<kC> op_k(const bf16* t) { return operand<kC>(t, false, kC * D); }
template <int D>
__device__ __forceinline__ Op<kC> op_mn(const bf16* t) { return operand<kC>(t, true, kC * D); }
template <int D>
__device__ __forceinline__ Op<D> state_k(const bf16* t) { return operand<D>(t, false, D * D); }
template <int D>
__device__ __forceinline__ Op<D> state_mn(const bf16* t) { return operand<D>(t, true, D * D); }

// One warp issues the products, by a thread that it elects: warp-uniform control
// flow lets descriptors stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(r));
  return r != 0;
}
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}
__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc)
      : "memory");
}

// The products below take the level pairs (i, j) with i + j <= 2, the small
// ones first: the accumulators round towards zero at each step of 16, by what
// the sum has reached, so only the steps of the leading pair count.
constexpr int kMaxPair = 2;

// D (M x N) (+)= A B over K = 16 ks. One thread.
template <int NA, int NB, int M, int N, int KS, int RA, int RB>
__device__ __forceinline__ void product(uint32_t d, const Op<RA>& a, const Op<RB>& b, bool acc = false) {
  const uint32_t id = um::idesc64(a.mn, b.mn, M == 128, N);
#pragma unroll
  for (int o = kMaxPair; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = o - i;
      if (j < 0 || j >= NB) continue;
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        mma(d, a.d + a.at(k) + i * a.level, b.d + b.at(k) + j * b.level, id, acc);
        acc = true;
      }
    }
}
// A masked product in TMEM, 128 deep, as an operand. One level lies packed at the
// two ends of the accumulator it was made from, columns 0..31 and 96..127, so that
// each warp packs what it alone has read, with no word to the others, and the 64
// columns between are free; more levels lie one after the other, 64 columns each.
template <int NL>
__device__ __forceinline__ int packed_at(int col) {  // of product column `col`, a multiple of 16
  return col / 2 + (NL == 1 && col >= 64 ? 64 : 0);
}
// The same with A (128 rows, 128 deep) in TMEM, NA levels.
template <int NA, int NB, int N>
__device__ __forceinline__ void product_ta(uint32_t d, uint32_t a, const Op<kC>& b, bool acc) {
  const uint32_t id = um::idesc64(false, b.mn, true, N);
#pragma unroll
  for (int o = kMaxPair; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = o - i;
      if (j < 0 || j >= NB) continue;
#pragma unroll
      for (int k = 0; k < kC / 16; ++k) {
        mma_ta(d, a + packed_at<NA>(16 * k) + i * 64, b.d + b.at(k) + j * b.level, id, acc);
        acc = true;
      }
    }
}

__device__ __forceinline__ void st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void st8(uint32_t taddr, const uint32_t* r) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr),
               "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

// 16 fp32 values of this lane's row -> NL levels, two to a 32-bit TMEM column.
template <int NL>
__device__ __forceinline__ void st_levels16(uint32_t taddr, const float* x) {
  float a[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = x[i];
#pragma unroll
  for (int l = 0; l < NL; ++l) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(a[2 * i], a[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
      const float2 f = __bfloat1622float2(h);
      a[2 * i] -= f.x;
      a[2 * i + 1] -= f.y;
    }
    st8(taddr + 64 * l, w);
  }
}

// The blocks of 16 columns of a 128-wide product that fall to a part, W parts in all.
// One level, two parts: a half each, in an order in which a block packed in place
// (packed_at) lands on columns that the warp has read, from the outer end inwards;
// a loop, for the sake of the instruction cache, which a chunk's straight code
// would fill by itself. Otherwise blocks are held until they have been read.
template <int NL, int W>
__device__ __forceinline__ int block_of(int part, int k) {
  if (W == 4) return 64 * (part >> 1) + 32 * k + 16 * (part & 1);
  return NL == 1 && part == 1 ? 112 - 16 * k : 64 * part + 16 * k;
}
template <int NL, int W, class F>
__device__ __forceinline__ void masked_blocks(int part, F&& f) {
  if constexpr (NL == 1 && W == 2) {
#pragma unroll 1
    for (int k = 0; k < 4; ++k) f(k, block_of<NL, W>(part, k));
  } else {
#pragma unroll
    for (int k = 0; k < 8 / W; ++k) f(k, block_of<NL, W>(part, k));
  }
}

// The masked blocks of a lane's row, on their way to an operand's place.
template <int NL, int W>
struct Held {
  static constexpr bool kDirect = NL == 1 && W == 2;
  std::conditional_t<NL == 1, uint32_t, float> v[kDirect ? 1 : (NL == 1 ? 8 : 16) * (8 / W)];
  __device__ __forceinline__ void put(int k, int c0, uint32_t taddr, const float (&x)[16]) {
    if constexpr (kDirect) {
      st_levels16<1>(taddr + packed_at<1>(c0), x);
    } else if constexpr (NL == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        v[8 * k + i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[16 * k + i] = x[i];
    }
  }
  __device__ __forceinline__ void store(uint32_t taddr, int part) const {
    if constexpr (!kDirect) {
#pragma unroll
      for (int k = 0; k < 8 / W; ++k) {
        const uint32_t at = taddr + packed_at<NL>(block_of<NL, W>(part, k));
        if constexpr (NL == 1)
          st8(at, v + 8 * k);
        else
          st_levels16<NL>(at, v + 16 * k);
      }
    }
  }
};

// Four parts, one level: the two warps that share a lane quarter and a half of the
// columns have both read it (barriers 1..8).
__device__ __forceinline__ void half_read(int q, int part) {
  um::fence_before();
  named_bar(1 + q + 4 * (part >> 1), 64);
  um::fence_after();
}

// ------------------------------------------------------------------ state --

// The D x D fp32 state in registers, as the accumulator of a D-row product is
// read: M = 64 keeps row 16 q + lane in lanes 0-15 of quarter q, M = 128 row
// 32 q + lane; a part holds its share of the columns.
template <int D, int NT>
struct State {
  static constexpr int kCols = D * 128 / NT;
  float v[kCols];
  __device__ static int row() {
    const int q = (threadIdx.x >> 5) & 3, lane = threadIdx.x & 31;
    return D == 64 ? 16 * q + lane : 32 * q + lane;
  }
  __device__ static bool valid() { return D == 128 || (threadIdx.x & 31) < 16; }
  __device__ static int col0() { return (threadIdx.x >> 7) * kCols; }

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kCols; ++i) v[i] = 0.f;
  }
  // dk x dv entries of rows ld apart
  __device__ __forceinline__ void load(const float* p, int dk, int dv, int ld) {
    const int r = row(), c = col0();
#pragma unroll
    for (int i = 0; i < kCols; ++i)
      v[i] = valid() && r < dk && c + i < dv ? p[(long long)r * ld + c + i] : 0.f;
  }
  __device__ __forceinline__ void store(float* p, int dk, int dv, int ld) const {
    const int r = row(), c = col0();
    if (!valid() || r >= dk) return;
#pragma unroll
    for (int i = 0; i < kCols; ++i)
      if (c + i < dv) p[(long long)r * ld + c + i] = v[i];
  }
  // D x D in the order [column / 4][row][4]: whole lines to a warp's access
  __device__ __forceinline__ void load_own(const float* p) {
    if (!valid()) return zero();
#pragma unroll
    for (int i = 0; i < kCols; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(p + (((col0() + i) / 4) * D + row()) * 4);
      v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
  }
  __device__ __forceinline__ void store_own(float* p) const {
    if (!valid()) return;
#pragma unroll
    for (int i = 0; i < kCols; i += 4)
      *reinterpret_cast<float4*>(p + (((col0() + i) / 4) * D + row()) * 4) =
          make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  }
  // levels into D x D tiles
  template <int NL>
  __device__ __forceinline__ void to_smem(bf16* t) const {
    if (!valid()) return;
    const int r = row();
#pragma unroll
    for (int i = 0; i < kCols; i += 8)
      store_levels8<NL>(t, D * D, sw<D>(r, col0() + i), v + i);
  }
  // v = g v + accumulator at TMEM column `col` (every lane of the warp takes part)
  __device__ __forceinline__ void update(float g, uint32_t tb, int col) {
    const uint32_t a = tb + ((uint32_t)(32 * ((threadIdx.x >> 5) & 3)) << 16) + col + col0();
#pragma unroll
    for (int i = 0; i < kCols; i += 16) {
      float u[16];
      um::ld16(a + i, u);
#pragma unroll
      for (int k = 0; k < 16; ++k) v[i + k] = fmaf(g, v[i + k], u[k]);
    }
  }
};

// Rows of a tile (NL levels) times w(row), as three levels in dst[0..2].
template <int NL, int D, int NT, typename W>
__device__ __forceinline__ void scale_rows(const bf16* src, bf16* const (&dst)[3], W w) {
  using I = Items<D, NT>;
#pragma unroll
  for (int it = 0; it < I::kN; ++it) {
    const int o = I::offset(it);
    const float f = w(I::row(it));
    float x[8];
    load_levels8<NL>(src, kC * D, o, x);
    uint32_t lv[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      um::split3_pack(x[2 * i] * f, x[2 * i + 1] * f, lv[0][i], lv[1][i], lv[2][i]);
#pragma unroll
    for (int l = 0; l < 3; ++l)
      *reinterpret_cast<uint4*>(dst[l] + o) = make_uint4(lv[l][0], lv[l][1], lv[l][2], lv[l][3]);
  }
}

// Three-level product of scaled rows (dst[0..2], anywhere in shared memory)
// with a tile: D (D x D) (+)= sum_rows dst^T x.
template <int NL, int D>
__device__ __forceinline__ void product_rows(uint32_t d, bf16* const (&a)[3], const bf16* b, bool acc) {
  const uint32_t id = um::idesc64(true, true, D == 128, D);
  const Op<kC> o = op_mn<D>(b);
  const uint64_t da[3] = {op_mn<D>(a[0]).d, op_mn<D>(a[1]).d, op_mn<D>(a[2]).d};
#pragma unroll
  for (int r = kMaxPair; r >= 0; --r)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int j = r - i;
      if (j < 0 || j >= NL) continue;
#pragma unroll
      for (int k = 0; k < kC / 16; ++k) {
        mma(d, da[i] + o.at(k), o.d + o.at(k) + j * o.level, id, acc);
        acc = true;
      }
    }
}

struct Small {  // a CTA's barriers, TMEM address and decays
  uint64_t bar, bar2, full[3];
  uint32_t tbase;
  uint32_t pad;
  Decays dec;
};
constexpr int kSmallBytes = 2048;
static_assert(sizeof(Small) <= kSmallBytes, "");
constexpr int kDecayWarp = 4;  // builds the next chunk's table, during the products that no longer need this one's

// An mbarrier's phases are waited for by every thread; two of them in a row need
// a __syncthreads between the first wait and the second phase's arrival, or a
// thread that is late for the first never sees it.

// ----------------------------------------------------------- state kernel --

template <typename E, int D>
struct Sums {
  static constexpr int NL = kLevels<E>, kTileE = kC * D;
  // bf16: two buffers, the next chunk's tiles on their way during this one
  static constexpr int kBufs = NL == 1 ? 2 : 1;
  static constexpr size_t kSmem = kSmallBytes + 2 * (NL == 1 ? 6 : 3 + NL) * (size_t)kTileE;
  static constexpr int kPerSm = (int)(228 * 1024 / (kSmem + 1024)) < 3 ? (int)(228 * 1024 / (kSmem + 1024)) : 3;
  static constexpr int kThreads = kPerSm == 1 ? 512 : 256;
};

// What part s of a sequence (ms chunks) adds to the state: forward
// sum_j e^{c_end - c_j} k_j v_j^T, backward (kBwd) sum_i e^{c_i} q_i dy_i^T with
// c from the part's start. Every factor is <= 1, so the chunks just add up, in
// registers, without a chain through a state; the scaled rows take three levels since
// their sum is an fp32 state. Two CTAs to an SM (bf16 heads of 64), each with the next
// chunk on its way: 64 heads, T = 8192: 36 us (2.8 TB/s). One buffer and three CTAs
// to an SM: 35, but heads of 128 then 22 instead of 20.
template <typename E, int D, bool kBwd>
__global__ void __launch_bounds__(Sums<E, D>::kThreads, Sums<E, D>::kPerSm)
    state_kernel(const __grid_constant__ Args<E> p) {
  constexpr int NL = kLevels<E>, kTileE = kC * D, NT = Sums<E, D>::kThreads;
  extern __shared__ __align__(1024) unsigned char smem[];
  Small& sm = *reinterpret_cast<Small*>(smem);
  constexpr int kBufs = Sums<E, D>::kBufs;
  // one buffer: three levels of rows (NL on arrival) and the other tile; two: rows, the
  // other tiles, and the second and third levels
  bf16* const tiles = reinterpret_cast<bf16*>(smem + kSmallBytes);
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const long long bh = blockIdx.x % p.BH;
  const int s = (int)(blockIdx.x / p.BH) + (kBwd ? p.r : 0);
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const float* lg = p.lg + b * p.lsb + h * p.lsh;
  const int seg = s / p.r, c0 = seg * p.m + (s % p.r) * p.ms;
  const int c1 = min(min(c0 + p.ms, (seg + 1) * p.m), p.nchunks), count = c1 - c0;
  const int first = kBwd ? c0 : c1 - 1, step = kBwd ? 1 : -1;
  auto rows = [&](int c) { return (int)min((long long)kC, p.T - (long long)c * kC); };
  const bool tma = NL == 1 && p.tma;
  auto rows_tile = [&](int i) { return tiles + (kBufs == 2 ? (i & 1) : 0) * kTileE; };
  auto other_tile = [&](int i) { return tiles + (kBufs == 2 ? 2 + (i & 1) : 3) * kTileE; };
  auto load = [&](int i) {  // the part's i-th chunk, by one thread
    const long long t0 = (long long)(first + i * step) * kC;
    uint64_t* full = &sm.full[i & 1];
    mbar_arrive_expect_tx(full, 2 * tile_bytes(D));
    tma_load<D>(rows_tile(i), kBwd ? &p.mQ : &p.mK, t0, h, b, full);
    tma_load<D>(other_tile(i), kBwd ? &p.mdy : &p.mV, t0, h, b, full);
  };

  if (warp == 0) um::alloc(&sm.tbase, D);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_init(&sm.full[0], 1);
    mbar_init(&sm.full[1], 1);
    mbar_fence_init();
    if (tma && count > 0) load(0);
  }
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  State<D, NT> st;
  st.zero();
  DecayWarp dw;
  if (warp == kDecayWarp && count > 0) {
    dw.load(lg + (long long)first * kC * p.lst, p.lst, rows(first));
    dw.table<false>(sm.dec);
  }
  sync();
  Two run{0.f, 0.f};  // log2 decay of the chunks already summed
  for (int i = 0, c = first; i < count; ++i, c += step) {
    const bool more = i + 1 < count;
    bf16 *const A = rows_tile(i), *const Bt = other_tile(i);
    bf16* const lv[3] = {A, kBufs == 2 ? tiles + 4 * kTileE : A + kTileE,
                         kBufs == 2 ? tiles + 5 * kTileE : A + 2 * kTileE};
    if (tma) {
      if (ok && tid == 0 && more) load(i + 1);  // the products of i - 1 are done
      if (ok) ok = mbar_wait(&sm.full[i & 1], (i >> 1) & 1, &g_sticky_err, kPolls);
    } else {
      load_tile<E, D, NT>(A, kBwd ? p.Q : p.K, b, h, (long long)c * kC, rows(c), p.dk);
      load_tile<E, D, NT>(Bt, kBwd ? p.dy : p.V, b, h, (long long)c * kC, rows(c), p.dv);
    }
    if (warp == kDecayWarp && more) dw.load(lg + (long long)(c + step) * kC * p.lst, p.lst, rows(c + step));
    const float rh = run.s, rl = run.e, th = sm.dec.ch[kC - 1], tl = sm.dec.cl[kC - 1];
    scale_rows<NL, D, NT>(A, lv, [&](int r) {  // a thread's own items, in place
      const Decays& d = sm.dec;
      return kBwd ? ex2((d.ch[r] + rh) + (d.cl[r] + rl)) : ex2(((th - d.ch[r]) + rh) + ((tl - d.cl[r]) + rl));
    });
    run.add(th), run.add(tl);
    sync();
    if (warp == 0 && elect_one() && ok) {
      product_rows<NL, D>(sm.tbase, lv, Bt, false);
      um::commit(&sm.bar);
    }
    if (warp == kDecayWarp && more) dw.table<false>(sm.dec);
    if (ok) ok = mbar_wait(&sm.bar, i & 1, &g_sticky_err, kPolls);
    um::fence_after();
    st.update(1.f, sm.tbase, 0);  // in registers: round to nearest
    sync();                       // the next table; the sum has been read
  }
  // forward: the state that enters part s + 1; backward: the gradient that leaves s - 1
  if (ok) {
    st.store_own(p.seg + (bh * p.nsub + s + (kBwd ? -1 : 1)) * (D * D));
    if (tid == 0) p.segl[bh * p.nsub + s] = run.s + run.e;
  }
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, D);
}

// Joins the parts along the sequence: slot s + 1 = e^{L_s} slot s + what s
// added, from H0 (backward: slot s - 1 from slot s, from dH_T). One thread to
// four elements of one (batch, head), eight parts' loads under way together: with few
// heads it is their latency that counts (8 heads of 64, 37 parts: 6.8 us; 74: 10.8,
// with sixteen under way 15.7, or 13.7 at one element to a thread). Parts before the
// first segment's end (backward: after the last one's start) have nobody to add for.
template <int D, bool kBwd>
__global__ void __launch_bounds__(256) scan_kernel(float* seg, const float* segl, const float* init,
                                                   long long BH, int nsub, int steps, int dk, int dv,
                                                   long long sbh, int sld) {
  const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long bh = g / (D * D / 4);
  if (bh >= BH) return;
  const int e = (int)(g % (D * D / 4)), row = e % D, col = (e / D) * 4;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = init && row < dk && col + i < dv ? init[bh * sbh + row * sld + col + i] : 0.f;
  float4* sp = reinterpret_cast<float4*>(seg + bh * nsub * (long long)(D * D)) + e;
  const float* lp = segl + bh * nsub;
  constexpr int kN = 8;  // loads on their way together
  for (int i0 = 0; i0 < steps; i0 += kN) {
    float4 u[kN];
    float f[kN];
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int i = i0 + k, s = kBwd ? nsub - 1 - i : i, to = kBwd ? s - 1 : s + 1;
      if (i < steps) {
        f[k] = lp[s];
        u[k] = sp[(long long)to * (D * D / 4)];
      }
    }
#pragma unroll
    for (int k = 0; k < kN; ++k) {
      const int i = i0 + k, s = kBwd ? nsub - 1 - i : i, to = kBwd ? s - 1 : s + 1;
      if (i < steps) {
        const float e = ex2(f[k]);
        x[0] = fmaf(e, x[0], u[k].x), x[1] = fmaf(e, x[1], u[k].y);
        x[2] = fmaf(e, x[2], u[k].z), x[3] = fmaf(e, x[3], u[k].w);
        sp[(long long)to * (D * D / 4)] = make_float4(x[0], x[1], x[2], x[3]);
      }
    }
  }
}

// ---------------------------------------------------------------- forward --

// A segment, chunk by chunk: P = D * Q K^T in TMEM, y = P V + decayed Q S, then S for
// the next chunk, whose sum over the scaled K rows runs during P's masking and whose
// tiles load meanwhile. Bound by that chain, with two CTAs to an SM (bf16 heads of 64)
// to fill it; one level of P, and of S as an operand, where the output is 16 bits: each
// rounding is of the size of the output's (bf16 errors of 0.0023 for 0.0017), and a second
// level of either, 64 TMEM columns or 8 KB, would leave one CTA to an SM. 64 heads, T = 8192, bf16: 86 us, 3.1 TB/s, 8 heads, T = 65536: 70;
// heads of 128 (16, T = 4096): 43; fp32 (64 heads, T = 1024, 512 threads and one CTA
// to an SM): 52, where three levels make each product six. 512 threads at 64
// registers with two CTAs to an SM took 115.
//
// TMEM columns: Q K^T 0..127 (one level: P packed in its place), y 128.., the
// states' sum after it, P's levels after that.
template <typename E, int D>
struct Fwd {
  static constexpr int NL = kLevels<E>, kTileE = kC * D;
  static constexpr int kY = 128, kU = 128 + D, kP = NL == 1 ? 0 : kU + D;
  static constexpr int kCols = (NL == 1 ? kU + D : kP + 64 * NL) <= 256 ? 256 : 512;
  // bf16: two buffers for Q and K, the next chunk's on their way during this one
  static constexpr int kBufs = NL == 1 ? 2 : 1;
  static constexpr int kExtra = NL == 1 ? 1 : 0;  // third level of the scaled K rows
  static constexpr size_t kSmem =
      kSmallBytes + 2 * (((2 * kBufs + 1) * NL + kExtra) * (size_t)kTileE + NL * (size_t)D * D);
  static constexpr int kPerSm = 2 * (kSmem + 1024) <= 228 * 1024 && kCols <= 256 ? 2 : 1;
  static constexpr int kThreads = kPerSm == 1 ? 512 : 256;
  static_assert(kSmem <= 227 * 1024, "");
};

template <typename E, int D>
__global__ void __launch_bounds__(Fwd<E, D>::kThreads, Fwd<E, D>::kPerSm)
    fwd_kernel(const __grid_constant__ Args<E> p) {
  using F = Fwd<E, D>;
  constexpr int NL = F::NL, kTileE = F::kTileE, NT = F::kThreads, W = NT / 128;
  extern __shared__ __align__(1024) unsigned char smem[];
  Small& sm = *reinterpret_cast<Small*>(smem);
  bf16* const Q0 = reinterpret_cast<bf16*>(smem + kSmallBytes);
  bf16 *const K0 = Q0 + F::kBufs * NL * kTileE, *const V = K0 + F::kBufs * NL * kTileE,
              *const X = V + (NL + F::kExtra) * kTileE;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int q = warp & 3, wg = warp >> 2;
  const long long bh = blockIdx.x % p.BH;
  const int s = (int)(blockIdx.x / p.BH);
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const float* lg = p.lg + b * p.lsb + h * p.lsh;
  const int c0 = s * p.m, c1 = min(c0 + p.m, p.nchunks);
  auto rows = [&](int c) { return (int)min((long long)kC, p.T - (long long)c * kC); };
  const bool tma = NL == 1 && p.tma;
  auto load_v = [&](int c) {  // by one thread
    mbar_arrive_expect_tx(&sm.full[2], tile_bytes(D));
    tma_load<D>(V, &p.mV, (long long)c * kC, h, b, &sm.full[2]);
  };

  if (warp == 0) um::alloc(&sm.tbase, F::kCols);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_init(&sm.bar2, 1);
    for (int i = 0; i < 3; ++i) mbar_init(&sm.full[i], 1);
    mbar_fence_init();
    if (tma) {
      mbar_arrive_expect_tx(&sm.full[0], 2 * tile_bytes(D));
      tma_load<D>(Q0, &p.mQ, (long long)c0 * kC, h, b, &sm.full[0]);
      tma_load<D>(K0, &p.mK, (long long)c0 * kC, h, b, &sm.full[0]);
      load_v(c0);
    }
  }
  DecayWarp dw;
  if (warp == kDecayWarp) {
    dw.load(lg + (long long)c0 * kC * p.lst, p.lst, rows(c0));
    dw.table<false>(sm.dec);
  }
  State<D, NT> S;
  if (s > 0)
    S.load_own(p.seg + (bh * p.nsub + s * p.r) * (D * D));
  else if (p.H0)
    S.load(p.H0 + bh * p.sbh, p.dk, p.dv, p.sld);
  else
    S.zero();
  S.template to_smem<NL>(X);
  // After a wait that runs out (recorded in the sticky word) the CTA issues no
  // MMA or copy, waits on nothing and writes no output; sync makes the flag common. That
  // wait is over a second, by when the CTA's other copies have long arrived.
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  unsigned phase = 0;
  auto wait = [&]() {
    if (ok) ok = mbar_wait(&sm.bar, phase & 1, &g_sticky_err, kPolls);
    ++phase;
    um::fence_after();
  };
  if (tma) sync();  // the barriers
  const int row = 32 * q + lane;
  for (int c = c0; c < c1; ++c) {
    const int n = rows(c), i_ = c - c0, buf = tma ? i_ & 1 : 0;
    const long long t0 = (long long)c * kC;
    const bool more = c + 1 < c1;
    Decays& dec = sm.dec;
    bf16 *const Q = Q0 + buf * NL * kTileE, *const K = K0 + buf * NL * kTileE;
    bf16 *const Qn = Q0 + (buf ^ 1) * NL * kTileE, *const Kn = K0 + (buf ^ 1) * NL * kTileE;
    // the scaled K rows go over K and, below three levels, over Q (read by then) and the extra tile
    bf16* const lv[3] = {K, NL == 1 ? Q : K + kTileE, NL == 1 ? V + kTileE : NL == 2 ? Q : K + 2 * kTileE};
    if (tma) {
      if (ok) ok = mbar_wait(&sm.full[buf], (i_ >> 1) & 1, &g_sticky_err, kPolls);
    } else {
      load_tile<E, D, NT>(Q, p.Q, b, h, t0, n, p.dk);
      load_tile<E, D, NT>(K, p.K, b, h, t0, n, p.dk);
      load_tile<E, D, NT>(V, p.V, b, h, t0, n, p.dv);
    }
    sync();
    const uint32_t tb = sm.tbase;
    if (warp == 0 && elect_one() && ok) {
      product<NL, NL, 128, 128, D / 16>(tb, op_k<D>(Q), op_k<D>(K));
      product<NL, NL, 128, D, D / 16>(tb + F::kY, op_k<D>(Q), state_mn<D>(X));
      um::commit(&sm.bar);
    }
    if (tma && ok && tid == 0) {
      if (c > c0) tma_store<D>(&p.my, t0 - kC, h, b, p.dv, Qn);  // the last chunk's y
      if (more) {
        mbar_arrive_expect_tx(&sm.full[buf ^ 1], 2 * tile_bytes(D));
        tma_load<D>(Kn, &p.mK, t0 + kC, h, b, &sm.full[buf ^ 1]);
      }
    }
    if (warp == kDecayWarp && more) dw.load(lg + (t0 + kC) * p.lst, p.lst, rows(c + 1));
    if (p.saved) S.store_own(p.saved + (bh * p.nchunks + c) * (D * D));
    wait();
    const uint32_t lb = tb + ((uint32_t)(32 * q) << 16);
    const float rh = dec.ch[row], rl = dec.cl[row], th = dec.ch[kC - 1], tl = dec.cl[kC - 1];
    const bool add = more || s + 1 == p.nseg;  // a later chunk of this CTA, or H_T, needs S'
    if (add) {  // its products run while the masked product is read
      scale_rows<NL, D, NT>(K, lv, [&](int r) { return dec.to(th, tl, r); });
      sync();
      if (warp == 0 && elect_one() && ok) {
        if (tma) ok = mbar_wait(&sm.full[2], i_ & 1, &g_sticky_err, kPolls);
        if (ok) {
          product_rows<NL, D>(tb + F::kU, lv, V, false);
          um::commit(&sm.bar2);
        }
      }
    } else if (tma && ok && tid == 0) {
      ok = mbar_wait(&sm.full[2], i_ & 1, &g_sticky_err, kPolls);
    }
    {  // the state's part of y: diag(e^c) Q S
      const float f = ex2(rh + rl);
#pragma unroll
      for (int k = 0; k < D / (16 * W); ++k) {
        const uint32_t a = lb + F::kY + wg * (D / W) + 16 * k;
        float v[16];
        uint32_t w[16];
        um::ld16(a, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * f);
        st16(a, w);
      }
    }
    // P = D * Q K^T, a half of the columns to a warp
    Held<1, W> held;
    masked_blocks<NL, W>(wg, [&](int bk_, int j0) {
      float v[16];
      if (j0 > 32 * q + 31) {  // after every row of the warp
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
      } else {
        um::ld16(lb + j0, v);
        if (j0 + 15 < 32 * q) {  // before every row
          const float f = dec.to(rh, rl, j0 + 15);
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] *= f * dec.cf[j0 + i];
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float f = dec.to(rh, rl, j0 + i);
            v[i] = j0 + i <= row ? v[i] * f : 0.f;
          }
        }
      }
      if constexpr (NL == 1)
        held.put(bk_, j0, lb, v);
      else  // in columns of their own
        st_levels16<NL>(lb + F::kP + packed_at<NL>(j0), v);
    });
    if constexpr (NL == 1) {
      if constexpr (W == 4) half_read(q, wg);
      held.store(lb, wg);
    }
    if (tma && ok && tid == 0 && more) {
      bulk_wait_read();  // y has left
      tma_load<D>(Qn, &p.mQ, t0 + kC, h, b, &sm.full[buf ^ 1]);
    }
    st_wait();
    sync();
    if (warp == 0 && elect_one() && ok) {
      product_ta<NL, NL, D>(tb + F::kY, tb + F::kP, op_mn<D>(V), true);
      um::commit(&sm.bar);
    }
    if (warp == kDecayWarp && more) dw.table<false>(dec);
    if (add) {
      if (ok) ok = mbar_wait(&sm.bar2, i_ & 1, &g_sticky_err, kPolls);
      um::fence_after();
      S.update(ex2(th + tl), tb, F::kU);
      S.template to_smem<NL>(X);
    }
    wait();
    if (tma && ok && tid == 0 && more) load_v(c + 1);
#pragma unroll
    for (int k = 0; k < D / (16 * W); ++k) {
      const int j0 = wg * (D / W) + 16 * k;
      float v[16];
      um::ld16(lb + F::kY + j0, v);
      if (tma)
        row16_to_tile(Q, row, j0, v);
      else if (ok && row < n)
        store_row16<E>(p.y, b, h, p.H, t0 + row, p.T, j0, p.dv, v);
    }
    if (!tma) sync();  // the tiles are loaded over at once
  }
  if (tma) {
    sync();
    if (ok && tid == 0) {
      tma_store<D>(&p.my, (long long)(c1 - 1) * kC, h, b, p.dv, Q0 + ((c1 - 1 - c0) & 1) * NL * kTileE);
      bulk_wait_read();
    }
  }
  if (ok && s + 1 == p.nseg) S.store(p.HT + bh * p.sbh, p.dk, p.dv, p.sld);
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, F::kCols);
}

// --------------------------------------------------------------- backward --
//
// Two kernels. dQ and what it needs come from single chunks, with the states
// that the forward saved: dq_kernel takes chunks in any order. dK, dV and the
// states' gradient go through a segment's chunks from its end: dkv_kernel. Both
// form the masked products anew, each as its own rows want them.
//
// dlog_gamma is the sum of all that crosses token t. What has come through the state
// is added up as it is: q_i . dQ'_i for i >= t, k_j . dK'_j for j < t (prime: the state
// parts) and e^{c_C} <S, dS>. Pairs inside the chunk, X_t = sum_{i >= t > j} R_ij, go
// from row sums less column sums, X_t = X_{t+1} + sum_{j < t} R_tj - sum_{i > t} R_it,
// but only over the 16 tokens to the next edge of a quarter, where X is summed anew
// from the quarters' sums: dq_kernel's rows and dkv_kernel's columns round R
// differently, and with a decay of a few tokens X is no larger than what 100 tokens
// of that leave (2e-6 to 5e-6 of a head's summed gradient, now below 1e-6).

struct SmallB {
  uint64_t bar, bar2, full;
  uint32_t tbase, pad;
  float red[2][16];  // by warp
  float a[2][kC];    // a token's two sums
  Decays dec;
};
constexpr int kSmallB = 3 * 1024;
static_assert(sizeof(SmallB) <= kSmallB, "");
// In dkv_kernel the first rows have most masked blocks, so the last quarter's warps
// do the sundries: kSumWarp puts dlog_gamma together during the next chunk's first
// products.
constexpr int kSumWarp = 7, kDkvDecayWarp = 3;

// D = 64: 16 or 8 entries of one row of a state to each thread, all lanes busy.
template <int NT>
struct Even {
  static constexpr int D = 64, kN = D * D / NT;
  __device__ static int row() { return threadIdx.x & 63; }
  __device__ static int col() { return (threadIdx.x >> 6) * kN; }
  __device__ static void load_own(const float* src, float (&v)[kN]) {  // State's own order
#pragma unroll
    for (int i = 0; i < kN; i += 4) {
      const float4 f = *reinterpret_cast<const float4*>(src + (((col() + i) / 4) * D + row()) * 4);
      v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
    }
  }
  __device__ static void to_smem(bf16* t, const float (&v)[kN]) {
#pragma unroll
    for (int i = 0; i < kN; i += 8) store_levels8<3>(t, D * D, sw<D>(row(), col() + i), v + i);
  }
};

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// A token's two values, summed over the parts, to a[0] and a[1]; 32 tokens, the warps
// of all parts that share them, at a barrier of their own.
template <int W>
__device__ __forceinline__ void token_sums(float (&a)[2][kC], int q, int part, int row, float x, float y) {
  if constexpr (W == 4) {
    if (part >= 2) a[part - 2][row] = x;
    named_bar(9 + q, 128);
    if (part < 2) x += a[part][row];
    named_bar(9 + q, 128);
    if (part >= 2) a[part - 2][row] = y;
    named_bar(9 + q, 128);
    if (part < 2) y += a[part][row];
    named_bar(9 + q, 128);
  }
  if (part == 1) a[0][row] = x, a[1][row] = y;
  named_bar(9 + q, 32 * W);
  if (part == 0) a[0][row] += x, a[1][row] += y;
}

// 16 values, rounded to bf16 and packed, and back into a tile's row.
__device__ __forceinline__ void pack16(const float (&x)[16], uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const __nv_bfloat162 u = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&u);
  }
}
__device__ __forceinline__ void packed16_to_tile(bf16* tile, int r, int c0, const uint32_t* w) {
  *reinterpret_cast<uint4*>(tile + sw<kC>(r, c0)) = make_uint4(w[0], w[1], w[2], w[3]);
  *reinterpret_cast<uint4*>(tile + sw<kC>(r, c0 + 8)) = make_uint4(w[4], w[5], w[6], w[7]);
}

// dQ = A1 K + decayed dy S^T with A1 = D * dy V^T, and R's rows, from A1 and Q K^T.
// Chunks are independent, so that CTAs fill all SMs and take every so many; the next
// chunk's tiles load as each becomes free. Reads most of all kernels (four tiles and a
// state to a chunk) and comes nearest to DRAM's limit, 48%. 64 heads, T = 8192, bf16:
// 81 us (512 threads at 64 registers: 124); heads of 128 (16, T = 4096): 33; fp32 (64
// heads, T = 1024): 55.
//
// TMEM columns: (dy V^T) 0..127 and (Q K^T) 128..255. One level: the masked A1 in
// the former's place, and once both are read dQ and its state part in the latter's;
// more levels: A1 at 0, the others after it.
template <typename E, int D>
struct Dq {
  static constexpr int NL = kLevels<E>, kTileE = kC * D;
  static constexpr int kDq = NL == 1 ? 128 : 64 * NL, kIq = kDq + D, kCols = kIq + D <= 256 ? 256 : 512;
  static constexpr size_t kSmem = kSmallB + 2 * (4 * NL * (size_t)kTileE + 3 * (size_t)D * D);
  static constexpr int kPerSm = 2 * (kSmem + 1024) <= 228 * 1024 && kCols <= 256 ? 2 : 1;
  static constexpr int kThreads = kPerSm == 1 ? 512 : 256;
  static_assert(kSmem <= 227 * 1024, "");
};

template <typename E, int D>
__global__ void __launch_bounds__(Dq<E, D>::kThreads, Dq<E, D>::kPerSm)
    dq_kernel(const __grid_constant__ Args<E> p) {
  using F = Dq<E, D>;
  constexpr int NL = F::NL, kTileE = F::kTileE, NT = F::kThreads, W = NT / 128;
  extern __shared__ __align__(1024) unsigned char smem[];
  using Ev = Even<NT>;
  SmallB& sm = *reinterpret_cast<SmallB*>(smem);
  bf16* Q = reinterpret_cast<bf16*>(smem + kSmallB);
  bf16 *K = Q + NL * kTileE, *V = K + NL * kTileE, *G = V + NL * kTileE, *X = G + NL * kTileE;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int q = warp & 3, wg = warp >> 2;
  const int row = 32 * q + lane;
  const long long total = p.BH * p.nchunks;
  struct At {  // a chunk's place
    long long bh, t0;
    int b, h, c, n;
  };
  auto at = [&](long long id) {
    At a;
    a.bh = id % p.BH, a.c = (int)(id / p.BH);
    a.b = (int)(a.bh / p.H), a.h = (int)(a.bh % p.H);
    a.t0 = (long long)a.c * kC;
    a.n = (int)min((long long)kC, p.T - a.t0);
    return a;
  };
  const bool tma = NL == 1 && p.tma;
  Decays& dec = sm.dec;
  DecayWarp dw;
  auto load_decay = [&](const At& a) {
    dw.load(p.lg + a.b * p.lsb + a.h * p.lsh + a.t0 * p.lst, p.lst, a.n);
  };

  if (warp == 0) um::alloc(&sm.tbase, F::kCols);
  At a = at(blockIdx.x);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_init(&sm.full, 1);
    mbar_fence_init();
    if (tma) {
      mbar_arrive_expect_tx(&sm.full, 4 * tile_bytes(D));
      tma_load<D>(G, &p.mdy, a.t0, a.h, a.b, &sm.full);
      tma_load<D>(V, &p.mV, a.t0, a.h, a.b, &sm.full);
      tma_load<D>(Q, &p.mQ, a.t0, a.h, a.b, &sm.full);
      tma_load<D>(K, &p.mK, a.t0, a.h, a.b, &sm.full);
    }
  }
  if (warp == kDecayWarp) {
    load_decay(a);
    dw.table<false>(dec);
  }
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  unsigned phase = 0;
  auto wait = [&]() {
    if (ok) ok = mbar_wait(&sm.bar, phase & 1, &g_sticky_err, kPolls);
    ++phase;
    um::fence_after();
  };
  if (tma) sync();  // the barriers
  unsigned turn = 0;
  for (long long id = blockIdx.x; id < total; id += gridDim.x, turn ^= 1) {
    const bool more = id + gridDim.x < total;
    const At next = at(more ? id + gridDim.x : id);
    {  // the state that entered the chunk
      const float* src = p.saved + (a.bh * p.nchunks + a.c) * (D * D);
      if constexpr (D == 64) {
        float v[Ev::kN];
        Ev::load_own(src, v);
        Ev::to_smem(X, v);
      } else {
        State<D, NT> S;
        S.load_own(src);
        S.template to_smem<3>(X);
      }
    }
    if (tma) {
      if (ok) ok = mbar_wait(&sm.full, turn, &g_sticky_err, kPolls);
    } else {
      load_tile<E, D, NT>(Q, p.Q, a.b, a.h, a.t0, a.n, p.dk);
      load_tile<E, D, NT>(K, p.K, a.b, a.h, a.t0, a.n, p.dk);
      load_tile<E, D, NT>(V, p.V, a.b, a.h, a.t0, a.n, p.dv);
      load_tile<E, D, NT>(G, p.dy, a.b, a.h, a.t0, a.n, p.dv);
    }
    sync();
    const uint32_t tb = sm.tbase, lb = tb + ((uint32_t)(32 * q) << 16);
    if (warp == 0 && elect_one() && ok) {
      product<NL, NL, 128, 128, D / 16>(tb, op_k<D>(G), op_k<D>(V));
      product<NL, NL, 128, 128, D / 16>(tb + 128, op_k<D>(Q), op_k<D>(K));
      um::commit(&sm.bar);
    }
    if (tma && more && ok && tid == 0) {
      tma_prefetch<D>(&p.mdy, next.t0, next.h, next.b, p.dv);
      tma_prefetch<D>(&p.mV, next.t0, next.h, next.b, p.dv);
      tma_prefetch<D>(&p.mQ, next.t0, next.h, next.b, p.dk);
      tma_prefetch<D>(&p.mK, next.t0, next.h, next.b, p.dk);
    }
    if (tid < D * D / 32)  // the next state's lines
      asm volatile("prefetch.global.L2 [%0];" ::"l"(
          p.saved + (next.bh * p.nchunks + next.c) * (D * D) + tid * 32));
    if (warp == kDecayWarp && more) load_decay(next);
    wait();
    const float rh = dec.ch[row], rl = dec.cl[row], from_start = ex2(rh + rl);
    float tok = 0.f, left = 0.f, right = 0.f;  // R's row: in the diagonal quarter, in two quarters before it
    Held<NL, W> a1;
    // Lane: token i = row; columns: tokens j <= i. A1 = D * (dy V^T).
    masked_blocks<NL, W>(wg, [&](int bk_, int j0) {
      float x[16], z[16];
      if (j0 > 32 * q + 31) {  // after every row of the warp
#pragma unroll
        for (int i = 0; i < 16; ++i) z[i] = 0.f;
      } else {
        uint32_t r1[16], r2[16];
        um::ld16_async(lb + j0, r1);
        um::ld16_async(lb + 128 + j0, r2);
        um::ld_wait();
        um::ld_bind(r1, z);
        um::ld_bind(r2, x);
        if (j0 + 15 < 32 * q) {  // before every row
          const float f0 = dec.to(rh, rl, j0 + 15);
          float r = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            z[i] *= f0 * dec.cf[j0 + i];
            r = fmaf(z[i], x[i], r);
          }
          (j0 & 32 ? right : left) += r;
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float f = dec.to(rh, rl, j0 + i);
            const float zf = z[i] * f;
            tok += j0 + i < row ? zf * x[i] : 0.f;
            z[i] = j0 + i <= row ? zf : 0.f;
          }
        }
      }
      a1.put(bk_, j0, lb, z);
    });
    if constexpr (NL > 1)
      sync();  // both products have been read
    else if constexpr (W == 4)
      half_read(q, wg);
    a1.store(lb, wg);
    st_wait();
    sync();
    if (tma && ok && tid == 0 && more) {  // V has been used
      mbar_arrive_expect_tx(&sm.full, 4 * tile_bytes(D));
      tma_load<D>(V, &p.mV, next.t0, next.h, next.b, &sm.full);
    }
    if (warp == kDecayWarp && more) dw.table<false>(dec);
    if (warp == 0 && elect_one() && ok) {
      product_ta<NL, NL, D>(tb + F::kDq, tb, op_mn<D>(K), false);
      product<NL, 3, 128, D, D / 16>(tb + F::kIq, op_k<D>(G), state_k<D>(X));
      um::commit(&sm.bar);
    }
    wait();
    if (tma && ok && tid == 0 && more) {  // and so have dy and K
      tma_load<D>(G, &p.mdy, next.t0, next.h, next.b, &sm.full);
      tma_load<D>(K, &p.mK, next.t0, next.h, next.b, &sm.full);
    }
    float aq = 0.f;
#pragma unroll
    for (int k = 0; k < D / (16 * W); ++k) {
      const int j0 = wg * (D / W) + 16 * k;
      uint32_t r1[16], r2[16];
      float x[16], z[16], qr[16];
      um::ld16_async(lb + F::kDq + j0, r1);
      um::ld16_async(lb + F::kIq + j0, r2);
      load_levels8<NL>(Q, kTileE, sw<kC>(row, j0), qr);
      load_levels8<NL>(Q, kTileE, sw<kC>(row, j0 + 8), qr + 8);
      um::ld_wait();
      um::ld_bind(r1, x);
      um::ld_bind(r2, z);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        aq = fmaf(qr[i], z[i], aq);
        x[i] = fmaf(from_start, z[i], x[i]);
      }
      if (tma)
        row16_to_tile(Q, row, j0, x);  // over what this thread has read
      else if (ok && row < a.n)
        store_row16<E>(p.dQ, a.b, a.h, p.H, a.t0 + row, p.T, j0, p.dk, x);
    }
    aq *= from_start;
    token_sums<W>(sm.a, q, wg, row, tok + left + right, aq);
    left = warp_sum(left), right = warp_sum(right);
    if (lane == 0) sm.red[0][warp] = left, sm.red[1][warp] = right;
    sync();
    if (ok && tid < a.n) {
      p.rows_R[a.bh * p.T + a.t0 + tid] = sm.a[0][tid];
      p.state_q[a.bh * p.T + a.t0 + tid] = sm.a[1][tid];
    }
    if (ok && tid >= kC && tid < kC + 16) {  // rows' quarter i / 4, columns' quarter i % 4
      const int i = tid - kC, w = (i >> 2) + 4 * ((i >> 1) & 1) * (W / 2);
      float s = sm.red[i & 1][w];
      if (W == 4) s += sm.red[i & 1][w + 4];
      p.quarters[(a.bh * p.nchunks + a.c) * 16 + i] = s;
    }
    if (tma && ok && tid == 0) {
      tma_store<D>(&p.mdQ, a.t0, a.h, a.b, p.dk, Q);
      if (more) {
        bulk_wait_read();
        tma_load<D>(Q, &p.mQ, next.t0, next.h, next.b, &sm.full);
      }
    }
    a = next;
  }
  if (tma && tid == 0) bulk_wait_read();
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, F::kCols);
}

// A segment from its end: both masked products transposed, so that a thread has a key's
// row; dV = A2 dy + decayed K dS, dK = A1 Q + decayed V dS^T; then dS, in three levels
// as an operand, since dlog_gamma (fp32) is made from it. Its chain is the longest, four
// waits for products to a chunk, and bounds it: 64 heads, T = 8192, bf16: 168 us;
// heads of 128 (16, T = 4096): 84; fp32 (64 heads, T = 1024): 84. Outputs through
// staged tiles by TMA: stored from registers in 32-byte pieces 15 us more. 512 threads
// at 64 registers, two CTAs to an SM: a quarter more. The entering states, for
// dlog_gamma alone, take 8 us, loaded with the tiles (16 when loaded at their use).
//
// TMEM columns: (K Q^T) 0..127 and (V dy^T) 128..255. One level: their masked forms
// A2 and A1 in their places, dV and dK (D = 64) in the columns these leave free
// (D = 128: from 256 on); more levels: A2 at 0 and A1 at 64 NL once both are read, dV
// and dK after them. The state parts and the states' sum take the masked forms'
// places: for one level and D = 64 dK's state part the ends, 0..31 and 224..255.
template <typename E, int D>
struct Dkv {
  static constexpr int NL = kLevels<E>, kTileE = kC * D;
  // Two CTAs to an SM: dS is spread over all threads, and one tile more holds the
  // decayed K rows, so that dV's state part adds up in dV's own accumulator. One
  // level of these rows and two of dS: they end in dV's 16 bits alone.
  static constexpr bool kE = NL == 1 && D == 64;
  static constexpr int kA1 = NL == 1 ? 128 : 64 * NL;
  static constexpr int kDv = kE ? 32 : NL == 1 ? 256 : 128 * NL, kDk = kE ? 160 : kDv + D;
  static constexpr int kIk = D, kU = kE ? 96 : 0;
  static constexpr int kCols = kE ? 256 : 512;
  static_assert(kDk + D <= kCols && (kE || 2 * D <= kDv), "");
  static constexpr size_t kSmem =
      kSmallB + 2 * ((4 * NL + (kE ? 1 : 0)) * (size_t)kTileE + 3 * (size_t)D * D);
  static constexpr int kPerSm = 2 * (kSmem + 1024) <= 228 * 1024 && kCols <= 256 ? 2 : 1;
  static constexpr int kThreads = kPerSm == 1 ? 512 : 256;
  static_assert(kSmem <= 227 * 1024, "");
};

template <typename E, int D>
__global__ void __launch_bounds__(Dkv<E, D>::kThreads, Dkv<E, D>::kPerSm)
    dkv_kernel(const __grid_constant__ Args<E> p) {
  using F = Dkv<E, D>;
  constexpr int NL = F::NL, kTileE = F::kTileE, NT = F::kThreads, W = NT / 128;
  extern __shared__ __align__(1024) unsigned char smem[];
  using Ev = Even<NT>;
  SmallB& sm = *reinterpret_cast<SmallB*>(smem);
  bf16* Q = reinterpret_cast<bf16*>(smem + kSmallB);
  bf16 *K = Q + NL * kTileE, *V = K + NL * kTileE, *G = V + NL * kTileE, *X = G + NL * kTileE;
  bf16* Ex = X + 3 * D * D;
  // the scaled Q rows go over Q and, below three levels, over what has been read by then
  bf16* const lv[3] = {Q, F::kE ? V : NL == 1 ? K : Q + kTileE,
                       F::kE ? Ex : NL == 1 ? V : NL == 2 ? K : Q + 2 * kTileE};
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
  const int q = warp & 3, wg = warp >> 2;
  const long long bh = blockIdx.x % p.BH;
  const int s = p.nseg - 1 - (int)(blockIdx.x / p.BH);
  const int b = (int)(bh / p.H), h = (int)(bh % p.H);
  const float* lg = p.lg + b * p.lsb + h * p.lsh;
  const int c0 = s * p.m, c1 = min(c0 + p.m, p.nchunks);
  auto rows = [&](int c) { return (int)min((long long)kC, p.T - (long long)c * kC); };
  const bool tma = NL == 1 && p.tma;
  Decays& dec = sm.dec;

  if (warp == 0) um::alloc(&sm.tbase, F::kCols);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_init(&sm.bar2, 1);
    mbar_init(&sm.full, 1);
    mbar_fence_init();
    if (tma) {
      const long long t0 = (long long)(c1 - 1) * kC;
      mbar_arrive_expect_tx(&sm.full, 4 * tile_bytes(D));
      tma_load<D>(K, &p.mK, t0, h, b, &sm.full);
      tma_load<D>(Q, &p.mQ, t0, h, b, &sm.full);
      tma_load<D>(V, &p.mV, t0, h, b, &sm.full);
      tma_load<D>(G, &p.mdy, t0, h, b, &sm.full);
    }
  }
  DecayWarp dw;
  if (warp == kDkvDecayWarp) {
    dw.load(lg + (long long)(c1 - 1) * kC * p.lst, p.lst, rows(c1 - 1));
    dw.table<true>(dec);
  }
  float dSe[Ev::kN];  // kE
  State<D, NT> dS;    // otherwise
  {
    const float* end = s + 1 < p.nseg ? p.seg + (bh * p.nsub + (s + 1) * p.r - 1) * (D * D) : nullptr;
    if constexpr (F::kE) {
      const int er = Ev::row(), ec = Ev::col();
      if (end) {
        Ev::load_own(end, dSe);
      } else {
#pragma unroll
        for (int i = 0; i < Ev::kN; ++i)
          dSe[i] = p.dHT && er < p.dk && ec + i < p.dv ? p.dHT[bh * p.sbh + er * p.sld + ec + i] : 0.f;
      }
      Ev::to_smem(X, dSe);
    } else {
      if (end)
        dS.load_own(end);
      else if (p.dHT)
        dS.load(p.dHT + bh * p.sbh, p.dk, p.dv, p.sld);
      else
        dS.zero();
      dS.template to_smem<3>(X);
    }
  }
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  unsigned phase = 0;
  auto wait = [&]() {
    if (ok) ok = mbar_wait(&sm.bar, phase & 1, &g_sticky_err, kPolls);
    ++phase;
    um::fence_after();
  };
  sync();
  // <the state that enters chunk c, dS> by warps, as the chunk begins; dS has passed the
  // chunk's decay in dlog_gamma. The state loads with the tiles.
  using Entry = std::conditional_t<F::kE, float[Ev::kN], State<D, NT>>;
  auto entry_load = [&](int c, Entry& S) {
    const float* S_in = p.saved + (bh * p.nchunks + c) * (D * D);
    if constexpr (F::kE)
      Ev::load_own(S_in, S);
    else
      S.load_own(S_in);
  };
  auto through = [&](int c, const Entry& S) {
    float d = 0.f;
    if constexpr (F::kE) {
#pragma unroll
      for (int i = 0; i < Ev::kN; ++i) d = fmaf(S[i], dSe[i], d);
    } else {
#pragma unroll
      for (int i = 0; i < State<D, NT>::kCols; ++i) d = fmaf(S.v[i], dS.v[i], d);
    }
    d = warp_sum(d);
    if (lane == 0) sm.red[c & 1][warp] = d * ex2(dec.ch[kC - 1] + dec.cl[kC - 1]);
  };
  float rq[4], sq[4], lgs[4], edge = 0.f;
  // What chunk c's dlog_gamma needs from memory, and its sums once sm.a is complete:
  // four tokens to a lane, four lanes to an edge of a quarter.
  auto sums_load = [&](int c) {
    const long long t0 = (long long)c * kC;
    const int n = rows(c);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * lane + i;
      rq[i] = t < n ? p.rows_R[bh * p.T + t0 + t] : 0.f;
      sq[i] = t < n ? p.state_q[bh * p.T + t0 + t] : 0.f;
      lgs[i] = t < n ? lg[(t0 + t) * p.lst] : 0.f;
    }
    // this lane's edge is e quarters from the start: rows' quarters from e on, columns' before it
    const int e = (lane + 4) >> 3;
    const float4* x = reinterpret_cast<const float4*>(p.quarters + (bh * p.nchunks + c) * 16);
    edge = 0.f;
#pragma unroll
    for (int i = 1; i < 4; ++i) {
      const float4 f = x[i];
      if (i >= e) edge += (e > 0 ? f.x : 0.f) + (e > 1 ? f.y : 0.f) + (e > 2 ? f.z : 0.f);
    }
  };
  auto sums = [&](int c) {
    const long long t0 = (long long)c * kC;
    const int n = rows(c);
    const float4 a0 = *reinterpret_cast<const float4*>(sm.a[0] + 4 * lane);
    const float4 a1 = *reinterpret_cast<const float4*>(sm.a[1] + 4 * lane);
    const float *col = &a0.x, *bk = &a1.x;
    float past = 0.f;
    for (int i = 0; i < NT / 32; ++i) past += sm.red[c & 1][i];
    float x = 0.f, y = 0.f, z = 0.f;  // this lane's: rows less columns, q's and k's state parts
#pragma unroll
    for (int i = 0; i < 4; ++i) x += rq[i] - col[i], y += sq[i], z += bk[i];
    const bool after = lane & 4;  // the edge is after these tokens
    float nx = 0.f, iy = y, iz = z;
#pragma unroll
    for (int o = 1; o < 4; ++o) {  // lanes between this one and the edge
      const float u = __shfl_sync(0xffffffffu, x, after ? lane + o : lane - o);
      if (after ? (lane & 3) + o < 4 : (lane & 3) >= o) nx += u;
    }
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float u = __shfl_down_sync(0xffffffffu, iy, o), w = __shfl_up_sync(0xffffffffu, iz, o);
      if (lane + o < 32) iy += u;
      if (lane >= o) iz += w;
    }
    float in = after ? nx + x : -nx, sy = iy, sz = iz - z;  // at the lane's first token
    past += edge;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int t = 4 * lane + i;
      if (t < n && ok) {
        float* o = p.dlg + bh * p.T + t0 + t;
        float v = (in + past) + (sy + sz);
        if (p.dlg_add) v += *o;
        *o = lgs[i] * 1.4426950408889634f <= kMinLog2 ? 0.f : v;
      }
      in -= rq[i] - col[i], sy -= sq[i], sz += bk[i];
    }
  };
  const int row = 32 * q + lane;
  for (int c = c1 - 1; c >= c0; --c) {
    const long long t0 = (long long)c * kC;
    const int n = rows(c), turn = (c1 - 1 - c) & 1;
    const bool more = c > c0;
    Entry S_in;
    entry_load(c, S_in);
    if (tma) {
      if (ok) ok = mbar_wait(&sm.full, turn, &g_sticky_err, kPolls);
    } else {
      load_tile<E, D, NT>(K, p.K, b, h, t0, n, p.dk);
      load_tile<E, D, NT>(Q, p.Q, b, h, t0, n, p.dk);
      load_tile<E, D, NT>(V, p.V, b, h, t0, n, p.dv);
      load_tile<E, D, NT>(G, p.dy, b, h, t0, n, p.dv);
    }
    sync();
    const uint32_t tb = sm.tbase, lb = tb + ((uint32_t)(32 * q) << 16);
    if (warp == 0 && elect_one() && ok) {
      product<NL, NL, 128, 128, D / 16>(tb, op_k<D>(K), op_k<D>(Q));
      product<NL, NL, 128, 128, D / 16>(tb + 128, op_k<D>(V), op_k<D>(G));
      um::commit(&sm.bar);
    }
    if (tma && more && ok && tid == 0) {  // the next chunk's rows on their way into L2
      tma_prefetch<D>(&p.mK, t0 - kC, h, b, p.dk);
      tma_prefetch<D>(&p.mQ, t0 - kC, h, b, p.dk);
      tma_prefetch<D>(&p.mV, t0 - kC, h, b, p.dv);
      tma_prefetch<D>(&p.mdy, t0 - kC, h, b, p.dv);
    }
    if (!tma && more) {
      prefetch_rows(p.Q, b, h, t0 - kC, kC, p.dk);
      prefetch_rows(p.K, b, h, t0 - kC, kC, p.dk);
      prefetch_rows(p.V, b, h, t0 - kC, kC, p.dv);
      prefetch_rows(p.dy, b, h, t0 - kC, kC, p.dv);
    }
    if (warp == kDkvDecayWarp && more) dw.load(lg + (t0 - kC) * p.lst, p.lst, kC);
    if (warp == kSumWarp) {
      if (c + 1 < c1) sums(c + 1);
      sums_load(c);
    }
    through(c, S_in);  // while the products run
    if (more && tid < D * D / 32)  // the next state's lines
      asm volatile("prefetch.global.L2 [%0];" ::"l"(p.saved + (bh * p.nchunks + c - 1) * (D * D) + tid * 32));
    wait();
    const float rh = dec.ch[row], rl = dec.cl[row], th = dec.ch[kC - 1], tl = dec.cl[kC - 1];
    const float to_end = dec.to(th, tl, row);
    float tok = 0.f;  // this part's share of R's column `row`
    {
      // Lane: token j = row; columns: tokens i >= j. A2 = D * (K Q^T), A1 = D * (V dy^T).
      Held<NL, W> a1, a2;
      masked_blocks<NL, W>(wg, [&](int bk_, int i0) {
        float x[16], z[16];
        if (i0 + 15 < 32 * q) {  // before every row of the warp
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = z[i] = 0.f;
        } else {
          uint32_t r1[16], r2[16];
          um::ld16_async(lb + i0, r1);
          um::ld16_async(lb + 128 + i0, r2);
          um::ld_wait();
          um::ld_bind(r1, x);
          um::ld_bind(r2, z);
          if (i0 > 32 * q + 31) {  // after every row
            const float f0 = dec.from(rh, rl, i0);
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float f = f0 * dec.cf[i0 + i];
              x[i] *= f;
              tok = fmaf(x[i], z[i], tok);
              z[i] *= f;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float f = dec.from(rh, rl, i0 + i);
              const float pf = x[i] * f;
              tok += i0 + i > row ? pf * z[i] : 0.f;
              x[i] = i0 + i >= row ? pf : 0.f;
              z[i] = i0 + i >= row ? z[i] * f : 0.f;
            }
          }
        }
        a2.put(bk_, i0, lb, x);
        a1.put(bk_, i0, lb + F::kA1, z);
      });
      if constexpr (F::kE) {  // decayed K rows, one level: they end in dV alone
        using I = Items<D, NT>;
#pragma unroll
        for (int i = 0; i < I::kN; ++i) {
          float x[8];
          const float f = dec.to(th, tl, I::row(i));
          load_levels8<1>(K, 0, I::offset(i), x);
#pragma unroll
          for (int j = 0; j < 8; ++j) x[j] *= f;
          store_levels8<1>(Ex, 0, I::offset(i), x);
        }
      }
      if constexpr (NL > 1)
        sync();  // both products have been read
      else if constexpr (W == 4)
        half_read(q, wg);
      a2.store(lb, wg);
      a1.store(lb + F::kA1, wg);
      st_wait();
    }
    sync();
    if (warp == 0 && elect_one() && ok) {
      product_ta<NL, NL, D>(tb + F::kDv, tb, op_mn<D>(G), false);
      if (F::kE) product<1, 2, 128, D, D / 16>(tb + F::kDv, op_k<D>(Ex), state_mn<D>(X), true);
      product_ta<NL, NL, D>(tb + F::kDk, tb + F::kA1, op_mn<D>(Q), false);
      um::commit(&sm.bar);
    }
    wait();
    if (warp == 0 && elect_one() && ok) {
      if constexpr (F::kE) {  // in two halves of its columns: rows of dS
        product<NL, 3, 128, 32, D / 16>(tb, op_k<D>(V), state_k<D>(X));
        product<NL, 3, 128, 32, D / 16>(tb + 224, op_k<D>(V), state_k<D>(X + 32 * 64));
      } else {
        product<NL, 3, 128, D, D / 16>(tb, op_k<D>(K), state_mn<D>(X));
        product<NL, 3, 128, D, D / 16>(tb + F::kIk, op_k<D>(V), state_k<D>(X));
      }
      um::commit(&sm.bar2);
    }
    auto scale = [&]() { scale_rows<NL, D, NT>(Q, lv, [&](int r) { return ex2(dec.ch[r] + dec.cl[r]); }); };
    auto sum_states = [&]() {
      if (warp == 0 && elect_one() && ok) {
        product_rows<NL, D>(tb + F::kU, lv, G, false);
        um::commit(&sm.bar);
      }
      if (warp == kDkvDecayWarp && more) dw.table<true>(dec);  // the table has been used
    };
    if (ok) ok = mbar_wait(&sm.bar2, turn, &g_sticky_err, kPolls);
    um::fence_after();
    if (F::kE) {  // over Q, V and the extra tile; the gradients are read meanwhile
      scale();
      sync();
      sum_states();
    }
    float bk = 0.f;  // k . its gradient's state part
    uint32_t dvp[F::kE ? 8 * (D / (16 * W)) : 1];
#pragma unroll
    for (int k = 0; k < D / (16 * W); ++k) {
      const int j0 = wg * (D / W) + 16 * k;
      uint32_t r1[16], r2[16];
      float x[16], z[16];
      um::ld16_async(lb + F::kDv + j0, r1);
      if (!F::kE) um::ld16_async(lb + j0, r2);
      um::ld_wait();
      um::ld_bind(r1, x);
      if (!F::kE) {
        um::ld_bind(r2, z);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = fmaf(to_end, z[i], x[i]);
      }
      if (F::kE && tma)
        pack16(x, dvp + (F::kE ? 8 * k : 0));
      else if (ok && row < n)
        store_row16<E>(p.dV, b, h, p.H, t0 + row, p.T, j0, p.dv, x);
      um::ld16_async(lb + F::kDk + j0, r1);
      um::ld16_async(lb + (F::kE ? (j0 < 32 ? 0 : 192) : F::kIk) + j0, r2);
      float kr[16];
      load_levels8<NL>(K, kTileE, sw<kC>(row, j0), kr);
      load_levels8<NL>(K, kTileE, sw<kC>(row, j0 + 8), kr + 8);
      um::ld_wait();
      um::ld_bind(r1, x);
      um::ld_bind(r2, z);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        bk = fmaf(kr[i], z[i], bk);
        x[i] = fmaf(to_end, z[i], x[i]);
      }
      if (F::kE && tma)
        row16_to_tile(K, row, j0, x);  // over the row that this thread has read
      else if (ok && row < n)
        store_row16<E>(p.dK, b, h, p.H, t0 + row, p.T, j0, p.dk, x);
    }
    bk *= to_end;
    token_sums<W>(sm.a, q, wg, row, tok, bk);
    if (!F::kE) {  // over Q and what else has been read
      sync();
      scale();
      sync();
      sum_states();
    }
    wait();
    const float g = ex2(th + tl);
    if (F::kE && tma && ok && tid == 0 && more) {  // these two have been used
      mbar_arrive_expect_tx(&sm.full, 4 * tile_bytes(D));
      tma_load<D>(Q, &p.mQ, t0 - kC, h, b, &sm.full);
      tma_load<D>(G, &p.mdy, t0 - kC, h, b, &sm.full);
    }
    if constexpr (F::kE) {
      // the sum goes over the extra tile in its own order, then to all threads
      if (tma) {
#pragma unroll
        for (int k = 0; k < D / (16 * W); ++k) packed16_to_tile(V, row, wg * (D / W) + 16 * k, dvp + 8 * k);
      }
      State<D, NT> u;
      u.zero();
      u.update(0.f, tb, F::kU);
      u.store_own(reinterpret_cast<float*>(Ex));
      sync();
      if (tma && ok && tid == 0) {
        tma_store<D>(&p.mdV, t0, h, b, p.dv, V);
        tma_store<D>(&p.mdK, t0, h, b, p.dk, K);
        if (more) {
          bulk_wait_read();
          tma_load<D>(K, &p.mK, t0 - kC, h, b, &sm.full);
          tma_load<D>(V, &p.mV, t0 - kC, h, b, &sm.full);
        }
      }
      float v[Ev::kN];
      Ev::load_own(reinterpret_cast<const float*>(Ex), v);
#pragma unroll
      for (int i = 0; i < Ev::kN; ++i) dSe[i] = fmaf(g, dSe[i], v[i]);
      Ev::to_smem(X, dSe);
    } else {
      if (tma && ok && tid == 0 && more) {
        mbar_arrive_expect_tx(&sm.full, 4 * tile_bytes(D));
        tma_load<D>(K, &p.mK, t0 - kC, h, b, &sm.full);
        tma_load<D>(Q, &p.mQ, t0 - kC, h, b, &sm.full);
        tma_load<D>(V, &p.mV, t0 - kC, h, b, &sm.full);
        tma_load<D>(G, &p.mdy, t0 - kC, h, b, &sm.full);
      }
      dS.update(g, tb, F::kU);
      dS.template to_smem<3>(X);
      sync();
    }
  }
  sync();
  if (warp == kSumWarp) sums(c0);
  if (tma && tid == 0) bulk_wait_read();
  if (ok && s == 0 && p.dH0) {
    if constexpr (F::kE) {
      const int er = Ev::row(), ec = Ev::col();
#pragma unroll
      for (int i = 0; i < Ev::kN; ++i)
        if (er < p.dk && ec + i < p.dv) p.dH0[bh * p.sbh + er * p.sld + ec + i] = dSe[i];
    } else {
      dS.store(p.dH0 + bh * p.sbh, p.dk, p.dv, p.sld);
    }
  }
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, F::kCols);
}

// How the kernels above leave a wait that runs out, on a barrier that nothing arrives on.
__global__ void __launch_bounds__(256) stall_kernel(long long polls) {
  __shared__ Small sm;
  const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  if (warp == 0) um::alloc(&sm.tbase, 64);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_fence_init();
  }
  bool ok = true;
  auto sync = [&]() {
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  sync();
  if (tid < 32) ok = mbar_wait(&sm.bar, 0, &g_sticky_err, polls);
  sync();  // now for all threads: the second wait is not begun
  if (ok) ok = mbar_wait(&sm.bar, 0, &g_sticky_err, kPolls);
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, 64);
}

// ------------------------------------------------------------------- host --

struct Plan {
  int D, nchunks, m, nseg, ms, r, nsub;
};

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    n = 148;  // no device here: the sizes of a B200
  }
  return n;
}

// Segments of m chunks for the main kernel, each in r parts of ms chunks for the
// state sums. CTAs of a kernel take equally long, so its time goes by whole waves
// of them: the plan is the cheapest of one segment and of as many as fill 1 to 8
// waves, in units of a chunk of the state sums (2.6 us, bf16 heads of 64). In these
// a chunk of the forward is 2.1 to 4 and one of dkv_kernel 4 to 6.4, by type and
// width; a wave starts and ends in some 0.6 of a chunk; a part's state costs 0.04
// in scan_kernel, more with many heads; the two further launches are worth 2.
// Parts, state and scan together, bf16: 8 heads, T = 65536, 37 segments: r = 1 takes
// 47 us, 2 takes 53, 4 takes 68; 64 heads, T = 8192, 4 segments: r = 1 takes 44, 3
// takes 42, 6 takes 47. Segments, forward and backward, this rule against as many
// as fill one wave in parts for two: 104 heads, T = 4096 of 64: 361 us, 374; 16,
// T = 4096 of 128: 196, 209; 4, T = 256: 17 forward, 24. Heads that fill a wave by
// themselves are not split: a last wave of few CTAs is quicker than the model's
// (200 heads, T = 2048 of 128: forward 185 us, 214 in segments; 320 of 64: 136, 159).
Plan plan_for(long long BH, long long T, int D, bool fwd, int per_sm, int sums_per_sm) {
  Plan best{};
  best.D = D;
  const int n = (int)((T + kC - 1) / kC);
  best.nchunks = n;
  if (BH <= 0 || n <= 0) return best;
  const long long sms = sm_count(), places = sms * per_sm, sums_places = sms * sums_per_sm;
  const float main = fwd ? 2.5f : 5.f, slot = 0.04f + 0.001f * (float)BH;
  auto waves = [](long long ctas, long long at_once) { return (float)((ctas + at_once - 1) / at_once); };
  float least = 0.f;
  for (int w = 0; w <= (BH < places ? 8 : 0); ++w) {
    const long long fill = w == 0 ? 1 : w * places / BH;
    if (w > 0 && fill < 2) continue;
    Plan pl = best;
    pl.m = (int)(fill < n ? (n + fill - 1) / fill : 1);
    pl.nseg = (n + pl.m - 1) / pl.m;
    pl.ms = pl.m, pl.r = 1;
    float cost = main * waves(BH * pl.nseg, places) * (pl.m + 0.5f);
    if (pl.nseg > 1) {
      float sums = 0.f;
      for (int r = 1; r <= 4 && r <= pl.m; ++r) {
        const int ms = (pl.m + r - 1) / r, rr = (pl.m + ms - 1) / ms;
        const float c = waves(BH * (pl.nseg - 1) * rr, sums_places) * (ms + 0.6f) + slot * (float)(rr * pl.nseg);
        if (r == 1 || c < sums) sums = c, pl.ms = ms, pl.r = rr;
      }
      cost += sums + 2.f;
    }
    pl.nsub = pl.nseg * pl.r;
    if (w == 0 || cost < least) least = cost, best = pl;
    if (fill >= n) break;
  }
  return best;
}

// Element type and the width that kernels run at. bf16 heads up to 128 run
// whole; fp32 and fp16, whose operands take two or three times the room, in
// blocks of 64: the recurrence is linear in q and k (a sum over blocks of dk)
// and separate in the columns of v.
template <class F>
int by_shape(int dtype, int dk, int dv, F&& f) {
  const int d = dk > dv ? dk : dv;
  switch (dtype) {
    case MGS_BF16:
      return d <= 64    ? f(bf16{}, std::integral_constant<int, 64>{})
             : d <= 128 ? f(bf16{}, std::integral_constant<int, 128>{})
                        : (int)MGS_UNSUPPORTED;
    case MGS_F32: return f(float{}, std::integral_constant<int, 64>{});
    case MGS_F16: return f(__half{}, std::integral_constant<int, 64>{});
    default: return MGS_BAD_DTYPE;
  }
}

size_t seg_bytes(const Plan& pl, long long BH) {
  return pl.nseg > 1 ? (size_t)BH * pl.nsub * ((size_t)pl.D * pl.D + 1) * sizeof(float) : 0;
}

template <typename E, int D>
Plan plan_of(bool fwd, long long BH, long long T) {
  return plan_for(BH, T, D, fwd, fwd ? Fwd<E, D>::kPerSm : Dkv<E, D>::kPerSm, Sums<E, D>::kPerSm);
}

bool shape_ok(int64_t B, int H, int64_t T, int dk, int dv) {
  return B >= 0 && H >= 0 && T >= 0 && dk >= 1 && dv >= 1 && T < (1ll << 38) &&
         (B == 0 || H == 0 || B <= 0x7fffffffLL / H);
}

// Whether every row starts on `bytes` and holds whole groups of them (of 8
// elements at least).
template <typename P>
bool whole(P* p, const int64_t* s, int d, int bytes) {
  const long long e = bytes / (int)sizeof(P);
  return reinterpret_cast<uintptr_t>(p) % bytes == 0 && d % (e > 8 ? e : 8) == 0 && s[0] % e == 0 &&
         s[1] % e == 0 && s[2] % e == 0;
}
template <typename P>
Ten<P> ten(P* p, const int64_t* s, int d) {
  const bool vec = whole(p, s, d, 16);
  return {p, (long long)s[0], (long long)s[1], (long long)s[2], vec, vec && whole(p, s, d, 32), nullptr, 0};
}

// Tensor map over (columns, time, head, batch) with boxes of 64 columns x 128
// tokens; false where the tensor does not lie as a map can say: addresses and
// strides in whole 16 bytes, no stride of zero, extents of 32 bits.
template <typename P>
bool map_of(CUtensorMap* m, const Ten<P>& x, int d, long long T, long long H, long long B) {
  EncodeTiledFn fn = encode_tiled_fn();
  const long long s[3] = {x.st, x.sh, x.sb}, n[3] = {T, H, B};
  cuuint64_t dims[4] = {(cuuint64_t)d, (cuuint64_t)T, (cuuint64_t)H, (cuuint64_t)B}, strides[3];
  bool ok = fn != nullptr && reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && T < (1ll << 31);
  for (int i = 0; i < 3; ++i) {
    const long long bytes = s[i] * (long long)sizeof(P);
    ok = ok && (n[i] == 1 || (bytes > 0 && bytes % 16 == 0 && bytes < (1ll << 40)));
    strides[i] = n[i] == 1 ? 16 * (cuuint64_t)((d * sizeof(P) + 15) / 16) : (cuuint64_t)bytes;
  }
  if (!ok) return false;
  const cuuint32_t box[4] = {64u, (cuuint32_t)kC, 1u, 1u}, step[4] = {1u, 1u, 1u, 1u};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(static_cast<const void*>(x.p)), dims,
            strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename K>
int set_smem(K kern, size_t bytes) {
  MGS_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
  return MGS_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? MGS_OK : MGS_LAUNCH_FAILED; }

// The segment states, where there is more than one segment.
template <typename E, int D, bool kBwd>
int run_segments(const Args<E>& a, cudaStream_t st) {
  if (a.nseg <= 1) return MGS_OK;
  constexpr size_t smem = Sums<E, D>::kSmem;
  auto k1 = state_kernel<E, D, kBwd>;
  if (int r = set_smem(k1, smem)) return r;
  k1<<<(unsigned)(a.BH * (a.nseg - 1) * a.r), Sums<E, D>::kThreads, smem, st>>>(a);
  if (int r = launched()) return r;
  const long long n = a.BH * (D * D / 4);
  scan_kernel<D, kBwd><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
      a.seg, a.segl, kBwd ? a.dHT : a.H0, a.BH, a.nsub, (a.nseg - 1) * a.r, a.dk, a.dv, a.sbh,
      a.sld);
  return launched();
}

template <typename E, int D>
int run_main(bool fwd, const Args<E>& a, cudaStream_t st) {
  if (int r = fwd ? run_segments<E, D, false>(a, st) : run_segments<E, D, true>(a, st)) return r;
  if (!fwd) {  // any order of chunks: a CTA takes every so many
    using F = Dq<E, D>;
    if (int r = set_smem(dq_kernel<E, D>, F::kSmem)) return r;
    const long long n = a.BH * a.nchunks, places = (long long)sm_count() * F::kPerSm;
    dq_kernel<E, D><<<(unsigned)(n < places ? n : places), F::kThreads, F::kSmem, st>>>(a);
    if (int r = launched()) return r;
  }
  auto k = fwd ? fwd_kernel<E, D> : dkv_kernel<E, D>;
  const size_t smem = fwd ? Fwd<E, D>::kSmem : Dkv<E, D>::kSmem;
  if (int r = set_smem(k, smem)) return r;
  k<<<(unsigned)(a.BH * a.nseg), fwd ? Fwd<E, D>::kThreads : Dkv<E, D>::kThreads, smem, st>>>(a);
  return launched();
}

struct Blocks {  // of a head, in both dimensions
  int nk, nv;
  Blocks(int dk, int dv, int D) : nk((dk + D - 1) / D), nv((dv + D - 1) / D) {}
};

// fp32 rows for sums over blocks: dV's of one block of dv, dQ's and dK's of all.
size_t part_floats(const Blocks& n, bool fwd) {
  return fwd ? (n.nk > 1 ? 1 : 0) : (n.nk > 1 ? 1 : 0) + (n.nv > 1 ? 2 * (size_t)n.nk : 0);
}

size_t up256(size_t n) { return (n + 255) / 256 * 256; }
size_t sums_floats(const Plan& pl, long long BH, long long T) { return (size_t)BH * (2 * T + 16 * (size_t)pl.nchunks); }

template <typename E, int D>
size_t workspace_bytes_of(bool fwd, int64_t B, int H, int64_t T, int dk, int dv) {
  const long long BH = B * (long long)H;
  const Plan pl = plan_of<E, D>(fwd, BH, T);
  return up256(seg_bytes(pl, BH)) + (fwd ? 0 : up256(sums_floats(pl, BH, T) * sizeof(float))) +
         part_floats(Blocks(dk, dv, D), fwd) * (size_t)BH * T * 64 * sizeof(float);
}

// One call, over a head's blocks. What all blocks share is set in `a`.
template <typename E, int D>
int run_blocks(Args<E>& a, bool fwd, const float* lg, const int64_t* s, int64_t B, int H, int64_t T, int dk,
               int dv, void* ws, size_t ws_bytes, cudaStream_t st) {
  const long long BH = B * (long long)H;
  const Plan pl = plan_of<E, D>(fwd, BH, T);
  const size_t need = workspace_bytes_of<E, D>(fwd, B, H, T, dk, dv);
  if (need > ws_bytes) return MGS_WORKSPACE_TOO_SMALL;
  if ((need && !aligned(ws, 16)) || !aligned(a.saved, 16)) return MGS_BAD_ALIGNMENT;
  a.lg = lg, a.lsb = s[9], a.lsh = s[10], a.lst = s[11];
  a.seg = static_cast<float*>(ws);
  a.segl = a.seg + (size_t)BH * pl.nsub * D * D;
  a.T = T, a.H = H, a.nchunks = pl.nchunks, a.m = pl.m, a.nseg = pl.nseg, a.BH = BH;
  a.ms = pl.ms, a.r = pl.r, a.nsub = pl.nsub;
  a.sbh = (long long)dk * dv, a.sld = dv;
  const Blocks n(dk, dv, D);
  const size_t rows = (size_t)BH * T * 64;
  char* rest = static_cast<char*>(ws) + up256(seg_bytes(pl, BH));
  if (!fwd) {
    a.quarters = reinterpret_cast<float*>(rest);  // aligned
    a.rows_R = a.quarters + (size_t)BH * 16 * pl.nchunks, a.state_q = a.rows_R + (size_t)BH * T;
    rest += up256(sums_floats(pl, BH, T) * sizeof(float));
  }
  float* part = reinterpret_cast<float*>(rest);
  float *part_v = part, *part_q = part + (n.nk > 1 ? rows : 0), *part_k = part_q + n.nk * rows;
  const Args<E> whole = a;
  auto sum = [](auto& x, float* rows_, int i, int last) {  // x: a sum over blocks 0..last
    if (last == 0) return;
    x.part = rows_, x.mode = (i > 0 ? kAdd : 0) | (i < last ? kKeep : 0);
  };
  for (int j = 0; j < n.nv; ++j)
    for (int i = 0; i < n.nk; ++i) {
      const int k0 = i * D, v0 = j * D, bk = dk - k0 < D ? dk - k0 : D, bv = dv - v0 < D ? dv - v0 : D;
      const long long s0 = (long long)k0 * dv + v0;
      a = whole;
      a.dk = bk, a.dv = bv;
      a.Q = ten(whole.Q.p + k0, s, bk), a.K = ten(whole.K.p + k0, s + 3, bk), a.V = ten(whole.V.p + v0, s + 6, bv);
      if (fwd) {
        a.y = ten(whole.y.p + v0, s + 12, bv);
        sum(a.y, part_v, i, n.nk - 1);
        a.HT = whole.HT + s0;
        if (whole.H0) a.H0 = whole.H0 + s0;
      } else {
        a.dy = ten(whole.dy.p + v0, s + 12, bv);
        a.dQ = ten(whole.dQ.p + k0, s + 15, bk), a.dK = ten(whole.dK.p + k0, s + 18, bk);
        a.dV = ten(whole.dV.p + v0, s + 21, bv);
        sum(a.dV, part_v, i, n.nk - 1);
        sum(a.dQ, part_q + i * rows, j, n.nv - 1);
        sum(a.dK, part_k + i * rows, j, n.nv - 1);
        if (whole.dHT) a.dHT = whole.dHT + s0;
        if (whole.dH0) a.dH0 = whole.dH0 + s0;
        a.dlg_add = i + j > 0;
      }
      if (whole.saved) a.saved = whole.saved + (size_t)(j * n.nk + i) * BH * pl.nchunks * D * D;
      if constexpr (std::is_same_v<E, bf16>) {
        bool ok = map_of(&a.mQ, a.Q, dk, T, H, B) && map_of(&a.mK, a.K, dk, T, H, B) &&
                  map_of(&a.mV, a.V, dv, T, H, B);
        if (fwd)
          ok = ok && map_of(&a.my, a.y, dv, T, H, B);
        else
          ok = ok && map_of(&a.mdy, a.dy, dv, T, H, B) && map_of(&a.mdQ, a.dQ, dk, T, H, B) &&
               map_of(&a.mdK, a.dK, dk, T, H, B) && map_of(&a.mdV, a.dV, dv, T, H, B);
        a.tma = ok;
      }
      if (int r = run_main<E, D>(fwd, a, st)) return r;
    }
  return MGS_OK;
}

}  // namespace
}  // namespace lattn

unsigned take_error_linear_attn(cudaStream_t s) { return take_sticky_error(s); }

}  // namespace mgs

extern "C" {

size_t mgs_linear_attn_workspace_size(int64_t B, int H, int64_t T, int dk, int dv, int dtype) {
  using namespace mgs::lattn;
  if (!shape_ok(B, H, T, dk, dv)) return 0;
  size_t n = 0;
  (void)by_shape(dtype, dk, dv, [&](auto e, auto d) -> int {
    using E = decltype(e);
    constexpr int D = decltype(d)::value;
    const size_t f = workspace_bytes_of<E, D>(true, B, H, T, dk, dv);
    const size_t b = workspace_bytes_of<E, D>(false, B, H, T, dk, dv);
    n = f > b ? f : b;
    return MGS_OK;
  });
  return n;
}

size_t mgs_linear_attn_saved_size(int64_t B, int H, int64_t T, int dk, int dv, int dtype) {
  using namespace mgs::lattn;
  if (!shape_ok(B, H, T, dk, dv)) return 0;
  size_t n = 0;
  (void)by_shape(dtype, dk, dv, [&](auto, auto d) -> int {
    constexpr int D = decltype(d)::value;
    const Blocks blocks(dk, dv, D);
    n = (size_t)blocks.nk * blocks.nv * (size_t)(B * H) * (size_t)((T + kC - 1) / kC) * D * D * sizeof(float);
    return MGS_OK;
  });
  return n;
}

int mgs_test_linear_attn_timeout(int64_t spin_limit, void* stream) {
  if (spin_limit < 1) return MGS_BAD_SHAPE;
  mgs::lattn::stall_kernel<<<1, 256, 0, static_cast<cudaStream_t>(stream)>>>(spin_limit);
  return mgs::lattn::launched();
}

int mgs_linear_attn_fwd(const void* Q, const void* K, const void* V, const float* log_gamma,
                        const float* H0, void* y, float* H_T, float* saved, const int64_t* strides,
                        int64_t B, int H, int64_t T, int dk, int dv, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
  using namespace mgs::lattn;
  if (!shape_ok(B, H, T, dk, dv)) return MGS_BAD_SHAPE;
  return by_shape(dtype, dk, dv, [&](auto e, auto d) -> int {
    using E = decltype(e);
    if (B == 0 || H == 0 || T == 0) return MGS_OK;
    Args<E> a{};
    a.Q.p = static_cast<const E*>(Q), a.K.p = static_cast<const E*>(K), a.V.p = static_cast<const E*>(V);
    a.y.p = static_cast<E*>(y), a.H0 = H0, a.HT = H_T, a.saved = saved;
    return run_blocks<E, decltype(d)::value>(a, true, log_gamma, strides, B, H, T, dk, dv, workspace,
                                             workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}

int mgs_linear_attn_bwd(const void* Q, const void* K, const void* V, const float* log_gamma,
                        const float* saved, const void* dy, const float* dH_T, void* dQ, void* dK,
                        void* dV, float* dlog_gamma, float* dH0, const int64_t* strides, int64_t B,
                        int H, int64_t T, int dk, int dv, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
  using namespace mgs::lattn;
  if (!shape_ok(B, H, T, dk, dv)) return MGS_BAD_SHAPE;
  return by_shape(dtype, dk, dv, [&](auto e, auto d) -> int {
    using E = decltype(e);
    if (B == 0 || H == 0 || T == 0) return MGS_OK;
    Args<E> a{};
    a.Q.p = static_cast<const E*>(Q), a.K.p = static_cast<const E*>(K), a.V.p = static_cast<const E*>(V);
    a.dy.p = static_cast<const E*>(dy);
    a.dQ.p = static_cast<E*>(dQ), a.dK.p = static_cast<E*>(dK), a.dV.p = static_cast<E*>(dV);
    a.saved = const_cast<float*>(saved), a.dHT = dH_T, a.dH0 = dH0, a.dlg = dlog_gamma;
    return run_blocks<E, decltype(d)::value>(a, false, log_gamma, strides, B, H, T, dk, dv, workspace,
                                             workspace_bytes, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
