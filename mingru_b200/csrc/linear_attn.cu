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
// Decays. The sums are formed in base 2 and fp64 and kept as ch + cl, ch a
// multiple of 2^-9 (exact differences in fp32) and cl the small rest, so that
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
#include "common.cuh"
#include "umma.cuh"

namespace mgs {
namespace lattn {
namespace {

using bf16 = __nv_bfloat16;
namespace um = umma;

constexpr int kC = 128;        // tokens of a chunk: the rows of an M = 128 accumulator
constexpr int kThreads = 256;  // two warps for each quarter of the TMEM lanes
constexpr float kMinLog2 = -128.f;

template <typename E>
constexpr int kLevels = 1;
template <>
constexpr int kLevels<__half> = 2;
template <>
constexpr int kLevels<float> = 3;

// A (B, H, T, d) tensor: base and strides in elements (the last dimension is
// dense); vec: every row starts on 16 bytes and holds whole groups of 8.
template <typename P>
struct Ten {
  P* p;
  long long sb, sh, st;
  int vec;
};

template <typename E>
struct Args {
  Ten<const E> Q, K, V, dy;
  Ten<E> y, dQ, dK, dV;
  const float* lg;
  long long lsb, lsh, lst;
  const float* H0;   // (B, H, dk, dv) or null: zeros
  float* HT;         // forward: (B, H, dk, dv)
  const float* dHT;  // (B, H, dk, dv) or null: zeros
  float* dH0;        // (B, H, dk, dv) or null: not wanted
  float* dlg;        // (B, H, T)
  float* saved;      // (BH, nchunks, D * D) chunk-start states, or null (forward without a backward)
  float* seg;        // (BH, nseg, D * D) segment states (workspace)
  float* segl;       // (BH, nseg) log2 of each segment's total decay (workspace)
  long long T;
  int H, dk, dv, nchunks, m, nseg;  // m chunks to a segment
  long long BH;
};

// ------------------------------------------------------------- tile loads --

__device__ __forceinline__ void cp_async16(void* dst, const void* src, int src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src),
               "r"(src_bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() {
  asm volatile("cp.async.commit_group;\ncp.async.wait_group 0;\n" ::: "memory");
}

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

// Row and first column of item `idx` (8 elements) of a blocked 128 x D tile;
// the item's element offset is 8 * idx. A warp's items are 8 rows x 4 groups:
// whole 32-byte sectors of global memory, and a conflict-free 512-byte run of
// shared memory.
template <int D>
__device__ __forceinline__ void item_rc(int idx, int& r, int& c) {
  r = (idx / D) * 8 + (idx & 7);
  c = ((idx >> 3) & (D / 8 - 1)) * 8;
}

// Rows [t0, t0 + n) of one head as NL bf16 levels in blocked tiles; rows from
// n and columns from d are zeros. bf16 rows that allow it go by cp.async (the
// caller waits), others through registers.
template <typename E, int D>
__device__ __forceinline__ void load_tile(bf16* tile, const Ten<const E>& x, const E* head, long long t0,
                                          int n, int d) {
  constexpr int NL = kLevels<E>, kItems = kC * D / 8 / kThreads;
  const E* base = head + t0 * x.st;
  if constexpr (NL == 1) {
    if (x.vec) {
#pragma unroll
      for (int it = 0; it < kItems; ++it) {
        const int idx = it * kThreads + (int)threadIdx.x;
        int r, c;
        item_rc<D>(idx, r, c);
        const bool in = r < n && c < d;
        cp_async16(tile + 8 * idx, in ? base + r * x.st + c : head, in ? 16 : 0);
      }
      return;
    }
  }
#pragma unroll
  for (int it = 0; it < kItems; ++it) {
    const int idx = it * kThreads + (int)threadIdx.x;
    int r, c;
    item_rc<D>(idx, r, c);
    float v[8];
    const E* s = base + r * x.st + c;
    if (x.vec) {
      if (r < n && c < d) {
        constexpr int kN = 16 / (int)sizeof(E);
#pragma unroll
        for (int k = 0; k < 8; k += kN) {
          const uint4 u = __ldg(reinterpret_cast<const uint4*>(s + k));
          const E* e = reinterpret_cast<const E*>(&u);
#pragma unroll
          for (int i = 0; i < kN; ++i) v[k + i] = to_f32<E>(e[i]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.f;
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = r < n && c + i < d ? to_f32<E>(s[i]) : 0.f;
    }
    store_levels8<NL>(tile, kC * D, 8 * idx, v);
  }
}

// 16 values of one row (columns c0..) to global memory.
template <typename E>
__device__ __forceinline__ void store_row16(E* row, int c0, int d, bool vec, const float (&v)[16]) {
  if (vec) {
    constexpr int kN = 16 / (int)sizeof(E);
#pragma unroll
    for (int k = 0; k < 16; k += kN)
      if (c0 + k < d) {
        uint4 u;
        E* e = reinterpret_cast<E*>(&u);
#pragma unroll
        for (int i = 0; i < kN; ++i) e[i] = from_f32<E>(v[k + i]);
        *reinterpret_cast<uint4*>(row + c0 + k) = u;
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

// Inclusive sums of a chunk's log2 decays as ch + cl, by one warp (four tokens
// to a lane, fp64). Tokens from n on add nothing.
__device__ __forceinline__ void decay_table(const float* lg, long long st, int n, float* ch, float* cl) {
  const int lane = threadIdx.x & 31;
  double s[4];
  double run = 0.0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 4 * lane + i;
    double v = 0.0;
    if (t < n) {
      v = (double)lg[t * st] * 1.4426950408889634;
      if (v < (double)kMinLog2) v = (double)kMinLog2;
    }
    run += v;
    s[i] = run;
  }
  double inc = run;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const double o = __shfl_up_sync(0xffffffffu, inc, d);
    if (lane >= d) inc += o;
  }
  const double before = inc - run;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const double c = before + s[i];
    const float h = rintf((float)c * 512.f) * (1.f / 512.f);
    ch[4 * lane + i] = h;
    cl[4 * lane + i] = (float)(c - (double)h);
  }
}

// ------------------------------------------------------------ MMA issuing --

// Descriptor of a blocked tile of `cols` columns: contraction over its columns
// (K-major) or over its rows (MN-major), and the step of 16 along it.
struct Op {
  uint64_t d;
  uint32_t step, level;  // in 16-byte units
  bool mn;
};
__device__ __forceinline__ Op op_k(const bf16* t, int cols, int level_elems) {
  return {um::desc(um::saddr(t), 128, cols * 16), 256 / 16, (uint32_t)(level_elems * 2 / 16), false};
}
__device__ __forceinline__ Op op_mn(const bf16* t, int cols, int level_elems) {
  return {um::desc(um::saddr(t), cols * 16, 128), (uint32_t)(2 * cols * 16 / 16),
          (uint32_t)(level_elems * 2 / 16), true};
}

__device__ __forceinline__ void mma_ta(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool acc) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n}\n" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)acc), "r"(0), "r"(0), "r"(0), "r"(0)
      : "memory");
}

// The products below take the level pairs (i, j) with i + j <= 2, the small
// ones first: the accumulators round towards zero at each step of 16, by what
// the sum has reached, so only the steps of the leading pair count.
constexpr int kMaxPair = 2;

// D (M x N) (+)= A B over K = 16 ks. One thread.
template <int NA, int NB, int M, int N>
__device__ __forceinline__ void product(uint32_t d, const Op& a, const Op& b, int ks, bool acc = false) {
  const uint32_t id = um::idesc64(a.mn, b.mn, M == 128, N);
#pragma unroll
  for (int o = kMaxPair; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = o - i;
      if (j < 0 || j >= NB) continue;
#pragma unroll 4
      for (int k = 0; k < ks; ++k) {
        um::mma(d, a.d + k * a.step + i * a.level, b.d + k * b.step + j * b.level, id, acc);
        acc = true;
      }
    }
}
// The same with A (128 rows, 128 deep) in TMEM: NA levels of 64 columns each.
template <int NA, int NB, int N>
__device__ __forceinline__ void product_ta(uint32_t d, uint32_t a, const Op& b, bool acc) {
  const uint32_t id = um::idesc64(false, b.mn, true, N);
#pragma unroll
  for (int o = kMaxPair; o >= 0; --o)
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int j = o - i;
      if (j < 0 || j >= NB) continue;
#pragma unroll 4
      for (int k = 0; k < kC / 16; ++k) {
        mma_ta(d, a + k * 8 + i * 64, b.d + k * b.step + j * b.level, id, acc);
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

// ------------------------------------------------------------------ state --

// The D x D fp32 state in registers, as the accumulator of a D-row product is
// read: M = 64 keeps row 16 q + lane in lanes 0-15 of quarter q, M = 128 row
// 32 q + lane; warps 0-3 hold the left half of the columns, 4-7 the right.
template <int D>
struct State {
  static constexpr int kCols = D / 2;
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
  // (dk, dv) row-major
  __device__ __forceinline__ void load(const float* p, int dk, int dv) {
    const int r = row(), c = col0();
#pragma unroll
    for (int i = 0; i < kCols; ++i)
      v[i] = valid() && r < dk && c + i < dv ? p[(long long)r * dv + c + i] : 0.f;
  }
  __device__ __forceinline__ void store(float* p, int dk, int dv) const {
    const int r = row(), c = col0();
    if (!valid() || r >= dk) return;
#pragma unroll
    for (int i = 0; i < kCols; ++i)
      if (c + i < dv) p[(long long)r * dv + c + i] = v[i];
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
  // levels into blocked D x D tiles
  template <int NL>
  __device__ __forceinline__ void to_smem(bf16* t) const {
    if (!valid()) return;
    const int r = row();
#pragma unroll
    for (int i = 0; i < kCols; i += 8)
      store_levels8<NL>(t, D * D, um::boff_n(r, col0() + i, D), v + i);
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
template <int NL, int D, typename W>
__device__ __forceinline__ void scale_rows(const bf16* src, bf16* const (&dst)[3], W w) {
#pragma unroll
  for (int it = 0; it < kC * D / 8 / kThreads; ++it) {
    const int idx = it * kThreads + (int)threadIdx.x;
    int r, c;
    item_rc<D>(idx, r, c);
    float x[8], f = w(r);
    load_levels8<NL>(src, kC * D, 8 * idx, x);
    uint32_t lv[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      um::split3_pack(x[2 * i] * f, x[2 * i + 1] * f, lv[0][i], lv[1][i], lv[2][i]);
#pragma unroll
    for (int l = 0; l < 3; ++l)
      *reinterpret_cast<uint4*>(dst[l] + 8 * idx) = make_uint4(lv[l][0], lv[l][1], lv[l][2], lv[l][3]);
  }
}

// Three-level product of scaled rows (dst[0..2], anywhere in shared memory)
// with a tile: D (D x D) (+)= sum_rows dst^T x.
template <int NL, int D>
__device__ __forceinline__ void product_rows(uint32_t d, bf16* const (&a)[3], const bf16* b, bool acc) {
  const uint32_t id = um::idesc64(true, true, D == 128, D);
  const Op o = op_mn(b, D, kC * D);
  const uint64_t da[3] = {op_mn(a[0], D, 0).d, op_mn(a[1], D, 0).d, op_mn(a[2], D, 0).d};
#pragma unroll
  for (int r = kMaxPair; r >= 0; --r)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const int j = r - i;
      if (j < 0 || j >= NL) continue;
#pragma unroll 4
      for (int k = 0; k < kC / 16; ++k) {
        um::mma(d, da[i] + k * o.step, o.d + k * o.step + j * o.level, id, acc);
        acc = true;
      }
    }
}

struct Small {  // the tables of a CTA
  uint64_t bar;
  uint32_t tbase;
  uint32_t pad;
  float ch[kC], cl[kC];
};
constexpr int kSmallBytes = 2048;
static_assert(sizeof(Small) <= kSmallBytes, "");

// ----------------------------------------------------------- state kernel --

// What segment s adds to the state: forward sum_j e^{c_end - c_j} k_j v_j^T,
// backward (kBwd) sum_i e^{c_i} q_i dy_i^T with c from the segment's start.
// Every factor is <= 1, so the chunks of a segment just add up.
template <typename E, int D, bool kBwd>
__global__ void __launch_bounds__(kThreads) state_kernel(const Args<E> p) {
  constexpr int NL = kLevels<E>, kTileE = kC * D;
  extern __shared__ __align__(1024) unsigned char smem[];
  Small& sm = *reinterpret_cast<Small*>(smem);
  bf16* A = reinterpret_cast<bf16*>(smem + kSmallBytes);  // three levels (NL on arrival)
  bf16* Bt = A + 3 * kTileE;
  const int tid = threadIdx.x, warp = tid >> 5;
  const long long bh = blockIdx.x % p.BH;
  const int s = (int)(blockIdx.x / p.BH) + (kBwd ? 1 : 0);
  const long long b = bh / p.H, h = bh % p.H;
  const Ten<const E>&ta = kBwd ? p.Q : p.K, &tv = kBwd ? p.dy : p.V;
  const E* ha = ta.p + b * ta.sb + h * ta.sh;
  const E* hv = tv.p + b * tv.sb + h * tv.sh;
  const float* lg = p.lg + b * p.lsb + h * p.lsh;
  bf16* const lv[3] = {A, A + kTileE, A + 2 * kTileE};

  if (warp == 0) um::alloc(&sm.tbase, D);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_fence_init();
  }
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  const int c0 = s * p.m, c1 = min(c0 + p.m, p.nchunks);
  State<D> st;
  st.zero();
  double run = 0.0;  // log2 decay of the chunks already summed
  unsigned phase = 0;
  for (int i = 0; i < c1 - c0; ++i) {
    const int c = kBwd ? c0 + i : c1 - 1 - i;
    const long long t0 = (long long)c * kC;
    const int n = (int)min((long long)kC, p.T - t0);
    load_tile<E, D>(A, ta, ha, t0, n, p.dk);
    load_tile<E, D>(Bt, tv, hv, t0, n, p.dv);
    if (warp == 0) decay_table(lg + t0 * p.lst, p.lst, n, sm.ch, sm.cl);
    cp_async_wait_all();
    sync();
    const double total = (double)sm.ch[kC - 1] + (double)sm.cl[kC - 1];
    const float rh = (float)run, th = sm.ch[kC - 1], tl = sm.cl[kC - 1];
    scale_rows<NL, D>(A, lv, [&](int r) {
      return kBwd ? ex2((sm.ch[r] + rh) + sm.cl[r]) : ex2(((th - sm.ch[r]) + rh) + (tl - sm.cl[r]));
    });
    run += total;
    sync();
    if (ok && tid == 0) {
      product_rows<NL, D>(sm.tbase, lv, Bt, false);
      um::commit(&sm.bar);
    }
    if (ok) ok = mbar_wait(&sm.bar, phase & 1, &g_sticky_err);
    ++phase;
    um::fence_after();
    st.update(1.f, sm.tbase, 0);  // in registers: round to nearest
  }
  // forward: the state that enters segment s + 1; backward: the gradient that leaves s - 1
  if (ok) {
    st.store_own(p.seg + (bh * p.nseg + s + (kBwd ? -1 : 1)) * (D * D));
    if (tid == 0) p.segl[bh * p.nseg + s] = (float)run;
  }
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, D);
}

// Joins the segments along the sequence: slot s + 1 = e^{L_s} slot s + what s
// added, from H0 (backward: slot s - 1 from slot s, from dH_T). One thread to
// four elements of one (batch, head).
template <int D, bool kBwd>
__global__ void __launch_bounds__(256) scan_kernel(float* seg, const float* segl, const float* init,
                                                   long long BH, int nseg, int dk, int dv) {
  const long long g = (long long)blockIdx.x * 256 + threadIdx.x;
  const long long bh = g / (D * D / 4);
  if (bh >= BH) return;
  const int e = (int)(g % (D * D / 4)), row = e % D, col = (e / D) * 4;
  float x[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[i] = init && row < dk && col + i < dv ? init[(bh * dk + row) * dv + col + i] : 0.f;
  float4* sp = reinterpret_cast<float4*>(seg + bh * nseg * (long long)(D * D)) + e;
  const float* lp = segl + bh * nseg;
#pragma unroll 4
  for (int i = 0; i < nseg - 1; ++i) {
    const int s = kBwd ? nseg - 1 - i : i, to = kBwd ? s - 1 : s + 1;
    const float f = ex2(lp[s]);
    float4 u = sp[(long long)to * (D * D / 4)];
    x[0] = fmaf(f, x[0], u.x), x[1] = fmaf(f, x[1], u.y);
    x[2] = fmaf(f, x[2], u.z), x[3] = fmaf(f, x[3], u.w);
    sp[(long long)to * (D * D / 4)] = make_float4(x[0], x[1], x[2], x[3]);
  }
}

// ---------------------------------------------------------------- forward --

// TMEM columns: masked product 0..127, y 128.., P (NL levels of 64) after it;
// the state's sum takes 0.. once the product has been read.
template <typename E, int D>
struct Fwd {
  static constexpr int NL = kLevels<E>, kTileE = kC * D;
  static constexpr int kY = 128, kP = 128 + D, kCols = kP + 64 * NL <= 256 ? 256 : 512;
  static constexpr int kExtra = NL == 1 ? 1 : 0;  // third level of the scaled K rows
  static constexpr size_t kSmem = kSmallBytes + 2 * ((3 * NL + kExtra) * (size_t)kTileE + NL * (size_t)D * D);
  static constexpr int kPerSm = 2 * (kSmem + 1024) <= 228 * 1024 && kCols <= 256 ? 2 : 1;
};

template <typename E, int D>
__global__ void __launch_bounds__(kThreads, Fwd<E, D>::kPerSm) fwd_kernel(const Args<E> p) {
  using F = Fwd<E, D>;
  constexpr int NL = F::NL, kTileE = F::kTileE;
  extern __shared__ __align__(1024) unsigned char smem[];
  Small& sm = *reinterpret_cast<Small*>(smem);
  bf16* Q = reinterpret_cast<bf16*>(smem + kSmallBytes);
  bf16 *K = Q + NL * kTileE, *V = K + NL * kTileE, *X = V + (NL + F::kExtra) * kTileE;
  // the scaled K rows go over K and, below three levels, over Q (read by then) and the extra tile
  bf16* const lv[3] = {K, NL == 1 ? Q : K + kTileE, NL == 1 ? V + kTileE : NL == 2 ? Q : K + 2 * kTileE};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = warp & 3, wg = warp >> 2;
  const long long bh = blockIdx.x % p.BH;
  const int s = (int)(blockIdx.x / p.BH);
  const long long b = bh / p.H, h = bh % p.H;
  const E* hq = p.Q.p + b * p.Q.sb + h * p.Q.sh;
  const E* hk = p.K.p + b * p.K.sb + h * p.K.sh;
  const E* hv = p.V.p + b * p.V.sb + h * p.V.sh;
  E* hy = p.y.p + b * p.y.sb + h * p.y.sh;
  const float* lg = p.lg + b * p.lsb + h * p.lsh;
  const long long dkv = (long long)p.dk * p.dv;

  if (warp == 0) um::alloc(&sm.tbase, F::kCols);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_fence_init();
  }
  State<D> S;
  if (s > 0)
    S.load_own(p.seg + (bh * p.nseg + s) * (D * D));
  else if (p.H0)
    S.load(p.H0 + bh * dkv, p.dk, p.dv);
  else
    S.zero();
  S.template to_smem<NL>(X);
  // After a wait that runs out (recorded in the sticky word) the CTA issues no
  // MMA, waits on nothing and writes no output; sync makes the flag common.
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  unsigned phase = 0;
  auto wait = [&]() {
    if (ok) ok = mbar_wait(&sm.bar, phase & 1, &g_sticky_err);
    ++phase;
    um::fence_after();
  };
  const int row = 32 * q + lane;
  const int c0 = s * p.m, c1 = min(c0 + p.m, p.nchunks);
  for (int c = c0; c < c1; ++c) {
    const long long t0 = (long long)c * kC;
    const int n = (int)min((long long)kC, p.T - t0);
    load_tile<E, D>(Q, p.Q, hq, t0, n, p.dk);
    load_tile<E, D>(K, p.K, hk, t0, n, p.dk);
    load_tile<E, D>(V, p.V, hv, t0, n, p.dv);
    if (warp == 0) decay_table(lg + t0 * p.lst, p.lst, n, sm.ch, sm.cl);
    if (p.saved) S.store_own(p.saved + (bh * p.nchunks + c) * (D * D));
    cp_async_wait_all();
    sync();
    const uint32_t tb = sm.tbase;
    if (ok && tid == 0) {
      product<NL, NL, 128, 128>(tb, op_k(Q, D, kTileE), op_k(K, D, kTileE), D / 16);
      product<NL, NL, 128, D>(tb + F::kY, op_k(Q, D, kTileE), op_mn(X, D, D * D), D / 16);
      um::commit(&sm.bar);
    }
    wait();
    const uint32_t lb = tb + ((uint32_t)(32 * q) << 16);
    const float rh = sm.ch[row], rl = sm.cl[row];
#pragma unroll
    for (int k = 0; k < 4; ++k) {  // P = D * Q K^T, 64 columns to a warp
      const int j0 = 64 * wg + 16 * k;
      float v[16];
      if (j0 > 32 * q + 31) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
      } else {
        um::ld16(lb + j0, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float f = ex2((rh - sm.ch[j0 + i]) + (rl - sm.cl[j0 + i]));
          v[i] = j0 + i <= row ? v[i] * f : 0.f;
        }
      }
      st_levels16<NL>(lb + F::kP + j0 / 2, v);
    }
    {  // the state's part of y: diag(e^c) Q S
      const float f = ex2(rh + rl);
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const uint32_t a = lb + F::kY + wg * (D / 2) + 16 * k;
        float v[16];
        uint32_t w[16];
        um::ld16(a, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) w[i] = __float_as_uint(v[i] * f);
        st16(a, w);
      }
    }
    st_wait();
    const float th = sm.ch[kC - 1], tl = sm.cl[kC - 1];
    const bool add = c + 1 < c1 || s + 1 == p.nseg;  // a later chunk of this CTA, or H_T, needs S'
    if (add)
      scale_rows<NL, D>(K, lv, [&](int r) { return ex2((th - sm.ch[r]) + (tl - sm.cl[r])); });
    sync();
    if (ok && tid == 0) {
      product_ta<NL, NL, D>(tb + F::kY, tb + F::kP, op_mn(V, D, kTileE), true);
      if (add) product_rows<NL, D>(tb, lv, V, false);
      um::commit(&sm.bar);
    }
    wait();
    if (ok) {
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const int j0 = wg * (D / 2) + 16 * k;
        float v[16];
        um::ld16(lb + F::kY + j0, v);
        if (row < n) store_row16<E>(hy + (t0 + row) * p.y.st, j0, p.dv, p.y.vec, v);
      }
    }
    if (add) {
      S.update(ex2(th + tl), tb, 0);
      S.template to_smem<NL>(X);
    }
    sync();
  }
  if (ok && s + 1 == p.nseg) S.store(p.HT + bh * dkv, p.dk, p.dv);
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, F::kCols);
}

// --------------------------------------------------------------- backward --

struct SmallB {
  uint64_t bar;
  uint32_t tbase;
  float dot;
  float ch[kC], cl[kC];  // decay table; at the end of a chunk what a token adds to later ones
  float a[2][kC];        // per half: what token i adds to dlog_gamma_t for t <= i
};
constexpr int kSmallB = 3072;
static_assert(sizeof(SmallB) <= kSmallB, "");

// NL = 1: 64 masked products of a lane's row, rounded and packed while both
// accumulators are still being read; NL > 1: as they are.
template <int NL>
struct Held {
  std::conditional_t<NL == 1, uint32_t, float> v[NL == 1 ? 32 : 64];
  __device__ __forceinline__ void set(int k, const float (&x)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      if constexpr (NL == 1) {
        if (i % 2 == 0) {
          const __nv_bfloat162 h = __floats2bfloat162_rn(x[i], x[i + 1]);
          v[8 * k + i / 2] = *reinterpret_cast<const uint32_t*>(&h);
        }
      } else {
        v[16 * k + i] = x[i];
      }
    }
  }
  __device__ __forceinline__ void store(uint32_t taddr) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (NL == 1)
        st8(taddr + 8 * k, v + 8 * k);
      else
        st_levels16<NL>(taddr + 8 * k, v + 16 * k);
    }
  }
};

// TMEM columns, first half of a chunk: (K Q^T) 0..127 and (V dy^T) 128..255;
// once read, their masked forms A2 at 0, A1 at 64 NL (NL levels of 64), dV at
// 128 NL, dK after it; once these are done, the state parts at kIv and kIk.
// Second half: (dy V^T) 0..127 and (Q K^T) 128..255; once read, A1 at 0, dQ at
// 64 NL, its state part after it, and at last the state's sum at 0.
template <typename E, int D>
struct Bwd {
  static constexpr int NL = kLevels<E>, kTileE = kC * D;
  static constexpr int kDv = 128 * NL, kDk = kDv + D;
  static constexpr int kIv = 0, kIk = 2 * D <= kDv ? D : kDk + D;
  static constexpr int kDq = 64 * NL, kIq = kDq + D;
  static constexpr int kCols = kDk + D <= 256 ? 256 : 512;
  static_assert(kDk + D <= 512 && kIk + D <= 512 && kIq + D <= kCols, "");
  // dS rests in shared memory between its uses where two CTAs share an SM's registers
  static constexpr bool kPark = NL == 1 && D == 64;
  static constexpr size_t kSmem =
      kSmallB + 2 * (4 * NL * (size_t)kTileE + 3 * (size_t)D * D) + (kPark ? 4 * D * D : 0);
  static constexpr int kPerSm = 2 * (kSmem + 1024) <= 228 * 1024 && kCols <= 256 ? 2 : 1;
};
template <typename E, int D>
__global__ void __launch_bounds__(kThreads, Bwd<E, D>::kPerSm) bwd_kernel(const Args<E> p) {
  using F = Bwd<E, D>;
  constexpr int NL = F::NL, kTileE = F::kTileE;
  extern __shared__ __align__(1024) unsigned char smem[];
  SmallB& sm = *reinterpret_cast<SmallB*>(smem);
  bf16* Q = reinterpret_cast<bf16*>(smem + kSmallB);
  bf16 *K = Q + NL * kTileE, *V = K + NL * kTileE, *G = V + NL * kTileE, *X = G + NL * kTileE;
  // the scaled Q rows go over Q and, below three levels, over K and V (read by then)
  bf16* const lv[3] = {Q, NL == 1 ? K : Q + kTileE, NL == 1 ? V : NL == 2 ? K : Q + 2 * kTileE};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, q = warp & 3, wg = warp >> 2;
  const long long bh = blockIdx.x % p.BH;
  const int s = p.nseg - 1 - (int)(blockIdx.x / p.BH);
  const long long b = bh / p.H, h = bh % p.H;
  const E* hq = p.Q.p + b * p.Q.sb + h * p.Q.sh;
  const E* hk = p.K.p + b * p.K.sb + h * p.K.sh;
  const E* hv = p.V.p + b * p.V.sb + h * p.V.sh;
  const E* hg = p.dy.p + b * p.dy.sb + h * p.dy.sh;
  const float* lg = p.lg + b * p.lsb + h * p.lsh;
  const long long dkv = (long long)p.dk * p.dv;

  if (warp == 0) um::alloc(&sm.tbase, F::kCols);
  if (tid == 0) {
    mbar_init(&sm.bar, 1);
    mbar_fence_init();
  }
  float* park = reinterpret_cast<float*>(X + 3 * D * D);
  State<D> dS;
  if (s + 1 < p.nseg)
    dS.load_own(p.seg + (bh * p.nseg + s) * (D * D));
  else if (p.dHT)
    dS.load(p.dHT + bh * dkv, p.dk, p.dv);
  else
    dS.zero();
  dS.template to_smem<3>(X);
  if (F::kPark) dS.store_own(park);
  bool ok = true;
  auto sync = [&]() {
    fence_proxy_async_smem();
    um::fence_before();
    ok = !__syncthreads_or(!ok);
    um::fence_after();
  };
  unsigned phase = 0;
  auto wait = [&]() {
    if (ok) ok = mbar_wait(&sm.bar, phase & 1, &g_sticky_err);
    ++phase;
    um::fence_after();
  };
  const int row = 32 * q + lane;
  const int c0 = s * p.m, c1 = min(c0 + p.m, p.nchunks);
  for (int c = c1 - 1; c >= c0; --c) {
    const long long t0 = (long long)c * kC;
    const int n = (int)min((long long)kC, p.T - t0);
    load_tile<E, D>(Q, p.Q, hq, t0, n, p.dk);
    load_tile<E, D>(K, p.K, hk, t0, n, p.dk);
    load_tile<E, D>(V, p.V, hv, t0, n, p.dv);
    load_tile<E, D>(G, p.dy, hg, t0, n, p.dv);
    if (warp == 0) decay_table(lg + t0 * p.lst, p.lst, n, sm.ch, sm.cl);
    cp_async_wait_all();
    sync();
    const uint32_t tb = sm.tbase, lb = tb + ((uint32_t)(32 * q) << 16);
    const Op kQ = op_k(Q, D, kTileE), kK = op_k(K, D, kTileE), kV = op_k(V, D, kTileE),
             kG = op_k(G, D, kTileE);
    if (ok && tid == 0) {
      product<NL, NL, 128, 128>(tb, kK, kQ, D / 16);
      product<NL, NL, 128, 128>(tb + 128, kV, kG, D / 16);
      um::commit(&sm.bar);
    }
    wait();
    const float rh = sm.ch[row], rl = sm.cl[row], th = sm.ch[kC - 1], tl = sm.cl[kC - 1];
    const float to_end = ex2((th - rh) + (tl - rl)), from_start = ex2(rh + rl);
    float tok = 0.f;  // this half's part of what token `row` adds for t <= row
    float bk = 0.f;   // what it adds for t > row
    {
      // Lane: token j = row; columns: tokens i >= j. A2 = D * (K Q^T), A1 = D * (V dy^T).
      Held<NL> a1, a2;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int i0 = 64 * wg + 16 * k;
        float x[16], z[16];
        if (i0 + 15 < 32 * q) {
#pragma unroll
          for (int i = 0; i < 16; ++i) x[i] = z[i] = 0.f;
        } else {
          uint32_t r1[16], r2[16];
          um::ld16_async(lb + i0, r1);
          um::ld16_async(lb + 128 + i0, r2);
          um::ld_wait();
          um::ld_bind(r1, x);
          um::ld_bind(r2, z);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float f = ex2((sm.ch[i0 + i] - rh) + (sm.cl[i0 + i] - rl));
            const float pf = x[i] * f;
            tok -= i0 + i > row ? pf * z[i] : 0.f;
            x[i] = i0 + i >= row ? pf : 0.f;
            z[i] = i0 + i >= row ? z[i] * f : 0.f;
          }
        }
        a2.set(k, x);
        a1.set(k, z);
      }
      sync();  // both products have been read
      a2.store(lb + 32 * wg);
      a1.store(lb + 64 * NL + 32 * wg);
      st_wait();
    }
    sync();
    if (ok && tid == 0) {
      product_ta<NL, NL, D>(tb + F::kDv, tb, op_mn(G, D, kTileE), false);
      product_ta<NL, NL, D>(tb + F::kDk, tb + 64 * NL, op_mn(Q, D, kTileE), false);
      um::commit(&sm.bar);
    }
    wait();
    if (ok && tid == 0) {
      product<NL, 3, 128, D>(tb + F::kIv, kK, op_mn(X, D, D * D), D / 16);
      product<NL, 3, 128, D>(tb + F::kIk, kV, op_k(X, D, D * D), D / 16);
      um::commit(&sm.bar);
    }
    wait();
    E* gv = p.dV.p + b * p.dV.sb + h * p.dV.sh + (t0 + row) * p.dV.st;
    E* gk = p.dK.p + b * p.dK.sb + h * p.dK.sh + (t0 + row) * p.dK.st;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      const int j0 = wg * (D / 2) + 16 * k;
      uint32_t r1[16], r2[16];
      float x[16], z[16];
      um::ld16_async(lb + F::kDv + j0, r1);
      um::ld16_async(lb + F::kIv + j0, r2);
      um::ld_wait();
      um::ld_bind(r1, x);
      um::ld_bind(r2, z);
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = fmaf(to_end, z[i], x[i]);
      if (ok && row < n) store_row16<E>(gv, j0, p.dv, p.dV.vec, x);
      um::ld16_async(lb + F::kDk + j0, r1);
      um::ld16_async(lb + F::kIk + j0, r2);
      um::ld_wait();
      um::ld_bind(r1, x);
      um::ld_bind(r2, z);
      float kr[16];
      load_levels8<NL>(K, kTileE, um::boff_n(row, j0, D), kr);
      load_levels8<NL>(K, kTileE, um::boff_n(row, j0 + 8, D), kr + 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        bk = fmaf(kr[i], z[i], bk);
        x[i] = fmaf(to_end, z[i], x[i]);
      }
      if (ok && row < n) store_row16<E>(gk, j0, p.dk, p.dK.vec, x);
    }
    bk *= to_end;
    {  // S, the state that entered the chunk, takes dS's place in shared memory
      State<D> S;
      S.load_own(p.saved + (bh * p.nchunks + c) * (D * D));
      if (F::kPark) dS.load_own(park);
      float d = 0.f;
#pragma unroll
      for (int i = 0; i < State<D>::kCols; ++i) d = fmaf(S.v[i], dS.v[i], d);
      if (!State<D>::valid()) d = 0.f;  // lanes without a row hold what their TMEM lanes held
      S.template to_smem<3>(X);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
      if (lane == 0) sm.a[0][warp] = d;  // joined below, in order
    }
    sync();
    if (ok && tid == 0) {
      product<NL, NL, 128, 128>(tb, kG, kV, D / 16);
      product<NL, NL, 128, 128>(tb + 128, kQ, kK, D / 16);
      um::commit(&sm.bar);
    }
    if (tid == 32) {
      float d = 0.f;
      for (int i = 0; i < 8; ++i) d += sm.a[0][i];
      sm.dot = d;
    }
    wait();
    {
      // Lane: token i = row; columns: tokens j <= i. A1 = D * (dy V^T).
      Held<NL> a1;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j0 = 64 * wg + 16 * k;
        float x[16], z[16];
        if (j0 > 32 * q + 31) {
#pragma unroll
          for (int i = 0; i < 16; ++i) z[i] = 0.f;
        } else {
          uint32_t r1[16], r2[16];
          um::ld16_async(lb + j0, r1);
          um::ld16_async(lb + 128 + j0, r2);
          um::ld_wait();
          um::ld_bind(r1, z);
          um::ld_bind(r2, x);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float f = ex2((rh - sm.ch[j0 + i]) + (rl - sm.cl[j0 + i]));
            const float zf = z[i] * f;
            tok += j0 + i < row ? zf * x[i] : 0.f;
            z[i] = j0 + i <= row ? zf : 0.f;
          }
        }
        a1.set(k, z);
      }
      sync();
      a1.store(lb + 32 * wg);
      st_wait();
    }
    sync();
    if (ok && tid == 0) {
      product_ta<NL, NL, D>(tb + F::kDq, tb, op_mn(K, D, kTileE), false);
      product<NL, 3, 128, D>(tb + F::kIq, kG, op_k(X, D, D * D), D / 16);
      um::commit(&sm.bar);
    }
    wait();
    E* gq = p.dQ.p + b * p.dQ.sb + h * p.dQ.sh + (t0 + row) * p.dQ.st;
    float aq = 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) {
      const int j0 = wg * (D / 2) + 16 * k;
      uint32_t r1[16], r2[16];
      float x[16], z[16], qr[16];
      um::ld16_async(lb + F::kDq + j0, r1);
      um::ld16_async(lb + F::kIq + j0, r2);
      um::ld_wait();
      um::ld_bind(r1, x);
      um::ld_bind(r2, z);
      load_levels8<NL>(Q, kTileE, um::boff_n(row, j0, D), qr);
      load_levels8<NL>(Q, kTileE, um::boff_n(row, j0 + 8, D), qr + 8);
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        aq = fmaf(qr[i], z[i], aq);
        x[i] = fmaf(from_start, z[i], x[i]);
      }
      if (ok && row < n) store_row16<E>(gq, j0, p.dk, p.dQ.vec, x);
    }
    sm.a[wg][row] = fmaf(from_start, aq, tok);
    sync();
    scale_rows<NL, D>(Q, lv, [&](int r) { return ex2(sm.ch[r] + sm.cl[r]); });
    sync();
    if (ok && tid == 0) {
      product_rows<NL, D>(tb, lv, G, false);
      um::commit(&sm.bar);
    }
    (wg == 0 ? sm.ch : sm.cl)[row] = bk;  // the decay table has been used
    wait();
    const float g = ex2(th + tl);
    if (F::kPark) dS.load_own(park);
    dS.update(g, tb, 0);
    dS.template to_smem<3>(X);
    if (F::kPark) dS.store_own(park);
    sync();
    if (warp == 0 && ok) {
      // Token i adds a to dlog_gamma_t for t <= i and bk for t > i: four tokens to a lane,
      // a summed from the end and bk from the start.
      double va[4], vb[4], ra = 0.0, rb = 0.0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int e = 4 * lane + 3 - i, f = 4 * lane + i;
        ra += (double)sm.a[0][e] + (double)sm.a[1][e];
        va[3 - i] = ra;
        vb[i] = rb;
        rb += (double)sm.ch[f] + (double)sm.cl[f];
      }
      double ia = ra, ib = rb;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double x = __shfl_down_sync(0xffffffffu, ia, o), y = __shfl_up_sync(0xffffffffu, ib, o);
        if (lane + o < 32) ia += x;
        if (lane >= o) ib += y;
      }
      const double rest = (ia - ra) + (ib - rb) + (double)(sm.dot * g);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int t = 4 * lane + i;
        if (t < n) {
          const float l = lg[(t0 + t) * p.lst] * 1.4426950408889634f;
          p.dlg[bh * p.T + t0 + t] = l <= kMinLog2 ? 0.f : (float)(va[i] + vb[i] + rest);
        }
      }
    }
    __syncwarp();
  }
  if (ok && s == 0 && p.dH0) dS.store(p.dH0 + bh * dkv, p.dk, p.dv);
  um::fence_before();
  __syncthreads();
  if (warp == 0) um::dealloc(sm.tbase, F::kCols);
}

// ------------------------------------------------------------------- host --

struct Plan {
  int D, nchunks, m, nseg;
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

// Segments: as many as there are places for CTAs, whole chunks to each.
Plan plan_for(long long BH, long long T, int D, int per_sm) {
  Plan pl;
  pl.D = D;
  pl.nchunks = (int)((T + kC - 1) / kC);
  const long long places = (long long)sm_count() * per_sm;
  long long want = BH > 0 ? places / BH : 1;
  want = want < 1 ? 1 : want > pl.nchunks ? pl.nchunks : want;
  pl.m = want > 0 ? (int)((pl.nchunks + want - 1) / want) : 1;
  pl.nseg = pl.m > 0 ? (pl.nchunks + pl.m - 1) / pl.m : 0;
  return pl;
}

template <class F>
int by_shape(int dtype, int dk, int dv, F&& f) {
  const int d = dk > dv ? dk : dv;
  if (dtype == MGS_BF16)
    return d <= 64    ? f(bf16{}, std::integral_constant<int, 64>{})
           : d <= 128 ? f(bf16{}, std::integral_constant<int, 128>{})
                      : (int)MGS_UNSUPPORTED;
  if (dtype != MGS_F32 && dtype != MGS_F16) return MGS_BAD_DTYPE;
  if (d > 64) return MGS_UNSUPPORTED;
  return dtype == MGS_F32 ? f(float{}, std::integral_constant<int, 64>{})
                          : f(__half{}, std::integral_constant<int, 64>{});
}

size_t seg_bytes(const Plan& pl, long long BH) {
  return pl.nseg > 1 ? (size_t)BH * pl.nseg * ((size_t)pl.D * pl.D + 1) * sizeof(float) : 0;
}

bool shape_ok(int64_t B, int H, int64_t T, int dk, int dv) {
  return B >= 0 && H >= 0 && T >= 0 && dk >= 1 && dv >= 1 && T < (1ll << 38) &&
         (B == 0 || H == 0 || B <= 0x7fffffffLL / H);
}

template <typename P>
Ten<P> ten(P* p, const int64_t* s, int d) {
  const long long e = 16 / sizeof(P);
  const bool vec = reinterpret_cast<uintptr_t>(p) % 16 == 0 && d % 8 == 0 && s[0] % e == 0 &&
                   s[1] % e == 0 && s[2] % e == 0;
  return {p, (long long)s[0], (long long)s[1], (long long)s[2], vec ? 1 : 0};
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
  constexpr size_t smem = kSmallBytes + 2 * (3 + kLevels<E>)*(size_t)(kC * D);
  auto k1 = state_kernel<E, D, kBwd>;
  if (int r = set_smem(k1, smem)) return r;
  k1<<<(unsigned)(a.BH * (a.nseg - 1)), kThreads, smem, st>>>(a);
  if (int r = launched()) return r;
  const long long n = a.BH * (D * D / 4);
  scan_kernel<D, kBwd><<<(unsigned)((n + 255) / 256), 256, 0, st>>>(
      a.seg, a.segl, kBwd ? a.dHT : a.H0, a.BH, a.nseg, a.dk, a.dv);
  return launched();
}

template <typename E, int D>
int run_main(bool fwd, const Args<E>& a, cudaStream_t st) {
  if (int r = fwd ? run_segments<E, D, false>(a, st) : run_segments<E, D, true>(a, st)) return r;
  auto k = fwd ? fwd_kernel<E, D> : bwd_kernel<E, D>;
  const size_t smem = fwd ? Fwd<E, D>::kSmem : Bwd<E, D>::kSmem;
  if (int r = set_smem(k, smem)) return r;
  k<<<(unsigned)(a.BH * a.nseg), kThreads, smem, st>>>(a);
  return launched();
}

template <typename E, int D>
int fill(Args<E>& a, bool fwd, const float* lg, const int64_t* ls, int64_t B, int H, int64_t T, int dk,
         int dv, void* ws, size_t ws_bytes) {
  const long long BH = B * (long long)H;
  const Plan pl = plan_for(BH, T, D, fwd ? Fwd<E, D>::kPerSm : Bwd<E, D>::kPerSm);
  if (seg_bytes(pl, BH) > ws_bytes) return MGS_WORKSPACE_TOO_SMALL;
  if (seg_bytes(pl, BH) && (!ws || reinterpret_cast<uintptr_t>(ws) % 16)) return MGS_BAD_ALIGNMENT;
  a.lg = lg, a.lsb = ls[0], a.lsh = ls[1], a.lst = ls[2];
  a.seg = static_cast<float*>(ws);
  a.segl = a.seg + (size_t)BH * pl.nseg * D * D;
  a.T = T, a.H = H, a.dk = dk, a.dv = dv, a.nchunks = pl.nchunks, a.m = pl.m, a.nseg = pl.nseg, a.BH = BH;
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
    const size_t f = seg_bytes(plan_for(B * H, T, D, Fwd<E, D>::kPerSm), B * H);
    const size_t b = seg_bytes(plan_for(B * H, T, D, Bwd<E, D>::kPerSm), B * H);
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
    n = (size_t)(B * H) * (size_t)((T + kC - 1) / kC) * D * D * sizeof(float);
    return MGS_OK;
  });
  return n;
}

int mgs_linear_attn_fwd(const void* Q, const void* K, const void* V, const float* log_gamma,
                        const float* H0, void* y, float* H_T, float* saved, const int64_t* strides,
                        int64_t B, int H, int64_t T, int dk, int dv, int dtype, void* workspace,
                        size_t workspace_bytes, void* stream) {
  using namespace mgs::lattn;
  if (!shape_ok(B, H, T, dk, dv)) return MGS_BAD_SHAPE;
  return by_shape(dtype, dk, dv, [&](auto e, auto d) -> int {
    using E = decltype(e);
    constexpr int D = decltype(d)::value;
    if (B == 0 || H == 0 || T == 0) return MGS_OK;
    if (reinterpret_cast<uintptr_t>(saved) % 16) return MGS_BAD_ALIGNMENT;
    Args<E> a{};
    a.Q = ten(static_cast<const E*>(Q), strides, dk);
    a.K = ten(static_cast<const E*>(K), strides + 3, dk);
    a.V = ten(static_cast<const E*>(V), strides + 6, dv);
    a.y = ten(static_cast<E*>(y), strides + 12, dv);
    a.H0 = H0, a.HT = H_T, a.saved = saved;
    if (int r = fill<E, D>(a, true, log_gamma, strides + 9, B, H, T, dk, dv, workspace, workspace_bytes))
      return r;
    return run_main<E, D>(true, a, static_cast<cudaStream_t>(stream));
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
    constexpr int D = decltype(d)::value;
    if (B == 0 || H == 0 || T == 0) return MGS_OK;
    if (reinterpret_cast<uintptr_t>(saved) % 16) return MGS_BAD_ALIGNMENT;
    Args<E> a{};
    a.Q = ten(static_cast<const E*>(Q), strides, dk);
    a.K = ten(static_cast<const E*>(K), strides + 3, dk);
    a.V = ten(static_cast<const E*>(V), strides + 6, dv);
    a.dy = ten(static_cast<const E*>(dy), strides + 12, dv);
    a.dQ = ten(static_cast<E*>(dQ), strides + 15, dk);
    a.dK = ten(static_cast<E*>(dK), strides + 18, dk);
    a.dV = ten(static_cast<E*>(dV), strides + 21, dv);
    a.saved = const_cast<float*>(saved), a.dHT = dH_T, a.dH0 = dH0, a.dlg = dlog_gamma;
    if (int r = fill<E, D>(a, false, log_gamma, strides + 9, B, H, T, dk, dv, workspace, workspace_bytes))
      return r;
    return run_main<E, D>(false, a, static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
