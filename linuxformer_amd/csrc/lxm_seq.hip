// The gated delta rule layer's core for many sequences at once: the short convolution, the recurrence for
// single tokens and short runs, and the chunked form of it for prompts (include/lxm_seq.h).
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <stdint.h>

#include "../../include/lxm_seq.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef int32_t i32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

template <int TY>
struct Elem;
template <>
struct Elem<LXM_BF16> {
  typedef uint16_t T;
};
template <>
struct Elem<LXM_FP16> {
  typedef uint16_t T;
};
template <>
struct Elem<LXM_FP32> {
  typedef float T;
};

__device__ __forceinline__ float half_up(uint32_t h) { return (float)__builtin_bit_cast(_Float16, (uint16_t)h); }

// one element, to and from float32 (to nearest even)
template <int TY>
__device__ __forceinline__ float up(typename Elem<TY>::T x) {
  if constexpr (TY == LXM_BF16) return __uint_as_float((uint32_t)x << 16);
  else if constexpr (TY == LXM_FP16) return half_up(x);
  else return x;
}
template <int TY>
__device__ __forceinline__ typename Elem<TY>::T down(float x) {
  if constexpr (TY == LXM_BF16) return __builtin_bit_cast(uint16_t, (__bf16)x);
  else if constexpr (TY == LXM_FP16) return __builtin_bit_cast(uint16_t, (_Float16)x);
  else return x;
}
__device__ __forceinline__ float up_of(const void* p, int64_t i, int type) {
  return type == LXM_BF16 ? up<LXM_BF16>(((const uint16_t*)p)[i])
         : type == LXM_FP16 ? up<LXM_FP16>(((const uint16_t*)p)[i])
                            : ((const float*)p)[i];
}

// the elements of one 16-byte word (8 of 16 bits, 4 of 32)
template <int TY>
constexpr int kVec = TY == LXM_FP32 ? 4 : 8;
template <int TY>
__device__ __forceinline__ void unpack(u32x4 u, float* x) {
  if constexpr (TY == LXM_FP32) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      x[2 * i] = up<TY>((uint16_t)(u[i] & 0xffff));
      x[2 * i + 1] = up<TY>((uint16_t)(u[i] >> 16));
    }
  }
}
template <int TY>
__device__ __forceinline__ u32x4 pack(const float* x) {
  u32x4 u;
  if constexpr (TY == LXM_FP32) {
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = __float_as_uint(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) u[i] = down<TY>(x[2 * i]) | (uint32_t)down<TY>(x[2 * i + 1]) << 16;
  }
  return u;
}

__device__ __forceinline__ float fma(float a, float b, float c) { return __builtin_fmaf(a, b, c); }
__device__ __forceinline__ int wave_of() { return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); }
// what this wave's lanes stored in LDS, for its other lanes (a wave's LDS accesses run in order)
__device__ __forceinline__ void wave_sync() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_wave_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}
// LDS writes seen by the other waves, without waiting for loads from memory in flight
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\ns_barrier" ::: "memory"); }
// MFMAs at the end of a branch are waited for there: where the branch joined another path the compiler has
// read the last one's rows with no wait states in between
__device__ __forceinline__ void settle(f32x4& c) { asm volatile("s_nop 15" : "+v"(c)); }

// a sequence's and a chunk's record (lxm_seq_table)
struct Seq {
  int slot, first, end, chunk;
};
struct Chunk {
  int first, n, seq, number;
};
__device__ __forceinline__ Seq seq_at(const lxm_seq_table& t, int i) {
  return __builtin_bit_cast(Seq, ((const i32x4*)t.seqs)[i]);
}
__device__ __forceinline__ Chunk chunk_at(const lxm_seq_table& t, int i) {
  return __builtin_bit_cast(Chunk, ((const i32x4*)t.chunks)[i]);
}

// ---- the short convolution ----------------------------------------------------------------------------
// y_t = silu(sum_j w_j x_{t-3+j}): each input is read once and each output written once, so bytes bound it.
// A thread takes N channels (one 16-byte word, or one element where alignment or C allows no more) of up to
// kRun positions of one sequence, all its rows requested before any is used. Runs are counted from their
// sequence's start, so only a sequence's first run reads the window, and that same thread writes it:
// nobody else's read can come after. 1,928 positions of 16 sequences, 8,192 bf16 channels: 18.8 us a call, 3.5 TB/s
// of the bytes it cannot do without (runs of 16: 22.8, half the waves a CU for their registers; of 4: 19.5).
constexpr int kRun = 8;

template <int TY, int N>
__device__ __forceinline__ void load_n(const typename Elem<TY>::T* p, float* x) {
  if constexpr (N == 1) x[0] = up<TY>(p[0]);
  else unpack<TY>(*(const u32x4*)p, x);
}
template <int TY, int N>
__device__ __forceinline__ void store_n(typename Elem<TY>::T* p, const float* x) {
  if constexpr (N == 1) p[0] = down<TY>(x[0]);
  else *(u32x4*)p = pack<TY>(x);
}

template <int TY, int N>
__global__ __launch_bounds__(256) void short_conv(lxm_seq_table S, lxm_conv_io io, int runs, int cblocks) {
  typedef typename Elem<TY>::T T;
  const int cb = blockIdx.x % cblocks, u = blockIdx.x / cblocks;
  const Chunk ch = chunk_at(S, u / runs);
  const int run = u % runs, n = min(kRun, ch.n - run * kRun);
  const int t0 = ch.number * LXM_SEQ_CHUNK + run * kRun;  // in the sequence
  const int c = (cb * 256 + threadIdx.x) * N;
  if (n <= 0 || c >= io.C) return;
  const T* x = (const T*)io.x + (int64_t)(ch.first + run * kRun) * io.x_ts + c;
  T* y = (T*)io.y + (int64_t)(ch.first + run * kRun) * io.y_ts + c;

  float w[4][N], h[3][N];
  {
    float e[4 * N];
    const T* p = (const T*)io.w + (int64_t)c * 4;
#pragma unroll
    for (int i = 0; i < 4; i++) load_n<TY, N>(p + i * N, e + i * N);
#pragma unroll
    for (int i = 0; i < 4 * N; i++) w[i % 4][i / 4] = e[i];
  }
  float rows[kRun][N];
#pragma unroll
  for (int t = 0; t < kRun; t++)
    if (t < n) load_n<TY, N>(x + t * io.x_ts, rows[t]);
  if (t0 > 0) {
#pragma unroll
    for (int j = 0; j < 3; j++) load_n<TY, N>(x + (j - 3) * io.x_ts, h[j]);
  } else {
    const Seq q = seq_at(S, ch.seq);
    const int slot = q.slot, len = q.end - q.first;
    float e[4 * N] = {};
    T* p = (T*)io.window + (int64_t)slot * io.w_ss + (int64_t)c * 4;
    if (slot >= 0) {
#pragma unroll
      for (int i = 0; i < 4; i++) load_n<TY, N>(p + i * N, e + i * N);
    }
#pragma unroll
    for (int i = 0; i < 4 * N; i++)
      if (i % 4) h[i % 4 - 1][i / 4] = e[i];
    if (slot >= 0) {  // the last four of (the window's four, the sequence's inputs)
      float z[4 * N];
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int t = len - 4 + j;  // the sequence's input, or (negative) the window's 4 + t
        float row[N];
        if (t >= 0) {
          load_n<TY, N>(x + t * io.x_ts, row);
        } else {
#pragma unroll
          for (int i = 0; i < N; i++)
            row[i] = t == -1 ? e[4 * i + 3] : t == -2 ? e[4 * i + 2] : e[4 * i + 1];
        }
#pragma unroll
        for (int i = 0; i < N; i++) z[4 * i + j] = row[i];
      }
#pragma unroll
      for (int i = 0; i < 4; i++) store_n<TY, N>(p + i * N, z + i * N);
    }
  }
#pragma unroll
  for (int t = 0; t < kRun; t++) {
    if (t < n) {
      float a[N];
#pragma unroll
      for (int i = 0; i < N; i++) {
        const float* p0 = t >= 3 ? rows[t - 3] : h[t];
        const float* p1 = t >= 2 ? rows[t - 2] : h[t + 1];
        const float* p2 = t >= 1 ? rows[t - 1] : h[t + 2];
        const float s = fma(w[3][i], rows[t][i], fma(w[2][i], p2[i], fma(w[1][i], p1[i], w[0][i] * p0[i])));
        a[i] = s * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.44269504f * s));
      }
      store_n<TY, N>(y + t * io.y_ts, a);
    }
  }
}

// inclusive sum over the lanes below (row_shr 1, 2, 4, 8 within rows of 16, then the rows' last lanes), and the sum
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)u, CTRL, ROWS, 0xf, false);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(u >> 32), CTRL, ROWS, 0xf, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
template <class T>
__device__ __forceinline__ T wave_scan(T x) {
  x += dpp<0x111, 0xf>(x);
  x += dpp<0x112, 0xf>(x);
  x += dpp<0x114, 0xf>(x);
  x += dpp<0x118, 0xf>(x);
  x += dpp<0x142, 0xa>(x);
  x += dpp<0x143, 0xc>(x);
  return x;
}

__device__ __forceinline__ float wave_sum(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, wave_scan(x)), 63));
}

// ---- the recurrence -----------------------------------------------------------------------------------
// One workgroup per (sequence, value head, CB state columns): no sum crosses columns. Thread (group, column
// quad) holds rows group x R .. + R - 1 of its four columns in registers for the whole sequence. A position
// needs two sums over the rows, S^T k and S^T q; with the state before the position's decay and write,
//   o = scale (exp(g) S^T q + (k . q) d),
// so both come in one pass and one exchange between the waves. A single token is bound by its state's bytes,
// read once and written once: 64 sequences of 32 heads, 128 x 128, 52.3 us on states that are not in a cache,
// 5.1 TB/s, where a large copy reaches 4.8. A run of tokens is bound by its chain of exchanges, 1.2 us a position.
template <int TY, int K, int CB>
__global__ __launch_bounds__(256) void gd_recurrent(lxm_seq_table S, lxm_gd_io io) {
  typedef typename Elem<TY>::T T;
  constexpr int kQuads = CB / 4, kGroups = 256 / kQuads, R = K / kGroups;
  static_assert(R >= 1 && kQuads <= 64, "a wave holds whole row groups");
  const int nv = io.nk * io.r, ncb = io.V / CB;
  const int cb = blockIdx.x % ncb, h = blockIdx.x / ncb % nv;
  const Seq seq = seq_at(S, blockIdx.x / ncb / nv);
  const int f = seq.first, len = seq.end - f, slot = seq.slot;
  if (len == 0) return;
  const int tid = threadIdx.x, lane = tid & 63, wave = wave_of();
  const int quad = tid % kQuads, row0 = tid / kQuads * R, col = cb * CB + quad * 4;
  __shared__ float kq[2][2][K];      // key and query of this position and the next
  __shared__ f32x4 part[2][4][kQuads];  // the waves' sums
  __shared__ float red[4][4];

  float* sp = io.state + (int64_t)slot * io.s_ss + ((int64_t)h * K + row0) * io.V + col;
  f32x4 s[R];
#pragma unroll
  for (int i = 0; i < R; i++) s[i] = slot >= 0 ? *(const f32x4*)(sp + (int64_t)i * io.V) : f32x4{0, 0, 0, 0};

  const T* qp = (const T*)io.q + f * io.q_ts + (h / io.r) * io.q_hs;
  const T* kp = (const T*)io.k + f * io.k_ts + (h / io.r) * io.k_hs;
  const T* vp = (const T*)io.v + f * io.v_ts + h * io.v_hs + col;
  T* op = (T*)io.o + f * io.o_ts + h * io.o_hs + col;
  for (int t = 0; t < len; t++) {
    float kt = 0, qt = 0;
    if (tid < K) kt = up<TY>(kp[t * io.k_ts + tid]), qt = up<TY>(qp[t * io.q_ts + tid]);
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = up<TY>(vp[t * io.v_ts + i]);
    const float eg = expf(io.g[(f + t) * io.g_ts + h * io.g_hs]);
    const float be = up_of(io.beta, (f + t) * io.b_ts + h * io.b_hs, io.beta_type);
    float* kl = kq[t & 1][0];
    float* ql = kq[t & 1][1];
    if (tid < K) kl[tid] = kt, ql[tid] = qt;
    const float nk = wave_sum(kt * kt), nq = wave_sum(qt * qt), dot = wave_sum(kt * qt);
    if (lane == 0) red[wave][0] = nk, red[wave][1] = nq, red[wave][2] = dot;
    lds_barrier();
    float rk = 1, rq = io.scale, kd = red[0][2] + red[1][2] + red[2][2] + red[3][2];
    if (io.unit) {
      rk = 1 / sqrtf(red[0][0] + red[1][0] + red[2][0] + red[3][0] + 1e-6f);
      rq = io.scale / sqrtf(red[0][1] + red[1][1] + red[2][1] + red[3][1] + 1e-6f);
    }
    f32x4 a = {0, 0, 0, 0}, c = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < R; i++) {
      const float kx = kl[row0 + i], qx = ql[row0 + i];
#pragma unroll
      for (int j = 0; j < 4; j++) a[j] = fma(kx, s[i][j], a[j]), c[j] = fma(qx, s[i][j], c[j]);
    }
#pragma unroll
    for (int m = kQuads; m < 64; m *= 2)
#pragma unroll
      for (int j = 0; j < 4; j++) a[j] += __shfl_xor(a[j], m), c[j] += __shfl_xor(c[j], m);
    if (lane < kQuads) part[0][wave][lane] = a, part[1][wave][lane] = c;
    lds_barrier();
    a = part[0][0][quad] + part[0][1][quad] + part[0][2][quad] + part[0][3][quad];
    c = part[1][0][quad] + part[1][1][quad] + part[1][2][quad] + part[1][3][quad];
    f32x4 d;
    float o[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      d[j] = be * fma(-eg * rk, a[j], v[j]);
      o[j] = rq * fma(eg, c[j], rk * kd * d[j]);
    }
    if (tid < kQuads) {
#pragma unroll
      for (int j = 0; j < 4; j++) op[t * io.o_ts + j] = down<TY>(o[j]);
    }
#pragma unroll
    for (int i = 0; i < R; i++) {
      const float kx = rk * kl[row0 + i];
#pragma unroll
      for (int j = 0; j < 4; j++) s[i][j] = fma(kx, d[j], eg * s[i][j]);
    }
  }
  if (slot >= 0) {
#pragma unroll
    for (int i = 0; i < R; i++) *(f32x4*)(sp + (int64_t)i * io.V) = s[i];
  }
}

// ---- the chunked form ---------------------------------------------------------------------------------
// Over a chunk's positions i (chunk-relative decays gc_i = g_0 + .. + g_i, G_ij = exp(gc_i - gc_j), the state S
// before it, unit keys and queries):
//   L_ij = beta_i (k_i . k_j) G_ij for j < i,  T = (I + L)^-1,  A_ij = scale (q_i . k_j) G_ij for j <= i
//   R_i = beta_i (v_i - exp(gc_i) S^T k_i),  D = T R
//   o_i = scale exp(gc_i) S^T q_i + sum_j A_ij d_j,  S <- exp(gc_last) S + sum_i exp(gc_last - gc_i) k_i d_i^T
// T and A need no state: gd_prep forms them for all chunks at once. gd_run walks a sequence's chunks.
//
// Products on v_mfma_f32_16x16x32_bf16 (lane l: A[l % 16][8 (l / 16) + j], B[8 (l / 16) + j][l % 16],
// D[4 (l / 16) + r][l % 16]) with float32's precision, whatever the outputs' type: a float32 is the sum of three
// bf16 (8 of its 24 significant bits each, cut off, nothing rounded), a float16 of two, and a product of two such
// sums the sum of their parts' products but for the third by the third, below 2^-30 of it. (Without the second by
// the third, too, up to 2^-21 would be lost, always towards zero, for 231 us against 239 of 24 ragged prompts in
// fp32; parts rounded to nearest would lose 2^-23, but take longer to form: a bf16 prompt 72.9 us against 65.6.)
// Keys and queries go in as they were given (one part in bf16), their norms in the float32 factors beside the
// products. One such product of bf16 by float32 takes 3 instructions of 16 cycles per 32 k where the float32
// instruction takes 8 of 32. (The instruction takes a part below 2^-126 as zero: values below 2^-110 lose their last
// parts. A state that is 1e-33 throughout is off by 1e-6 of its largest value, one of 1e-36 by 1e-3.)
//
// 2,048 positions of 32 heads, bf16, 128 x 128: 66 us (gd_prep 17, gd_run 56), where the fp32 matrix
// instructions and a workspace of 75 KB a (head, chunk) take 234 for the same sums of float32 inputs.
template <int TY>
constexpr int kParts = TY == LXM_BF16 ? 1 : TY == LXM_FP16 ? 2 : 3;

__device__ __forceinline__ f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}
// the top halves of two words as one
__device__ __forceinline__ uint32_t tops(uint32_t lo, uint32_t hi) { return __builtin_amdgcn_perm(hi, lo, 0x07060302); }

// x's parts: p[s][i] holds part s of x[2 i], x[2 i + 1]
template <int N, int NP>
__device__ __forceinline__ void parts(const float* x, uint32_t (*p)[N / 2]) {
  float y[N];
#pragma unroll
  for (int i = 0; i < N; i++) y[i] = x[i];
#pragma unroll
  for (int s = 0; s < NP; s++) {
#pragma unroll
    for (int i = 0; i < N / 2; i++) p[s][i] = tops(__float_as_uint(y[2 * i]), __float_as_uint(y[2 * i + 1]));
    if (s + 1 < NP) {
#pragma unroll
      for (int i = 0; i < N; i++) y[i] -= __uint_as_float(__float_as_uint(y[i]) & 0xffff0000u);
    }
  }
}

// loads before this are requested before anything after it
__device__ __forceinline__ void issued() { asm volatile("" ::: "memory"); }

// acc += A B over one block of 32 k: the parts' products, small ones first, without the last by the last of three
template <int NA, int NB>
__device__ __forceinline__ f32x4 product(const u32x4* a, const u32x4* b, f32x4 c) {
#pragma unroll
  for (int sum = NA + NB < 6 ? NA + NB - 2 : 3; sum >= 0; sum--)
#pragma unroll
    for (int i = 0; i < NA; i++)
      if (sum - i >= 0 && sum - i < NB) c = mfma(a[i], b[sum - i], c);
  return c;
}

// The workspace: per (chunk, key head) the queries' and keys' parts as operands, [row tile 4][block K/32][part]
// each, then the keys transposed, [dim tile K/16][block 2][part]; per (chunk, value head) T as operands (3 parts
// of the 6 blocks on or below the diagonal: row tiles 0, 1 have one block of 32 columns, 2, 3 two), A the
// same, and 4 x 64 factors and the chunk's decay. A fragment is 64 lanes x 16 bytes.
constexpr int kFrag = 1024;
template <int TY, int K>
constexpr int kKeyWs = 3 * (64 * K * 2) * kParts<TY>;
constexpr int kHeadWs = 6 * (3 + 3) * kFrag + 5 * 256;

__device__ __forceinline__ int block_of(int tile, int p) { return tile < 2 ? tile : 2 * tile - 2 + p; }  // 0, 1, 2 3, 4 5

constexpr int kLd = 68;  // row stride of a 64 x 64 float32 matrix in LDS: 16-byte rows, banks spread
constexpr float kLow = -1e5f;  // exp is 0 far above it; sums of 64 of them keep their low digits in float64

// gd_prep's LDS: the chunk's keys, or the triangular matrices of up to 4 heads, and their decays
template <int TY, int K>
constexpr int kStage = kParts<TY> * 64 * (K + 8) * 2;
constexpr int kMat = 64 * kLd * 4;
struct PrepLds {
  double gc[4][64];  // in units of log 2
  float beta[4][64], rk[64], rq[64];
};

__device__ __forceinline__ f32x4 mfma32(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
// c + (16 x 16 block at a) (16 x 16 block at b), float32
__device__ __forceinline__ f32x4 block_product(const float* a, const float* b, f32x4 c, int lane) {
#pragma unroll
  for (int s = 0; s < 4; s++) {
    const int k = 4 * s + (lane >> 4);
    c = mfma32(a[(lane & 15) * kLd + k], b[k * kLd + (lane & 15)], c);
  }
  return c;
}
__device__ __forceinline__ void block_store(float* d, f32x4 c, int lane) {
#pragma unroll
  for (int r = 0; r < 4; r++) d[(4 * (lane >> 4) + r) * kLd + (lane & 15)] = c[r];
}

// (I + L)^-1 of the unit lower triangular matrix at l, by one wave, in place: the diagonal blocks of 16 by forward
// substitution (lane: a column of one), then blocks of 32 and of 64 from their halves,
// X_21 = -X_22 (L_21 X_11).
__device__ __forceinline__ void invert(float* l, int lane) {
  {
    const int b = lane >> 4, c = lane & 15;
    const float* d = l + 16 * b * kLd + 16 * b;
    float x[16];
#pragma unroll
    for (int i0 = 0; i0 < 16; i0 += 4) {  // (four rows' loads at a time: all at once take the registers of a second workgroup)
      f32x4 e[4][4];
#pragma unroll
      for (int i = 0; i < 4; i++)
#pragma unroll
        for (int j = 0; 4 * j < i0 + i; j++) e[i][j] = *(const f32x4*)(d + (i0 + i) * kLd + 4 * j);
      issued();
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float s = i0 + i == c ? 1.f : 0.f;
#pragma unroll
        for (int j = 0; j < i0 + i; j++) s = fma(-e[i][j / 4][j % 4], x[j], s);
        x[i0 + i] = s;
      }
    }
    float* e = l + 16 * b * kLd + 16 * b;
#pragma unroll
    for (int i = 0; i < 16; i++) e[i * kLd + c] = x[i];
    wave_sync();
  }
  auto at = [&](int i, int j) { return l + 16 * i * kLd + 16 * j; };
  const f32x4 zero = {0, 0, 0, 0};
  {
    const f32x4 p = block_product(at(1, 0), at(0, 0), zero, lane), q = block_product(at(3, 2), at(2, 2), zero, lane);
    block_store(at(1, 0), -p, lane);
    block_store(at(3, 2), -q, lane);
    wave_sync();
    const f32x4 x = block_product(at(1, 1), at(1, 0), zero, lane), y = block_product(at(3, 3), at(3, 2), zero, lane);
    block_store(at(1, 0), x, lane);
    block_store(at(3, 2), y, lane);
    wave_sync();
  }
  f32x4 p[2][2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    p[i][0] = block_product(at(2 + i, 1), at(1, 0), block_product(at(2 + i, 0), at(0, 0), zero, lane), lane);
    p[i][1] = block_product(at(2 + i, 1), at(1, 1), zero, lane);
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) block_store(at(2 + i, j), -p[i][j], lane);
  wave_sync();
#pragma unroll
  for (int j = 0; j < 2; j++) {
    p[1][j] = block_product(at(3, 3), at(3, j), block_product(at(3, 2), at(2, j), zero, lane), lane);
    p[0][j] = block_product(at(2, 2), at(2, j), zero, lane);
  }
#pragma unroll
  for (int i = 0; i < 2; i++)
#pragma unroll
    for (int j = 0; j < 2; j++) block_store(at(2 + i, j), p[i][j], lane);
  wave_sync();
}

// One workgroup per (chunk, key head, up to 4 of its value heads): wave w has query rows 16 w .. 16 w + 15 of both
// Gram matrices, in registers (formed as keys x rows, the keys permuted within a block of 32 so that a lane holds its
// row's 8 elements of an operand), then T and A of each of the value heads from them. Decays are summed in
// float64: behind a forgotten state (clamped to -1e5) the differences keep their digits.
// Few chunks are bound by one workgroup's latency (17 us for 512, all at once on the card), many by the
// workspace's bytes: 98 chunks of 16 key heads write 191 MB and read 61 in 51 us, 4.9 TB/s.
template <int TY, int K>
__global__ __launch_bounds__(256) void gd_prep(lxm_seq_table S, lxm_gd_io io, char* ws, int c0) {
  typedef typename Elem<TY>::T T;
  constexpr int NP = kParts<TY>, NB = K / 32, RS = K + 8;
  extern __shared__ __align__(16) char lds[];
  PrepLds& m = *(PrepLds*)lds;
  uint16_t* kt = (uint16_t*)(lds + sizeof(PrepLds));
  float* mat = (float*)(lds + sizeof(PrepLds));
  const int groups = (io.r + 3) / 4, h0 = blockIdx.x % groups * 4, nh = min(4, io.r - h0);
  const int ci = blockIdx.x / groups / io.nk, kh = blockIdx.x / groups % io.nk;
  const Chunk ch = chunk_at(S, c0 + ci);
  const int t0 = ch.first, n = ch.n;
  const int lane = threadIdx.x & 63, wave = wave_of(), g = lane >> 4, c = lane & 15, row = wave * 16 + c;
  const int nv = io.nk * io.r;
  char* wk = ws + ((int64_t)ci * io.nk + kh) * kKeyWs<TY, K>;
  char* wh = ws + (int64_t)(gridDim.x / groups) * kKeyWs<TY, K> + ((int64_t)ci * nv + kh * io.r + h0) * kHeadWs;

  // the wave's 16 rows, dims 32 i + 8 g .. + 7
  u32x4 kf[NB][NP], qf[NB][NP];
  float rq, gx = 0, be = 0;  // (and the decays and write strengths of head h0 + wave, lane = position)
  double gc;
  {
    u32x4 raw[2][NB][TY == LXM_FP32 ? 2 : 1] = {};
    if (row < n) {
      const T* kp = (const T*)io.k + (t0 + row) * io.k_ts + kh * io.k_hs + 8 * g;
      const T* qp = (const T*)io.q + (t0 + row) * io.q_ts + kh * io.q_hs + 8 * g;
#pragma unroll
      for (int i = 0; i < NB; i++) {
        raw[0][i][0] = *(const u32x4*)(kp + 32 * i);
        raw[1][i][0] = *(const u32x4*)(qp + 32 * i);
        if constexpr (TY == LXM_FP32) {
          raw[0][i][1] = *(const u32x4*)(kp + 32 * i + 4);
          raw[1][i][1] = *(const u32x4*)(qp + 32 * i + 4);
        }
      }
    }
    if (wave < nh && lane < n) {
      const int h = kh * io.r + h0 + wave;
      gx = io.g[(t0 + lane) * io.g_ts + h * io.g_hs];
      be = up_of(io.beta, (t0 + lane) * io.b_ts + h * io.b_hs, io.beta_type);
    }
    gc = wave_scan((double)(gx < kLow ? kLow : gx) * 1.4426950408889634);
    float sq[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < 2; w++)
#pragma unroll
      for (int i = 0; i < NB; i++) {
        float x[8];
        unpack<TY>(raw[w][i][0], x);
        if constexpr (TY == LXM_FP32) unpack<TY>(raw[w][i][1], x + 4);
#pragma unroll
        for (int j = 0; j < 8; j++) sq[w] = fma(x[j], x[j], sq[w]);
        u32x4* f = w ? qf[i] : kf[i];
        if constexpr (TY == LXM_BF16) f[0] = raw[w][i][0];
        else parts<8, NP>(x, (uint32_t(*)[4])f);
      }
#pragma unroll
    for (int w = 0; w < 2; w++) sq[w] += __shfl_xor(sq[w], 16), sq[w] += __shfl_xor(sq[w], 32);
    rq = io.unit ? io.scale / sqrtf(sq[1] + 1e-6f) : io.scale;
    if (g == 0) m.rk[row] = io.unit ? 1 / sqrtf(sq[0] + 1e-6f) : 1.f, m.rq[row] = rq;
  }
#pragma unroll
  for (int i = 0; i < NB; i++)
#pragma unroll
    for (int s = 0; s < NP; s++) {
      const int at = ((wave * NB + i) * NP + s) * kFrag + lane * 16;
      if (h0 == 0) {
        *(u32x4*)(wk + at) = qf[i][s];
        *(u32x4*)(wk + 64 * K * 2 * NP + at) = kf[i][s];
      }
      *(u32x4*)&kt[(s * 64 + row) * RS + 32 * i + 8 * g] = kf[i][s];
    }
  __syncthreads();
  const float rk = m.rk[row];
  float kk[2][8], qk[2][8];  // with keys 32 p + 8 g + j
#pragma unroll
  for (int p = 0; p < 2; p++)
#pragma unroll
    for (int half = 0; half < 2; half++) {
      f32x4 x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
      if (2 * p <= wave) {
        const int key = 32 * p + 8 * (c >> 2) + 4 * half + (c & 3);
#pragma unroll
        for (int i = 0; i < NB; i++) {
          u32x4 f[NP];
#pragma unroll
          for (int s = 0; s < NP; s++) f[s] = *(const u32x4*)&kt[(s * 64 + key) * RS + 32 * i + 8 * g];
          x = product<NP, NP>(f, kf[i], x);
          y = product<NP, NP>(f, qf[i], y);
        }
        settle(x);
        settle(y);
      }
#pragma unroll
      for (int r = 0; r < 4; r++) kk[p][4 * half + r] = x[r], qk[p][4 * half + r] = y[r];
    }
  // the keys transposed
  if (h0 == 0) {
#pragma unroll
    for (int u = 0; u < K / 32; u++) {
      const int f = 4 * u + wave, dim = f / 2 * 16 + c, pos = f % 2 * 32 + 8 * g;
#pragma unroll
      for (int s = 0; s < NP; s++) {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++)
          v[j] = kt[(s * 64 + pos + 2 * j) * RS + dim] | (uint32_t)kt[(s * 64 + pos + 2 * j + 1) * RS + dim] << 16;
        *(u32x4*)(wk + 2 * 64 * K * 2 * NP + (f * NP + s) * kFrag + lane * 16) = v;
      }
    }
  }

  if (wave < nh) {  // a head's factors
    const double last = __shfl(gc, 63);  // (positions past n add nothing)
    m.gc[wave][lane] = gc;
    m.beta[wave][lane] = be;
    float* fac = (float*)(wh + wave * (int64_t)kHeadWs + 6 * (3 + 3) * kFrag);
    const float e = __builtin_amdgcn_exp2f((float)gc), kr = m.rk[lane];
    fac[lane] = be;
    fac[64 + lane] = be * e * kr;
    fac[128 + lane] = e * m.rq[lane];
    fac[192 + lane] = lane < n ? __builtin_amdgcn_exp2f((float)(last - gc)) * kr : 0.f;
    if (lane == 0) fac[256] = __builtin_amdgcn_exp2f((float)last);
  }
  __syncthreads();  // (and the keys in LDS are read)
  for (int h = 0; h < nh; h++) {
    float* l = mat + h * (64 * kLd);
    const double gi = m.gc[h][row];
    const float bi = m.beta[h][row] * rk;
    char* to = wh + h * (int64_t)kHeadWs + 6 * 3 * kFrag + lane * 16;
    double gk[2][8];
    float rkey[2][8];
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int j = 0; j < 8; j++) gk[p][j] = m.gc[h][32 * p + 8 * g + j], rkey[p][j] = m.rk[32 * p + 8 * g + j];
#pragma unroll
    for (int p = 0; p < 2; p++) {
      if (2 * p > wave) continue;
      f32x4 lo[2];
      float x[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {  // (past the row's end e may overflow: selected, not multiplied)
        const int key = 32 * p + 8 * g + j;
        const float e = __builtin_amdgcn_exp2f((float)(gi - gk[p][j])) * rkey[p][j];
        const float a = bi * kk[p][j] * e, b = rq * qk[p][j] * e;
        lo[j / 4][j % 4] = key < row ? a : 0.f;
        x[j] = key <= row ? b : 0.f;
      }
      *(f32x4*)&l[row * kLd + 32 * p + 8 * g] = lo[0];
      *(f32x4*)&l[row * kLd + 32 * p + 8 * g + 4] = lo[1];
      u32x4 f[3];
      parts<8, 3>(x, (uint32_t(*)[4])f);
#pragma unroll
      for (int s = 0; s < 3; s++) *(u32x4*)(to + (block_of(wave, p) * 3 + s) * kFrag) = f[s];
    }
  }
  __syncthreads();
  if (wave < nh) invert(mat + wave * (64 * kLd), lane);
  __syncthreads();
  for (int u = wave; u < 6 * nh; u += 4) {
    const int h = u / 6, e = u % 6, tile = e < 2 ? e : (e + 2) / 2, p = e < 2 ? 0 : e & 1;
    char* to = wh + h * (int64_t)kHeadWs + lane * 16;
    const f32x4* src = (const f32x4*)(mat + h * (64 * kLd) + (tile * 16 + c) * kLd + 32 * p + 8 * g);
    const f32x4 x0 = src[0], x1 = src[1];
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; j++) x[j] = 2 * p + g / 2 <= tile ? (j < 4 ? x0 : x1)[j % 4] : 0.f;
    u32x4 f[3];
    parts<8, 3>(x, (uint32_t(*)[4])f);
#pragma unroll
    for (int s = 0; s < 3; s++) *(u32x4*)(to + (e * 3 + s) * kFrag) = f[s];
  }
}

// A chunk's chain, in 3 steps with a barrier each: the state's parts to R (S^T k), R to D (T R), D to the state.
// One workgroup of 8 waves per (sequence, value head, NC blocks of 16 state columns); right operands (the state, R,
// D) cross the waves through LDS as parts. Waves 0 to 3 have a row tile of R and of D, which is the chain; waves
// 4 to 7 one of the output, a step behind (S^T q while D is formed, A D in the next chunk's first step); all of
// them their tiles of the state. What a chunk reads from memory is requested a chunk ahead, each register
// again as soon as it has been used: nothing in the chain waits for memory. A chunk takes 1.7 us (3,500 cycles, of
// which the MFMAs are 1,090 a SIMD): the parts' way through LDS (192 KB read), the operands' through the CU's vector
// memory path (90 KB) and the barriers between them. In fp32 matrix instructions it took 5.6.
template <int TY, int K, int NC>
struct Run {
  typedef typename Elem<TY>::T T;
  static constexpr int NP = kParts<TY>, NB = K / 32, NT = K < 128 ? 1 : K / 128;
  struct Lds {
    u32x4 s[NC][NB][3][64], r[NC][2][3][64], d[NC][2][3][64], e[NC][2][3][64];
  };
  const lxm_gd_io& io;
  Lds& m;
  int lane, w, g, c, tile0;  // w: the wave's row tile; tile0: its first tile of the state
  bool writes;
  const char *wk, *wh;  // the chunk's operands, of this key head and this value head
  f32x4 s[NC][NT];
  u32x4 xf[NT][2][NP];
  float eg;

  __device__ u32x4 frag(const char* base, int i) const { return *(const u32x4*)(base + i * kFrag + (uint32_t)(lane * 16)); }
  __device__ const char* factors() const { return wh + 6 * (3 + 3) * kFrag; }
  // a D tile (rows 4 g + r of tile t) as part of a right operand of blocks of 32 rows
  __device__ void put(u32x4 (*d)[64], f32x4 v, int t) const {
    uint32_t p[3][2];
    float y[4] = {v[0], v[1], v[2], v[3]};
    parts<4, 3>(y, p);
#pragma unroll
    for (int i = 0; i < 3; i++)
      *(u32x2*)((char*)&d[i][c + 16 * (2 * (t & 1) + g / 2)] + 8 * (g & 1)) = u32x2{p[i][0], p[i][1]};
  }
  __device__ void put_state() const {
    if (writes) {
#pragma unroll
      for (int n = 0; n < NC; n++)
#pragma unroll
        for (int t = 0; t < NT; t++) put(m.s[n][(tile0 + t) / 2], s[n][t], tile0 + t);
    }
  }
  // one row tile of a left operand over the K dims
  __device__ void load_rows(u32x4 (*f)[NP], const char* base) const {
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
      for (int e = 0; e < NP; e++) f[i][e] = frag(base, (w * NB + i) * NP + e);
  }
  // one row tile of a triangular left operand (row tiles 0 and 1 have no second block: it stays zero)
  __device__ void load_tri(u32x4 (*f)[3], const char* base) const {
#pragma unroll
    for (int p = 0; p < 2; p++)
      if (p == 0 || w >= 2) {
#pragma unroll
        for (int e = 0; e < 3; e++) f[p][e] = frag(base, block_of(w, p) * 3 + e);
      }
  }
  __device__ void load_x() {
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int p = 0; p < 2; p++)
#pragma unroll
        for (int e = 0; e < NP; e++) xf[t][p][e] = frag(wk + 2 * 64 * K * 2 * NP, ((tile0 + t) * 2 + p) * NP + e);
    eg = ((const float*)factors())[256];
  }
  __device__ f32x4 factor(int i) const { return *(const f32x4*)(factors() + 256 * i + 64 * w + (uint32_t)(16 * g)); }
  __device__ void operand(u32x4 (*f)[3], const u32x4 (*from)[3][64]) const {  // a right operand's two blocks
#pragma unroll
    for (int p = 0; p < 2; p++)
#pragma unroll
      for (int e = 0; e < 3; e++) f[p][e] = from[p][e][lane];
    issued();
  }
  // S <- decay S + sum_i k_i e_i^T, the sum by itself and then one fma: added to the state part by part it would round
  // the state each time; then (wk, wh: the next chunk's) what the next needs for it
  __device__ void step_state() {
#pragma unroll
    for (int n = 0; n < NC; n++) {
      u32x4 ef[2][3];
      operand(ef, m.e[n]);
      f32x4 a[NT] = {};
#pragma unroll
      for (int p = 0; p < 2; p++)
#pragma unroll
        for (int t = 0; t < NT; t++) a[t] = product<NP, 3>(xf[t][p], ef[p], a[t]);
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) s[n][t][r] = fma(eg, s[n][t][r], a[t][r]);
    }
    put_state();
    load_x();
  }
  template <int AT>  // blocks of the state in registers at a time
  __device__ f32x4 times_state(const u32x4 (*f)[NP], int n) const {
    f32x4 a[2] = {};
#pragma unroll
    for (int i0 = 0; i0 < NB; i0 += AT) {
      u32x4 sf[AT][3];
#pragma unroll
      for (int i = 0; i < AT; i++)
#pragma unroll
        for (int e = 0; e < 3; e++) sf[i][e] = m.s[n][i0 + i][e][lane];
      issued();
#pragma unroll
      for (int i = 0; i < AT; i++) a[i & 1] = product<NP, 3>(f[i0 + i], sf[i], a[i & 1]);
    }
    return a[0] + a[1];
  }

  // waves 0 to 3; t0: the chunk's first position
  __device__ void solve(int chunks, int64_t kstep, int64_t hstep, int t0, int end, const T* vp) {
    u32x4 kf[NB][NP], tf[2][3] = {};
    f32x4 be, ck, cd;
    T v[NC][4];
    const int64_t ts = io.v_ts;
    const int row = w * 16 + 4 * g;
    __builtin_amdgcn_s_setprio(2);  // (the chain's waves before the output's: prompt of 16,384 553.8 -> 551.7 us)
    vp += (t0 + row) * ts;
    auto load_v = [&] {
      if (t0 + LXM_SEQ_CHUNK <= end) {
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
          for (int r = 0; r < 4; r++) v[n][r] = vp[r * ts + 16 * n];
      } else {
#pragma unroll
        for (int n = 0; n < NC; n++)
#pragma unroll
          for (int r = 0; r < 4; r++) {
            v[n][r] = 0;
            if (t0 + row + r < end) v[n][r] = vp[r * ts + 16 * n];
          }
      }
      be = factor(0), ck = factor(1);
    };
    load_rows(kf, wk + 64 * K * 2 * NP), load_v(), load_tri(tf, wh), cd = factor(3), load_x();
    put_state();
    for (int a = 0; a < chunks; a++) {
      const bool more = a + 1 < chunks;
      if (more) wk += kstep, wh += hstep;
      lds_barrier();
      f32x4 ks[NC];
#pragma unroll
      for (int n = 0; n < NC; n++) ks[n] = times_state<NB>(kf, n);
      load_rows(kf, wk + 64 * K * 2 * NP);
#pragma unroll
      for (int n = 0; n < NC; n++) {
        f32x4 R;
#pragma unroll
        for (int r = 0; r < 4; r++) R[r] = fma(-ck[r], ks[n][r], be[r] * up<TY>(v[n][r]));
        put(m.r[n][w / 2], R, w);
      }
      if (more) t0 += LXM_SEQ_CHUNK, vp += LXM_SEQ_CHUNK * ts;
      load_v();
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NC; n++) {
        u32x4 rf[2][3];
        operand(rf, m.r[n]);
        f32x4 d = {0, 0, 0, 0}, d1 = {0, 0, 0, 0};
        d = product<3, 3>(tf[0], rf[0], d);
        d1 = product<3, 3>(tf[1], rf[1], d1);
        d += d1;
        put(m.e[n][w / 2], d * cd, w);
        put(m.d[n][w / 2], d, w);
      }
      load_tri(tf, wh), cd = factor(3);
      lds_barrier();
      step_state();
    }
    lds_barrier();
  }

  // waves 4 to 7
  __device__ void output(int chunks, int64_t kstep, int64_t hstep, int t0, int end, T* op) {
    u32x4 qf[NB][NP], af[2][3] = {};
    f32x4 cq, o[NC] = {};
    const int64_t ts = io.o_ts;
    const int row = w * 16 + 4 * g;
    op += (t0 + row) * ts;
    auto finish = [&] {  // o of the chunk before
#pragma unroll
      for (int n = 0; n < NC; n++) {
        u32x4 df[2][3];
        operand(df, m.d[n]);
#pragma unroll
        for (int p = 0; p < 2; p++) o[n] = product<3, 3>(af[p], df[p], o[n]);
        if (t0 + LXM_SEQ_CHUNK <= end) {
#pragma unroll
          for (int r = 0; r < 4; r++) op[r * ts + 16 * n] = down<TY>(o[n][r]);
        } else {
#pragma unroll
          for (int r = 0; r < 4; r++)
            if (t0 + row + r < end) op[r * ts + 16 * n] = down<TY>(o[n][r]);
        }
      }
      t0 += LXM_SEQ_CHUNK, op += LXM_SEQ_CHUNK * ts;
    };
    load_rows(qf, wk), cq = factor(2), load_tri(af, wh + 6 * 3 * kFrag), load_x();
    put_state();
    for (int a = 0; a < chunks; a++) {
      const char* wa = wh;
      if (a + 1 < chunks) wk += kstep, wh += hstep;
      lds_barrier();
      if (a > 0) {
        finish();
        load_tri(af, wa + 6 * 3 * kFrag);
      }
      lds_barrier();
#pragma unroll
      for (int n = 0; n < NC; n++) o[n] = times_state<NB / 2>(qf, n) * cq;
      load_rows(qf, wk), cq = factor(2);
      lds_barrier();
      step_state();
    }
    lds_barrier();
    finish();
  }
};

// (Four waves a SIMD where the registers allow it, two workgroups a CU: 24 ragged prompts of bf16 118 us, 139 with
// 136 registers and one workgroup.)
template <int TY, int K, int NC>
__global__ __launch_bounds__(512, TY == LXM_BF16 && K <= 128 ? 4 : 2) void gd_run(lxm_seq_table S, lxm_gd_io io, const char* ws, int c0, int n_chunks,
                                              const float* carry, float* carry_to) {
  typedef typename Elem<TY>::T T;
  typedef Run<TY, K, NC> R;
  __shared__ typename R::Lds lds;
  const int nv = io.nk * io.r, ncb = io.V / (16 * NC), per = (nv + 7) / 8;
  // a head's column blocks on one XCD (workgroups are dealt to the 8 in turn), neighbouring heads beside them
  const int x = blockIdx.x % (8 * per * ncb), h = x % 8 * per + x / 8 / ncb, cb = x / 8 % ncb;
  if (h >= nv) return;
  const Seq seq = seq_at(S, blockIdx.x / (8 * per * ncb));
  const int slot = seq.slot, first = seq.first, end = seq.end;
  const int f0 = seq.chunk, f1 = f0 + (end - first + LXM_SEQ_CHUNK - 1) / LXM_SEQ_CHUNK;
  const int a0 = max(f0, c0), a1 = min(f1, c0 + n_chunks);
  if (a0 >= a1) return;
  const int lane = threadIdx.x & 63, wave = wave_of(), g = lane >> 4, c = lane & 15, w = wave & 3;

  const int64_t kstep = (int64_t)io.nk * kKeyWs<TY, K>, hstep = (int64_t)nv * kHeadWs;
  R run{io, lds, lane, w, g, c, K < 128 ? w : wave * R::NT, K >= 128 || wave < 4,
        ws + (h / io.r) * (int64_t)kKeyWs<TY, K> + (a0 - c0) * kstep,
        ws + n_chunks * kstep + (a0 - c0) * hstep + h * (int64_t)kHeadWs};
  const bool from = slot >= 0 || a0 > f0, to = slot >= 0 || a1 < f1;
  const int col = cb * 16 * NC + c;
  // (a sequence without a slot that goes on in another group of chunks: from the last launch's carry to the next's, of
  // which each has at most one)
  float* slot_state = io.state + (int64_t)slot * io.s_ss;
  const int64_t at = (int64_t)h * K * io.V + col;
  const float* sp = (slot >= 0 ? slot_state : carry) + at;
#pragma unroll
  for (int n = 0; n < NC; n++)
#pragma unroll
    for (int t = 0; t < R::NT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++)
        run.s[n][t][r] = from ? sp[((run.tile0 + t) * 16 + 4 * g + r) * io.V + 16 * n] : 0.f;
  const int t0 = first + (a0 - f0) * LXM_SEQ_CHUNK;
  if (wave < 4) run.solve(a1 - a0, kstep, hstep, t0, end, (const T*)io.v + h * io.v_hs + col);
  else run.output(a1 - a0, kstep, hstep, t0, end, (T*)io.o + h * io.o_hs + col);
  float* dp = (slot >= 0 ? slot_state : carry_to) + at;
  if (to && run.writes) {
#pragma unroll
    for (int n = 0; n < NC; n++)
#pragma unroll
      for (int t = 0; t < R::NT; t++)
#pragma unroll
        for (int r = 0; r < 4; r++) dp[((run.tile0 + t) * 16 + 4 * g + r) * io.V + 16 * n] = run.s[n][t][r];
  }
}

// ---- host ---------------------------------------------------------------------------------------------
// workgroups of a launch at most: its threads are counted in 32 bits
constexpr int64_t most(int threads) { return 0xffffffffll / threads; }

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

bool bad_table(const lxm_seq_table* s) {
  return !s || s->n_seqs < 0 || s->n_tokens < 0 || s->n_chunks < 0 || s->max_len < 0 ||
         (s->n_seqs && (!s->seqs || !aligned(s->seqs))) || (s->n_chunks && (!s->chunks || !aligned(s->chunks)));
}

bool bad_shape(const lxm_gd_io* io) {
  return !io || io->nk < 1 || io->r < 1 || (int64_t)io->nk * io->r > 65536 || (io->K != 64 && io->K != 128 && io->K != 256) || io->V < 16 ||
         io->V > 256 || io->V % 16 || io->type < 0 || io->type > 2;
}

bool bad_io(const lxm_gd_io* io) {
  if (bad_shape(io) || io->beta_type < 0 || io->beta_type > 2) return true;
  const int64_t vec = io->type == LXM_FP32 ? 4 : 8;
  return !io->q || !io->k || !io->v || !io->g || !io->beta || !io->state || !io->o || !aligned(io->q) ||
         !aligned(io->k) || !aligned(io->v) || !aligned(io->state) || !aligned(io->o) || io->q_ts % vec || io->q_hs % vec ||
         io->k_ts % vec || io->k_hs % vec || io->v_ts % vec || io->v_hs % vec || io->o_ts % vec || io->o_hs % vec ||
         io->s_ss % 4;
}

template <int TY, int K>
int recurrent(const lxm_seq_table* s, const lxm_gd_io* io, hipStream_t st) {
  const int64_t heads = (int64_t)s->n_seqs * io->nk * io->r;
  // columns a workgroup: as many as leave 2 workgroups a CU, so that a small batch is spread over the card and a large
  // one reads whole rows. 128 x 128: 8 positions of 8 sequences of 32 heads 16.8 us in 64 columns, 17.9 in 128, 23.7
  // in 16; one token of 64 sequences 39.5 in 128, 64.9 in 16.
  int cb = 128;
  while (cb > 16 && (io->V % cb || heads * (io->V / cb) < 512)) cb /= 2;
  const int each = io->nk * io->r * (io->V / cb), step = (int)(most(256) / each);  // (each <= 2^20: bad_io)
  lxm_seq_table t = *s;
  for (int left = s->n_seqs; left > 0; left -= step, t.seqs += 4 * (int64_t)step) {
    const int grid = (left < step ? left : step) * each;
    if (cb == 128) gd_recurrent<TY, K, 128><<<grid, 256, 0, st>>>(t, *io);
    else if (cb == 64) gd_recurrent<TY, K, 64><<<grid, 256, 0, st>>>(t, *io);
    else if (cb == 32) gd_recurrent<TY, K, 32><<<grid, 256, 0, st>>>(t, *io);
    else gd_recurrent<TY, K, 16><<<grid, 256, 0, st>>>(t, *io);
    if (int e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

constexpr int64_t kTwo = 350;

template <int TY, int K>
int chunks(const lxm_seq_table* s, const lxm_gd_io* io, char* ws, int64_t ws_bytes, hipStream_t st) {
  const int nv = io->nk * io->r, per = (nv + 7) / 8, preps = io->nk * ((io->r + 3) / 4);
  const int64_t carry = 2 * (int64_t)nv * K * io->V * 4, each = (int64_t)io->nk * kKeyWs<TY, K> + (int64_t)nv * kHeadWs;
  if (ws_bytes < carry + each) return hipErrorInvalidValue;
  int64_t group = (ws_bytes - carry) / each;
  if (group > s->n_chunks) group = s->n_chunks;
  if (group > most(256) / preps) group = most(256) / preps;
  // Two column blocks a workgroup share its left operands, one has the shorter chain: two where, over the time of the
  // longest sequence's chain, that many workgroups of one block would be at work on average. 128 x 128, one against
  // two: a prompt of 2,048 in 32 heads (256 at work) 68 us against 92, in 40 (320) 94 and 95, in 48 (384) 107
  // and 104, in 64 127 and 118, in 128 254 and 216, in fp32 48 heads 224 and 181; 24 ragged prompts (1,300) 144 and
  // 119, in fp32 306 and 240; fp32 with 256 x 128, where two spill 12 registers, 225 and 192.
  const int64_t chain = (s->max_len + LXM_SEQ_CHUNK - 1) / LXM_SEQ_CHUNK;
  const bool two = io->V % 32 == 0 && s->n_chunks * (int64_t)nv * (io->V / 16) >= kTwo * chain;
  const int runs = 8 * per * (io->V / (two ? 32 : 16)), step = (int)(most(512) / runs);  // (of a sequence; runs <= 2^20)
  const int mats = (io->r < 4 ? io->r : 4) * kMat;
  const int lds = (int)sizeof(PrepLds) + (mats > kStage<TY, K> ? mats : kStage<TY, K>);
  // (on every call: the attribute is the current device's)
  if (lds > 65536)
    if (int e = hipFuncSetAttribute((const void*)gd_prep<TY, K>, hipFuncAttributeMaxDynamicSharedMemorySize, lds)) return e;
  float* carries[2] = {(float*)ws, (float*)(ws + carry / 2)};
  for (int64_t c0 = 0, turn = 0; c0 < s->n_chunks; c0 += group, turn = !turn) {
    const int n = (int)(s->n_chunks - c0 < group ? s->n_chunks - c0 : group);
    gd_prep<TY, K><<<n * preps, 256, lds, st>>>(*s, *io, ws + carry, (int)c0);
    if (int e = hipGetLastError()) return e;
    lxm_seq_table t = *s;
    for (int left = s->n_seqs; left > 0; left -= step, t.seqs += 4 * (int64_t)step) {
      const int grid = (left < step ? left : step) * runs;
      if (two) gd_run<TY, K, 2><<<grid, 512, 0, st>>>(t, *io, ws + carry, (int)c0, n, carries[turn], carries[!turn]);
      else gd_run<TY, K, 1><<<grid, 512, 0, st>>>(t, *io, ws + carry, (int)c0, n, carries[turn], carries[!turn]);
      if (int e = hipGetLastError()) return e;
    }
  }
  return hipSuccess;
}

template <int TY>
int conv(const lxm_seq_table* s, const lxm_conv_io* io, hipStream_t st) {
  const int vec = kVec<TY>, runs = (min(s->max_len, LXM_SEQ_CHUNK) + kRun - 1) / kRun;
  const bool wide = io->C % vec == 0 && io->x_ts % vec == 0 && io->y_ts % vec == 0 && io->w_ss % vec == 0 && aligned(io->x) &&
                    aligned(io->y) && aligned(io->w) && aligned(io->window);
  const int64_t cols = 256 * (wide ? vec : 1), cblocks = (io->C + cols - 1) / cols, each = cblocks * runs;
  if (each > most(256) || cblocks * cols > 0x7fffffff) return hipErrorInvalidValue;
  const int step = (int)(most(256) / each);
  lxm_seq_table t = *s;
  for (int left = s->n_chunks; left > 0; left -= step, t.chunks += 4 * (int64_t)step) {
    const int grid = (int)((left < step ? left : step) * each);
    if (wide) short_conv<TY, kVec<TY>><<<grid, 256, 0, st>>>(t, *io, runs, (int)cblocks);
    else short_conv<TY, 1><<<grid, 256, 0, st>>>(t, *io, runs, (int)cblocks);
    if (int e = hipGetLastError()) return e;
  }
  return hipSuccess;
}

#define BY_TYPE(ty, f, ...)                                  \
  ((ty) == LXM_BF16 ? f<LXM_BF16>(__VA_ARGS__)               \
   : (ty) == LXM_FP16 ? f<LXM_FP16>(__VA_ARGS__) : f<LXM_FP32>(__VA_ARGS__))

template <int TY>
int recurrent_k(const lxm_seq_table* s, const lxm_gd_io* io, hipStream_t st) {
  return io->K == 64 ? recurrent<TY, 64>(s, io, st) : io->K == 128 ? recurrent<TY, 128>(s, io, st) : recurrent<TY, 256>(s, io, st);
}
template <int TY>
int chunks_k(const lxm_seq_table* s, const lxm_gd_io* io, char* ws, int64_t n, hipStream_t st) {
  return io->K == 64 ? chunks<TY, 64>(s, io, ws, n, st) : io->K == 128 ? chunks<TY, 128>(s, io, ws, n, st) : chunks<TY, 256>(s, io, ws, n, st);
}
template <int TY>
int64_t ws_of(const lxm_gd_io* io, int64_t n) {
  const int64_t nv = (int64_t)io->nk * io->r;
  const int64_t key = io->K == 64 ? kKeyWs<TY, 64> : io->K == 128 ? kKeyWs<TY, 128> : kKeyWs<TY, 256>;
  return 2 * nv * io->K * io->V * 4 + n * (io->nk * key + nv * kHeadWs);
}

}  // namespace

extern "C" int lxm_short_conv(const lxm_seq_table* s, const lxm_conv_io* io, void* stream) {
  if (bad_table(s) || !io || io->C < 1 || io->type < 0 || io->type > 2 || !io->w || !io->window) return hipErrorInvalidValue;
  if (s->n_tokens == 0) return hipSuccess;
  if (!io->x || !io->y || s->n_chunks < 1 || s->max_len < 1) return hipErrorInvalidValue;
  return BY_TYPE(io->type, conv, s, io, (hipStream_t)stream);
}

extern "C" int lxm_gd_recurrent(const lxm_seq_table* s, const lxm_gd_io* io, void* stream) {
  if (bad_table(s)) return hipErrorInvalidValue;
  if (s->n_tokens == 0) return hipSuccess;
  if (bad_io(io)) return hipErrorInvalidValue;
  return BY_TYPE(io->type, recurrent_k, s, io, (hipStream_t)stream);
}

extern "C" int lxm_gd_ws(const lxm_gd_io* io, int32_t n_chunks, int64_t* bytes) {
  if (bad_shape(io) || !bytes || n_chunks < 1) return hipErrorInvalidValue;
  *bytes = BY_TYPE(io->type, ws_of, io, n_chunks);
  return hipSuccess;
}

extern "C" int lxm_gd_chunks(const lxm_seq_table* s, const lxm_gd_io* io, void* ws, int64_t ws_bytes, void* stream) {
  if (bad_table(s)) return hipErrorInvalidValue;
  if (s->n_tokens == 0) return hipSuccess;
  if (bad_io(io) || !ws || !aligned(ws) || s->n_chunks < 1) return hipErrorInvalidValue;
  return BY_TYPE(io->type, chunks_k, s, io, (char*)ws, ws_bytes, (hipStream_t)stream);
}
