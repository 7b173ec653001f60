// Log probabilities of given tokens with each row's entropy, the token's rank and the best alternatives
// (include/lxm_score.h), in one pass over the logits.
//
// With m a row's maximum, s = sum exp(x - m) and w = sum exp(x - m) (x - m):
//   lse = m + log s,  logprob = (x_t - m) - log s,  entropy = log s - w / s
// (w rather than sum p x: no large numbers cancel). A thread keeps its own m, s and w, moved to a new maximum
// once per kEach elements: s' = f s, w' = f (w + s (m - m')), f = exp(m - m'). A block's kEach terms are summed by
// themselves and then added to s and w with what that rounds off kept beside them: a row's sums are as good as a
// block's, however long it is and where equal terms round the same way each time.
//
// The alternatives: a wave walks its part of the row in blocks of 64 x kEach elements with a list of the best in LDS,
// and no barrier. Where a block has more of use than `top`, a bound that `top` lanes' maxima reach cuts it first.
// A later block's element comes after all before it among equals (its token is higher), so it matters only if it
// is greater than what `top` elements have: one comparison of the lane's maximum, which the softmax needs anyway.
// When the list is nearly full its best `top` are kept, sorted, and the gate rises. Everything is ordered by
// one 64-bit key (value, lower token).
//
// The rank: a token's own logit is compared with every element, from the float below it for lower tokens (equals count
// there); where a block's maximum is below it nothing is.
//
// Bytes bound many rows: 2,048 rows of 248,320 bf16 logits, top 8, 212 us, 4.8 TB/s (193 with no alternatives; a list
// for the workgroup, a barrier a block, took 518). Few rows are split over parts (a workgroup each), joined by a
// second kernel, and bound by the two kernels' latency: one row of 459,982, 7.9 and 7.1 us.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/lxm_score.h"

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned long long u64;

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kList = 128;  // keys a wave's list holds; 64 can come at once
static_assert(LXM_SCORE_TOP == 64 && kThreads == 4 * LXM_SCORE_TOP, "a lane a key");
constexpr float kInf = __builtin_inff(), kLog2e = 1.44269504f;

template <int TY>
struct Elem {
  typedef uint16_t T;
};
template <>
struct Elem<2> {
  typedef float T;
};
template <int TY>
__device__ __forceinline__ float up(typename Elem<TY>::T x) {
  if constexpr (TY == 0) return __uint_as_float((uint32_t)x << 16);
  else if constexpr (TY == 1) return (float)__builtin_bit_cast(_Float16, x);
  else return x;
}

// (value, token) as one number: larger values first, then lower tokens; NaN above all; 0 is no element. 32 bits of the
// value's order and 31 of the token below a clear sign, with the exponent's bits never all set: as doubles such
// patterns have the order of the integers, and a double's comparison takes one pass where a 64-bit integer's
// takes four.
__device__ __forceinline__ uint32_t order_of(float x) {  // the value's part
  const uint32_t b = __float_as_uint(x + 0.f);
  return x != x ? 0xffc00000u : b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ double key_of(uint32_t order, uint32_t token) {
  return __builtin_bit_cast(double, (u64)order << 31 | (0x7fffffffu - token));
}
__device__ __forceinline__ double key_of(float x, uint32_t token) { return key_of(order_of(x), token); }
__device__ __forceinline__ float value_of(uint32_t o) {
  return __uint_as_float(o >= 0xffc00000u ? 0x7fc00000u : o >> 31 ? o & 0x7fffffffu : ~o);
}
__device__ __forceinline__ float value_of(double key) { return value_of((uint32_t)(__builtin_bit_cast(u64, key) >> 31)); }
__device__ __forceinline__ int token_of(double key) { return (int)(0x7fffffffu - (uint32_t)(__builtin_bit_cast(u64, key) & 0x7fffffffu)); }

struct Lds {
  __attribute__((aligned(16))) double list[kWaves][kList + 8];
  __attribute__((aligned(16))) double all[kThreads + 8];  // the waves' best, and the workgroup's
  int n[kWaves];
  float m[kWaves], s[kWaves], w[kWaves];
  int c[kWaves];
};

// what this wave's lanes stored in LDS, for its other lanes (a wave's LDS accesses run in order)
__device__ __forceinline__ void wave_sync() {
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  __builtin_amdgcn_wave_barrier();
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
}

// r[i] += how many of buf[0 .. c - 1] (zeros behind, up to a multiple of 8) are greater than k[i]
template <int N>
__device__ __forceinline__ void greater(const double* buf, int c, const double* k, int* r) {
  typedef double f64x2 __attribute__((ext_vector_type(2)));
#pragma unroll 1
  for (int i = 0; i < c; i += 8) {
    f64x2 q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) q[j] = *(const f64x2*)(buf + i + 2 * j);
#pragma unroll
    for (int j = 0; j < 4; j++)
#pragma unroll
      for (int e = 0; e < N; e++) r[e] += (q[j].x > k[e]) + (q[j].y > k[e]);
  }
}

// A wave's list: its best `top` of n, sorted; returns how many.
__device__ __forceinline__ int cut(double* list, int n, int top) {
  constexpr int N = kList / 64;
  const int lane = threadIdx.x & 63;
  wave_sync();
  if (lane < 8) list[n + lane] = 0;
  wave_sync();
  double k[N];
  int r[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    const bool is = 64 * i + lane < n;
    k[i] = is ? list[64 * i + lane] : 0, r[i] = is ? 0 : top;
  }
  greater<N>(list, n, k, r);
  wave_sync();
#pragma unroll
  for (int i = 0; i < N; i++)
    if (r[i] < top) list[r[i]] = k[i];
  wave_sync();
  return min(n, top);
}

// The lanes' keys (0: none) added to a wave's list of n (at most kList - 64); the list's length.
__device__ __forceinline__ int add(double* list, int n, double key) {
  const u64 have = __ballot(key != 0);
  const int at = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(have >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)have, 0));
  if (key != 0) list[at] = key;
  return n + __popcll(have);
}

// The waves' lists (n each, at most `top`) as one: l.all[0 ..] sorted, at most `top`.
__device__ void join_lists(Lds& l, int n, int top) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  if (lane == 0) l.n[wave] = n;
  __syncthreads();
  int at = 0, c = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    if (i < wave) at += l.n[i];
    c += l.n[i];
  }
  if (lane < n) l.all[at + lane] = l.list[wave][lane];
  if (tid < 8) l.all[c + tid] = 0;
  __syncthreads();
  const double k = tid < c ? l.all[tid] : 0;
  int r = tid < c ? 0 : top;
  greater<1>(l.all, c, &k, &r);
  __syncthreads();
  if (r < top) l.all[r] = k;
  __syncthreads();
}

// s and w moved up to a maximum d = old - new <= 0 away (old = -inf: nothing summed yet, s = w = 0, and d may be
// NaN). Past -200 exp(d) is 0 in float32, and s d may overflow.
__device__ __forceinline__ void move(float& s, float& w, float d) {
  d = fmaxf(d, -200.f);
  const float f = __builtin_amdgcn_exp2f(d * kLog2e);
  w = f * __builtin_fmaf(s, d, w);
  s *= f;
}
// s += x, what the addition rounds off added to l
__device__ __forceinline__ void add_up(float& s, float& l, float x) {
  const float t = s + x;
  l += x - (t - s);
  s = t;
}
// a wave's sums and maximum, in every lane (DPP: row shifts within 16 lanes, then the rows' last lanes)
template <int CTRL, int ROWS, class T>
__device__ __forceinline__ T dpp(T x, T rest) {
  return __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, rest), __builtin_bit_cast(int, x), CTRL, ROWS, 0xf, false));
}
template <class T, class Op>
__device__ __forceinline__ T wave_all(T x, T none, Op op) {
  x = op(x, dpp<0x111, 0xf>(x, none));
  x = op(x, dpp<0x112, 0xf>(x, none));
  x = op(x, dpp<0x114, 0xf>(x, none));
  x = op(x, dpp<0x118, 0xf>(x, none));
  x = op(x, dpp<0x142, 0xa>(x, none));
  x = op(x, dpp<0x143, 0xc>(x, none));
  return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}
template <class T>
__device__ __forceinline__ T wave_sum(T x) {
  return wave_all(x, T(0), [](T a, T b) { return a + b; });
}

// the workgroup's (m, s, w) and count
__device__ void join_all(Lds& l, float& m, float& s, float& w, int& c) {
  const float wm = wave_all(m, -kInf, [](float a, float b) { return fmaxf(a, b); });
  move(s, w, m - wm);
  const float ws = wave_sum(s), ww = wave_sum(w);
  const int wc = wave_sum(c), wave = threadIdx.x >> 6;
  if ((threadIdx.x & 63) == 0) l.m[wave] = wm, l.s[wave] = ws, l.w[wave] = ww, l.c[wave] = wc;
  __syncthreads();
  m = fmaxf(fmaxf(l.m[0], l.m[1]), fmaxf(l.m[2], l.m[3]));
  s = w = 0, c = 0;
#pragma unroll
  for (int i = 0; i < kWaves; i++) {
    float a = l.s[i], b = l.w[i];
    move(a, b, l.m[i] - m);
    s += a, w += b, c += l.c[i];
  }
}

__device__ __forceinline__ int64_t token_at(const lxm_score_io& io, int row) {
  return io.wide ? ((const int64_t*)io.tokens)[row] : (int64_t)((const int32_t*)io.tokens)[row];
}

// the row's results, by thread 0 (top: by the first threads)
__device__ void write_row(const lxm_score_io& io, const Lds& l, int row, float m, float s, float w, int c, float xt, int64_t t) {
  const float ls = logf(s);
  if (threadIdx.x == 0) {
    io.logprob[row] = t < 0 ? 0.f : t >= io.V ? __builtin_nanf("") : (xt - m) - ls;
    io.entropy[row] = ls - w / s;
    io.rank[row] = t < 0 || t >= io.V || xt != xt ? -1 : c;
  }
  if (threadIdx.x < io.top) {
    io.top_tokens[(int64_t)row * io.top + threadIdx.x] = token_of(l.all[threadIdx.x]);
    io.top_logprobs[(int64_t)row * io.top + threadIdx.x] = (value_of(l.all[threadIdx.x]) - m) - ls;
  }
}

struct Part {
  float m, s, w;
  int c;
};

// One workgroup per (row, part). Between the row's first and last 16-byte boundary a part is whole words, dealt to the
// waves 64 at a time, kEach elements a lane of a block; what the row has before and after (less than a word each) is
// a block of one element a lane, before the first and after the last of the row. (Waves a SIMD: 2,048 bf16 rows of
// 248,320 in 212 us with 5, 215 with 4; fp32 would spill 32 registers with 5, 1,200 rows of 150,001 in 223 us for 164.)
template <int TY, int kEach>
__global__ __launch_bounds__(kThreads, TY == 2 ? 4 : 5) void score_part(lxm_score_io io, int n_parts, int words_per_part, Part* parts, double* lists) {
  typedef typename Elem<TY>::T T;
  constexpr int kVec = 16 / sizeof(T), U = kEach / kVec, kStep = kThreads * U;
  constexpr uint32_t kAll = kEach == 32 ? 0xffffffffu : (1u << kEach % 32) - 1;
  __shared__ Lds l;
  const int row = blockIdx.x / n_parts, part = blockIdx.x % n_parts, tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const T* x = (const T*)io.logits + row * io.stride;
  const int V = io.V, top = io.top;
  const int head = min(V, (int)((0 - (uintptr_t)x / sizeof(T)) % kVec)), words = (V - head) / kVec, tail = head + words * kVec;
  const int j0 = min(words, part * words_per_part), j1 = min(words, j0 + words_per_part);
  const int64_t t = token_at(io, row);
  const u32x4* xw = (const u32x4*)(x + head);
  u32x4 q[U];
  auto request = [&](int j) {
#pragma unroll
    for (int u = 0; u < U; u++)
      if (j + u * kThreads + tid < j1) q[u] = xw[j + u * kThreads + tid];
  };
  request(j0);
  const bool ranked = t >= 0 && t < V;
  const float xt = ranked ? up<TY>(x[t]) : __builtin_nanf("");
  // what comes before the token: among lower tokens a logit of xt too (greater than the float below it)
  float below = xt;
  if (xt == 0) below = -__uint_as_float(1);
  else if (xt == xt && xt != -kInf) below = __uint_as_float(__float_as_uint(xt) + (xt > 0 ? -1 : 1));

  float m = -kInf, s = 0, w = 0, gate = -kInf;
  float ls = 0, lw = 0;  // what the additions to s and w have rounded off
  int c = 0, n = 0;
  double* list = l.list[wave];
  // -1: the elements before the words; -2: those behind
  for (int j = part == 0 && head > 0 ? -1 : j0 < j1 ? j0 : -2;;) {
    float v[kEach];
    uint32_t in;   // a bit for each element that the row has
    int e0, width;  // the lane's first token (word u's: e0 + u kThreads kVec), how many lie side by side
    if (j >= 0) {
      in = kAll, e0 = head + (j + tid) * kVec, width = kVec;
#pragma unroll
      for (int u = 0; u < U; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          if constexpr (TY == 2) v[u * 4 + i] = __uint_as_float(q[u][i]);
          else {
            v[u * 8 + 2 * i] = up<TY>((uint16_t)(q[u][i] & 0xffff));
            v[u * 8 + 2 * i + 1] = up<TY>((uint16_t)(q[u][i] >> 16));
          }
        }
      if (j + kStep > j1) {
#pragma unroll
        for (int u = 0; u < U; u++) {
          const bool is = j + u * kThreads + tid < j1;
          if (!is) in &= ~(((1ull << kVec) - 1) << (u * kVec));
#pragma unroll
          for (int i = 0; i < kVec; i++) v[u * kVec + i] = is ? v[u * kVec + i] : -kInf;
        }
      }
      request(j + kStep);
    } else {
      e0 = (j == -1 ? 0 : tail) + tid, width = 1;
      in = e0 < (j == -1 ? head : part == n_parts - 1 ? V : 0);
#pragma unroll
      for (int i = 1; i < kEach; i++) v[i] = -kInf;
      v[0] = in ? up<TY>(x[e0]) : -kInf;
    }
    float hi = v[0], lo = v[0];
#pragma unroll
    for (int i = 1; i < kEach; i++) hi = fmaxf(hi, v[i]), lo = fminf(lo, v[i]);
    if (hi > m) {
      s += ls, w += lw, ls = lw = 0;
      move(s, w, m - hi);
      m = hi;
    }
    float bs = 0, bw = 0;  // the block's
    if (lo - m > -200.f) {
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        const float y = v[i] - m, e = __builtin_amdgcn_exp2f(y * kLog2e);
        bs += e;
        bw = __builtin_fmaf(e, y, bw);
      }
    } else {  // (exp is 0 there; 0 x -inf is not, and NaN stays NaN)
#pragma unroll
      for (int i = 0; i < kEach; i++) {
        const float d = v[i] - m, y = d < -200.f || v[i] == -kInf ? -200.f : d, e = __builtin_amdgcn_exp2f(y * kLog2e);
        bs += e;
        bw = __builtin_fmaf(e, y, bw);
      }
    }
    add_up(s, ls, bs);
    add_up(w, lw, bw);
    const bool odd = s != s;  // (a NaN or +inf was met: maxima say nothing)
    if (xt == xt && __any(!(hi < xt) || odd)) {
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool lower = e0 + u * kThreads * kVec + width <= t;
        const float y = lower ? below : xt;
        int r = 0;
#pragma unroll
        for (int i = 0; i < kVec; i++) r += !(v[u * kVec + i] <= y);
        c += lower && xt == -kInf ? 0 : r;
      }
    }
    const u64 pass = top > 0 ? __ballot(!(hi <= gate) || odd || n < top) : 0;
    if (pass) {
      uint32_t take = 0;  // a bit for each element that may be of use
      auto token = [&](int i) { return (uint32_t)(e0 + i / kVec * (kThreads * kVec) + i % kVec); };
      float least = n < top ? __builtin_nanf("") : gate;  // what is greater than it (NaN: all)
      if (n < top || __popcll(pass) > top) {
        uint32_t h = order_of(hi);
        if (in != kAll || odd) {
          h = 0;
#pragma unroll
          for (int i = 0; i < kEach; i++) h = max(h, in >> i & 1 ? order_of(v[i]) : 0u);
        }
        // at least `top` lanes' maxima reach this (its upper 16 bits by bisection; 0: fewer lanes have any element)
        uint32_t bound = 0;
#pragma unroll 1
        for (uint32_t bit = 0x80000000u; bit >= 0x10000u; bit >>= 1)
          if (__popcll(__ballot(h >= (bound | bit))) >= top) bound |= bit;
        if (bound) {  // at least that: greater than the float below
          float under = value_of(bound - 1);
          if (under == 0) under = -__uint_as_float(1);
          if (n < top || under > least) least = under;
        }
      }
#pragma unroll
      for (int i = 0; i < kEach; i++) take |= !(v[i] <= least) ? 1u << i : 0u;
      take &= in;
      while (__any(take != 0)) {  // a lane's next element
        if (n > kList - 64) {
          n = cut(list, n, top);
          gate = value_of(list[top - 1]);
        }
        const int i = take ? __builtin_ctz(take) : 0;
        float y = v[0];
#pragma unroll
        for (int e = 1; e < kEach; e++) y = i == e ? v[e] : y;
        n = add(list, n, take ? key_of(y, token(i)) : 0);
        take &= take - 1;
      }
      // what a later block needs to be of use: more than what `top` elements have
      if (n >= top) {
        if (n > kList - 64) {
          n = cut(list, n, top);
          gate = value_of(list[top - 1]);
        } else if (least > gate) {
          gate = least;
        }
      }
    }
    if (j == -2) break;
    j = j == -1 ? (j0 < j1 ? j0 : -2) : j + kStep < j1 ? j + kStep : -2;
    if (j == -2 && (part != n_parts - 1 || tail == V)) break;
  }
  s += ls, w += lw;
  // the token's own word was compared with xt: its lower tokens' equals count too
  const bool word = t >= head && t < tail;
  const int ts = word ? head + ((int)t - head) / kVec * kVec : (int)t;  // (its first token)
  const int in_part = word ? (ts - head) / kVec / words_per_part : t < head ? 0 : n_parts - 1;
  if (xt == xt && in_part == part && tid == 0) {
    for (int e = ts; e < (int)t; e++) {
      const float y = up<TY>(x[e]);
      c += xt == -kInf ? y <= xt : !(y <= below) && y <= xt;
    }
    if (xt == -kInf) c += ts;  // (every lower token comes before)
  }
  if (top > 0) join_lists(l, cut(list, n, top), top);
  join_all(l, m, s, w, c);
  if (n_parts == 1) {
    write_row(io, l, row, m, s, w, c, xt, t);
  } else {
    if (tid == 0) parts[blockIdx.x] = Part{m, s, w, c};
    if (tid < top) lists[(int64_t)blockIdx.x * top + tid] = tid < l.n[0] + l.n[1] + l.n[2] + l.n[3] ? l.all[tid] : 0;
  }
}

// One workgroup per row: its parts as one.
template <int TY>
__global__ __launch_bounds__(kThreads) void score_join(lxm_score_io io, int n_parts, const Part* parts, const double* lists) {
  typedef typename Elem<TY>::T T;
  __shared__ Lds l;
  const int row = blockIdx.x, tid = threadIdx.x, top = io.top;
  float m = -kInf, s = 0, w = 0;
  int c = 0;
  for (int i = tid; i < n_parts; i += kThreads) {
    Part p = parts[(int64_t)row * n_parts + i];
    const float n = fmaxf(m, p.m);
    move(s, w, m - n);
    move(p.s, p.w, p.m - n);
    m = n, s += p.s, w += p.w, c += p.c;
  }
  if (top > 0) {
    // each wave takes some parts' lists, 64 keys at a time
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), e1 = n_parts * top;
    const double* list = lists + (int64_t)row * e1;
    double gate = 0;
    int n = 0;
    for (int e = 64 * wave; e < e1; e += kThreads) {
      const double k = e + (tid & 63) < e1 ? list[e + (tid & 63)] : 0;
      n = add(l.list[wave], n, k > gate ? k : 0);
      if (n > kList - 64 || e + kThreads >= e1) {
        n = cut(l.list[wave], n, top);
        if (n == top) gate = l.list[wave][top - 1];
      }
    }
    join_lists(l, n, top);
  }
  join_all(l, m, s, w, c);
  const int64_t t = token_at(io, row);
  const float xt = t >= 0 && t < io.V ? up<TY>(((const T*)io.logits)[row * io.stride + t]) : __builtin_nanf("");
  write_row(io, l, row, m, s, w, c, xt, t);
}

bool bad(const lxm_score_io* io) {
  return !io || io->rows < 0 || io->V < 1 || io->V > 0x7fffffff - 64 || io->top < 0 || io->top > LXM_SCORE_TOP || io->top > io->V ||
         io->type < 0 || io->type > 2;
}

// How many parts a row is split into: enough for 4 workgroups a CU, each of at least 4,096 elements (top 8, least of
// 4,096 / 8,192 / 32,768: one row of 459,982 in 14.8 / 15.4 / 20.5 us, 61 of 31,999 in 15.2 / 15.7 / 25.1; 2 and 8
// workgroups a CU: 600 rows of 248,320 94.7 and 91.4 against 89.2).
constexpr int kLeast = 4096, kRows = 0xffffffffu / kThreads;
int parts_of(const lxm_score_io* io) {
  const int64_t most = ((int64_t)io->V + kLeast - 1) / kLeast;
  int64_t n = io->rows > 0 ? ((int64_t)io->rows + 1023) / io->rows : 1;
  return (int)(n > most ? most : n < 1 ? 1 : n);
}

template <int TY>
int launch(const lxm_score_io* io, char* ws, hipStream_t st) {
  const int vec = TY == 2 ? 4 : 8, n = parts_of(io);
  const int64_t words = (int64_t)io->V / vec;
  const int per = (int)((words + n - 1) / n) + (words < n);  // (at least 1)
  Part* parts = (Part*)ws;
  double* lists = (double*)(ws + (int64_t)io->rows * n * sizeof(Part));
  // Blocks of 16 elements a lane for a part that is one block, of 32 for whole rows, whose loads they keep in flight
  // (2,048 rows of 248,320, top 8: 210 us, in blocks of 8 219).
  if (n > 1) {  // (rows x n <= 2,046)
    score_part<TY, 16><<<io->rows * n, kThreads, 0, st>>>(*io, n, per, parts, lists);
    score_join<TY><<<io->rows, kThreads, 0, st>>>(*io, n, parts, lists);
  } else {
    lxm_score_io r = *io;
    for (int left = io->rows; left > 0; left -= kRows) {  // (a launch's threads are counted in 32 bits)
      score_part<TY, 32><<<left < kRows ? left : kRows, kThreads, 0, st>>>(r, n, per, parts, lists);
      if (int e = hipGetLastError()) return e;
      r.logits = (const char*)r.logits + kRows * r.stride * (TY == 2 ? 4 : 2);
      r.tokens = (const char*)r.tokens + (int64_t)kRows * (r.wide ? 8 : 4);
      r.logprob += kRows, r.entropy += kRows, r.rank += kRows;
      r.top_tokens += (int64_t)kRows * r.top, r.top_logprobs += (int64_t)kRows * r.top;
    }
  }
  return hipGetLastError();
}

}  // namespace

extern "C" int lxm_score_ws(const lxm_score_io* io, int64_t* bytes) {
  if (bad(io) || !bytes) return hipErrorInvalidValue;
  const int64_t n = parts_of(io);
  *bytes = n == 1 ? 0 : io->rows * n * ((int64_t)sizeof(Part) + 8 * io->top);
  return hipSuccess;
}

extern "C" int lxm_score(const lxm_score_io* io, void* ws, int64_t ws_bytes, void* stream) {
  int64_t need = 0;
  if (int e = lxm_score_ws(io, &need)) return e;
  if (io->rows == 0) return hipSuccess;
  if (!io->logits || !io->tokens || !io->logprob || !io->entropy || !io->rank || (io->top && (!io->top_tokens || !io->top_logprobs)) ||
      ws_bytes < need || (need && (!ws || ((uintptr_t)ws & 15))))
    return hipErrorInvalidValue;
  const hipStream_t st = (hipStream_t)stream;
  return io->type == 0 ? launch<0>(io, (char*)ws, st) : io->type == 1 ? launch<1>(io, (char*)ws, st) : launch<2>(io, (char*)ws, st);
}
