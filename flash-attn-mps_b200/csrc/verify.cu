// Verification of drafted tokens against the target's probabilities.
//
// One pass over a row's logits gives its maximum, its sum of exponentials and
// (for greedy requests) its first maximum; the acceptance chain of a request
// then names one row, whose second pass finds the first maximum of
// w / noise. HBM-bound: every row of logits once, one row of draft
// probabilities and of noise per request.
//
// Two launches: verify_stats_kernel over (row, chunk of the vocabulary), then
// verify_pick_kernel over (request, chunk), whose CTAs each join the chunks'
// statistics (a few numbers), walk the acceptance chain and search their chunk
// of the row it names; the last CTA of a request writes its tokens. The second
// launch may begin before the first ends and waits for it on the device.
// 64 requests of 1..5 drafts, 151936 tokens, bf16: 45 us for 154 MB (3.4 TB/s),
// 19 and 27 us by themselves: latency (the chain statistics -> acceptance -> row)
// before bandwidth. One request: 19 us a call, the host's time; 12 on the GPU.
// Weights and their quotients are good to a few units of float32; of two that
// lie closer together either may be taken, whichever route a call goes.
#include <algorithm>

#include "common.cuh"
#include "ptx.cuh"

namespace fab {
namespace {

struct VerifyArgs {
  const void* x; int32_t xt; int64_t xs0, xs1;
  const void* tok; int32_t tt; int64_t tk0;
  const int32_t* cu; int64_t cu0;
  const float* u; int64_t u0;
  const float* noise; int64_t no0, no1;
  const void* dp; int32_t dt; int64_t dp0, dp1;
  const float* temp; int64_t te0;
  int64_t* out; int64_t o0, o1;
  int32_t* acc; int64_t a0;
  int32_t B, V, K;
};

// Larger value, lower index on a tie.
__device__ __forceinline__ void best_of(float& v, int& i, float w, int j) {
  if (w > v || (w == v && j < i)) { v = w; i = j; }
}

constexpr float kLog2e = 1.4426950408889634f;

// log2(e) / temperature. It multiplies differences to a row's maximum only: a
// scaled score itself may need more than float32's bits (2^25 at a temperature
// of 1e-6). Bounded, so that 0 and -inf stay what they are at any temperature.
__device__ __forceinline__ float per_temperature(float temp) { return fminf(fmaxf(kLog2e / temp, 1e-30f), 1e30f); }

// Order of w / e at token v as an integer: the larger quotient, then the lower
// token; 0 without one (w not positive, e negative or NaN). float32 holds neither
// 1 / 2^-149 nor 2^-30 / 2^127: the mantissas' quotient is rounded to float32 and
// takes the exponents' difference beside it (its 23 bits and 9 of exponent fit 32).
__device__ __forceinline__ unsigned long long quotient_key(float w, float e, int v) {
  if (!(w > 0.f && e >= 0.f)) return 0;
  uint32_t key = 1;                              // e infinite
  if (e == 0.f || w == INFINITY) {
    key = 0xffffffffu;
  } else if (e < INFINITY) {
    int shift = 256;                             // of the quotient's exponent field
    if (w < 0x1p-126f) { w *= 0x1p24f; shift -= 24; }
    if (e < 0x1p-126f) { e *= 0x1p24f; shift += 24; }
    const uint32_t wb = __float_as_uint(w), eb = __float_as_uint(e);
    const float q = __fdiv_rn(__uint_as_float((wb & 0x7fffffu) | 0x3f800000u), __uint_as_float((eb & 0x7fffffu) | 0x3f800000u));
    shift += (int)(wb >> 23) - (int)(eb >> 23);  // |difference| < 256 + 24
    const int64_t k = (int64_t)__float_as_uint(q) + ((int64_t)(shift - 127) << 23);
    key = (uint32_t)min(max(k, (int64_t)1), (int64_t)0xfffffffe);
  }
  return (unsigned long long)key << 32 | (0xffffffffu - (uint32_t)v);
}
// The same of a quotient that float32 holds.
__device__ __forceinline__ unsigned long long quotient_key(float y, int v) {
  return (unsigned long long)(__float_as_uint(y) + (129u << 23)) << 32 | (0xffffffffu - (uint32_t)v);
}
__device__ __forceinline__ int token_of(unsigned long long key) { return (int)(0xffffffffu - (uint32_t)key); }
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long k) {
#pragma unroll
  for (int o = 16; o; o >>= 1) k = max(k, __shfl_xor_sync(~0u, k, o));
  return k;
}

// One CTA per request, rows in turn: strided vocabularies and very many rows.
__global__ void __launch_bounds__(1024) verify_kernel(const VerifyArgs a) {
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = a.cu[b * a.cu0], n = min(max(a.cu[(b + 1) * a.cu0] - begin, 0), a.K);
  const float temp = a.temp ? a.temp[b * a.te0] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float k = per_temperature(greedy ? 1.f : temp);
  __shared__ float sv[32], ss[32];
  __shared__ int si[32];
  __shared__ unsigned long long sr[32], sf[32];
  float mx = -INFINITY, sum = 0.f;
  int hot = 0, i = 0;
  for (;; ++i) {
    const int64_t row = (int64_t)(begin + b + i) * a.xs0;
    float m = -INFINITY;
    int at = 0x7fffffff;
    for (int v = tid; v < a.V; v += 1024) best_of(m, at, load_float(a.x, a.xt, row + v * a.xs1), v);
    for (int o = 16; o; o >>= 1) {
      const float w = __shfl_xor_sync(~0u, m, o);
      const int j = __shfl_xor_sync(~0u, at, o);
      best_of(m, at, w, j);
    }
    if (lane == 0) { sv[warp] = m; si[warp] = at; }
    __syncthreads();
    mx = sv[0]; hot = si[0];
    for (int w = 1; w < 32; ++w) best_of(mx, hot, sv[w], si[w]);
    if (hot >= a.V) hot = 0;
    float s = 0.f;
    if (!greedy)
      for (int v = tid; v < a.V; v += 1024) s += fast_exp2((load_float(a.x, a.xt, row + v * a.xs1) - mx) * k);
    s = warp_sum(s);
    if (lane == 0) ss[warp] = s;
    __syncthreads();
    sum = 0.f;
    for (int w = 0; w < 32; ++w) sum += ss[w];
    __syncthreads();
    if (i >= n) break;
    const int64_t tok = load_index(a.tok, a.tt, (int64_t)(begin + i) * a.tk0);
    float p = 0.f;
    if (tok >= 0 && tok < a.V) p = greedy ? (tok == hot ? 1.f : 0.f) : fast_exp2((load_float(a.x, a.xt, row + tok * a.xs1) - mx) * k) / sum;
    const float q = a.dp ? (tok >= 0 && tok < a.V ? load_float(a.dp, a.dt, (int64_t)(begin + i) * a.dp0 + tok * a.dp1) : 0.f) : 1.f;
    if (!(a.u[(int64_t)(begin + i) * a.u0] * q < p)) break;
  }
  // Row i: the first rejected draft's (i < n) or the one behind the last.
  const int64_t row = (int64_t)(begin + b + i) * a.xs0;
  const int64_t drafted = i < n && !a.dp ? load_index(a.tok, a.tt, (int64_t)(begin + i) * a.tk0) : -1;
  const float is = 1.f / sum;
  unsigned long long r = 0, f = 0;  // best of the residual, of p
  for (int v = tid; v < a.V; v += 1024) {
    const float p = greedy ? (v == hot ? 1.f : 0.f) : fast_exp2((load_float(a.x, a.xt, row + v * a.xs1) - mx) * k) * is;
    float q = 0.f;
    if (i < n) q = a.dp ? load_float(a.dp, a.dt, (int64_t)(begin + i) * a.dp0 + v * a.dp1) : (v == drafted ? 1.f : 0.f);
    const float e = a.noise[(int64_t)b * a.no0 + v * a.no1];
    f = max(f, quotient_key(p, e, v));
    r = max(r, quotient_key(p - q, e, v));
  }
  r = warp_max_key(r);
  f = warp_max_key(f);
  if (lane == 0) { sr[warp] = r; sf[warp] = f; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < 32; ++w) { r = max(r, sr[w]); f = max(f, sf[w]); }
    const int got = r ? token_of(r) : f ? token_of(f) : 0;
    for (int k = 0; k <= a.K; ++k)
      a.out[b * a.o0 + k * a.o1] = k < i ? load_index(a.tok, a.tt, (int64_t)(begin + k) * a.tk0) : k == i ? got : -1;
    a.acc[b * a.a0] = i;
  }
}

constexpr int kVerifyThreads = 256;
constexpr int kVerifyCtas = 8;  // per SM that a pass is cut into (4 and 16 measured alike or slower)

struct VerifyPlan {
  VerifyArgs v;
  int32_t rows, chunks, span;          // statistics: chunks of a row, their elements
  int32_t pick_chunks, pick_span;      // second pass, per request
  int32_t x_vec, y_vec;                // 16-byte vectors: logits; logits, draft rows and noise together
  float4* stats;                       // [rows][chunks] {maximum, sum of 2^((x - it) k), first maximum, -}
  unsigned long long* best;            // [B] largest w / noise (quotient_key)
  int32_t* done;                       // [B] CTAs of the second pass that are through
};

// N = 8 (16-bit) or 4 (f32) neighbours of a row.
template <int DT>
struct Vec {
  static constexpr int N = DT == FA_F32 ? 4 : 8;
  static __device__ __forceinline__ void load(const void* p, int64_t off, float* x) {
    const uint4 v = __ldg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(p) + off * (DT == FA_F32 ? 4 : 2)));
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (DT == FA_F32) {
        x[i] = __uint_as_float(w[i]);
      } else {
        float2 f;
        if constexpr (DT == FA_BF16) f = unpack2<__nv_bfloat16>(w[i]);
        else f = unpack2<__half>(w[i]);
        x[2 * i] = f.x;
        x[2 * i + 1] = f.y;
      }
    }
  }
  static __device__ __forceinline__ float one(const void* p, int64_t off) { return load_float(p, DT, off); }
};

// Running maximum and sum of 2^((y - maximum) k) over values y.
struct Running {
  float k, m = -INFINITY, s = 0.f;
  __device__ __forceinline__ explicit Running(float k) : k(k) {}
  template <int N>
  __device__ __forceinline__ void add(const float (&y)[N]) {
    float t[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) t[i] = y[i];
#pragma unroll
    for (int i = 4; i < N; ++i) t[i & 3] = fmaxf(t[i & 3], y[i]);
    const float n = fmaxf(m, fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
    const float c = n == -INFINITY ? 0.f : n;
    float a[4] = {s * fast_exp2((m - c) * k), 0.f, 0.f, 0.f};  // m = -inf: 0
    m = n;
#pragma unroll
    for (int i = 0; i < N; ++i) a[i & 3] += fast_exp2((y[i] - c) * k);
    s = (a[0] + a[1]) + (a[2] + a[3]);
  }
  __device__ __forceinline__ void join(float m2, float s2) {
    const float t = fmaxf(m, m2), c = t == -INFINITY ? 0.f : t;
    s = s * fast_exp2((m - c) * k) + s2 * fast_exp2((m2 - c) * k);
    m = t;
  }
};

// Request of logits row r, the last b with cu[b] + b <= r, by a whole warp (a
// search by halves would wait for one load after another).
__device__ __forceinline__ int request_of(const VerifyArgs& a, int r, int lane) {
  int n = 0;
#pragma unroll 4
  for (int b0 = 0; b0 < a.B; b0 += 32) {
    const int b = b0 + lane;
    n += __popc(__ballot_sync(~0u, b < a.B && __ldg(a.cu + (int64_t)b * a.cu0) + b <= r));
  }
  return max(n - 1, 0);
}

// A larger value wins; called with rising indices, so ties stay with the lowest.
__device__ __forceinline__ void rising(float& v, int& i, float w, int j) {
  if (w > v) { v = w; i = j; }
}

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads) verify_stats_kernel(const VerifyPlan pl) {
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");
  const VerifyArgs& a = pl.v;
  using V = Vec<DT>;
  constexpr int N = V::N, kU = 4;
  const int r = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  if (chunk == 0 && r < a.B && tid == 0) {
    pl.best[r] = 0;
    pl.done[r] = 0;
  }
  const int64_t row = (int64_t)r * a.xs0;
  const int v0 = chunk * pl.span, v1 = min(a.V, v0 + pl.span);
  // Elements up to the first 16-byte boundary, whole vectors, the rest.
  const uintptr_t addr = (uintptr_t)a.x + (row + v0) * (DT == FA_F32 ? 4 : 2);
  const int head = min(v1 - v0, (int)(((16 - (addr & 15)) & 15) / (DT == FA_F32 ? 4 : 2)));
  const int b0 = v0 + head, nvec = pl.x_vec ? (v1 - b0) / N : 0;
  auto load = [&](int i0, float (&x)[kU * N]) {
#pragma unroll
    for (int q = 0; q < kU; ++q) {
      const int i = i0 + q * kVerifyThreads;
      if (i < nvec) {
        V::load(a.x, row + b0 + (int64_t)i * N, x + q * N);
      } else {
#pragma unroll
        for (int h = 0; h < N; ++h) x[q * N + h] = -INFINITY;  // adds nothing
      }
    }
  };
  float x[kU * N];
  load(tid, x);  // on its way while the row's request is looked up
  const float temp = a.temp ? __ldg(a.temp + (int64_t)request_of(a, r, lane) * a.te0) : 1.f;
  const bool greedy = !(temp > 0.f);
  Running run(per_temperature(greedy ? 1.f : temp));
  float top = -INFINITY;
  int at = 0x7fffffff;
  for (int i0 = tid; i0 < nvec; i0 += kU * kVerifyThreads) {
    if (greedy) {
#pragma unroll
      for (int q = 0; q < kU; ++q)
#pragma unroll
        for (int h = 0; h < N; ++h) rising(top, at, x[q * N + h], b0 + (i0 + q * kVerifyThreads) * N + h);
    } else {
      run.add(x);
    }
    if (i0 + kU * kVerifyThreads < nvec) load(i0 + kU * kVerifyThreads, x);
  }
  auto use_one = [&](int v) {
    const float y = V::one(a.x, row + v);
    if (greedy) best_of(top, at, y, v);
    else run.join(y, y == -INFINITY ? 0.f : 1.f);
  };
  if (pl.x_vec && tid < head) use_one(v0 + tid);
  for (int v = (pl.x_vec ? b0 + nvec * N : v0) + tid; v < v1; v += kVerifyThreads) use_one(v);
  __shared__ float sm[8], ss[8];
  __shared__ int si[8];
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    run.join(__shfl_xor_sync(~0u, run.m, o), __shfl_xor_sync(~0u, run.s, o));
    const float w = __shfl_xor_sync(~0u, top, o);
    best_of(top, at, w, __shfl_xor_sync(~0u, at, o));
  }
  if (lane == 0) { sm[warp] = greedy ? top : run.m; ss[warp] = run.s; si[warp] = at; }
  __syncthreads();
  if (tid == 0) {
    for (int w = 1; w < kVerifyThreads / 32; ++w) {
      if (greedy) best_of(top, at, sm[w], si[w]);
      else run.join(sm[w], ss[w]);
    }
    pl.stats[(int64_t)r * pl.chunks + chunk] = make_float4(greedy ? top : run.m, run.s, __int_as_float(at), 0.f);
  }
}

constexpr int kPick = 1;    // vectors of a thread in flight (2 need the registers of a CTA per SM: 50 us against 46)
constexpr int kRows = 64;   // rows of a request whose numbers stay in shared memory

// N noise values from v on (1 past the end).
template <int N>
__device__ __forceinline__ void load_noise(const float* row, int v, int end, float (&e)[N]) {
#pragma unroll
  for (int h = 0; h < N / 4; ++h) {
    const float4 w = v < end ? __ldcs(reinterpret_cast<const float4*>(row + v + 4 * h)) : make_float4(1.f, 1.f, 1.f, 1.f);
    e[4 * h] = w.x; e[4 * h + 1] = w.y; e[4 * h + 2] = w.z; e[4 * h + 3] = w.w;
  }
}
// N draft probabilities from v on.
template <int N>
__device__ __forceinline__ void load_probs(const VerifyArgs& a, bool with_q, int64_t row, int v, int end, float (&q)[N]) {
  if (!with_q || v >= end) {
#pragma unroll
    for (int h = 0; h < N; ++h) q[h] = 0.f;
  } else if (a.dt == FA_F32) {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const float4 w = __ldcs(reinterpret_cast<const float4*>(reinterpret_cast<const float*>(a.dp) + row + v + 4 * h));
      q[4 * h] = w.x; q[4 * h + 1] = w.y; q[4 * h + 2] = w.z; q[4 * h + 3] = w.w;
    }
  } else {
#pragma unroll
    for (int h = 0; h < N / 4; ++h) {
      const uint2 w = __ldcs(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(a.dp) + row + v + 4 * h));
      const float2 lo = a.dt == FA_BF16 ? unpack2<__nv_bfloat16>(w.x) : unpack2<__half>(w.x);
      const float2 hi = a.dt == FA_BF16 ? unpack2<__nv_bfloat16>(w.y) : unpack2<__half>(w.y);
      q[4 * h] = lo.x; q[4 * h + 1] = lo.y; q[4 * h + 2] = hi.x; q[4 * h + 3] = hi.y;
    }
  }
}

template <int DT>
__global__ void __launch_bounds__(kVerifyThreads, 4) verify_pick_kernel(const VerifyPlan pl) {
  const VerifyArgs& a = pl.v;
  using V = Vec<DT>;
  const int b = blockIdx.y, chunk = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int begin = a.cu[b * a.cu0], n = min(max(a.cu[(b + 1) * a.cu0] - begin, 0), a.K);
  const float temp = a.temp ? a.temp[b * a.te0] : 1.f;
  const bool greedy = !(temp > 0.f);
  const float k = per_temperature(greedy ? 1.f : temp);
  // What does not depend on the statistics is read while they are computed:
  // a warp's draft and this thread's first noise.
  const int v0 = chunk * pl.pick_span, v1 = min(a.V, v0 + pl.pick_span);
  constexpr int N = V::N;
  const int64_t nrow = (int64_t)b * a.no0;
  float e0[kPick][N];
  if (pl.y_vec && !greedy) {
#pragma unroll
    for (int q = 0; q < kPick; ++q) load_noise<N>(a.noise + nrow, v0 + (tid + q * kVerifyThreads) * N, v1, e0[q]);
  }
  struct Draft { int64_t tok; float x, q, u; bool in; };
  auto draft_of = [&](int i) {
    Draft d;
    const int64_t at = begin + i;
    d.tok = load_index(a.tok, a.tt, at * a.tk0);
    d.in = d.tok >= 0 && d.tok < a.V;
    d.x = d.in ? V::one(a.x, (at + b) * a.xs0 + d.tok) : 0.f;
    d.q = a.dp ? (d.in ? load_float(a.dp, a.dt, at * a.dp0 + d.tok) : 0.f) : 1.f;
    d.u = a.u[at * a.u0];
    return d;
  };
  Draft mine;
  if (warp < n) mine = draft_of(warp);
  __shared__ int first_no;
  __shared__ float4 rows[kRows];
  if (tid == 0) first_no = n;
  __syncthreads();
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  // A row's maximum, sum and first maximum, by one warp.
  auto row_stats = [&](int i, float& m, float& s, int& hot) {
    const float4* st = pl.stats + (int64_t)(begin + b + i) * pl.chunks;
    Running run(k);
    float top = -INFINITY;
    int at = 0x7fffffff;
    for (int c = lane; c < pl.chunks; c += 32) {
      const float4 x = st[c];
      if (greedy) best_of(top, at, x.x, __float_as_int(x.z));
      else run.join(x.x, x.y);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      run.join(__shfl_xor_sync(~0u, run.m, o), __shfl_xor_sync(~0u, run.s, o));
      const float w = __shfl_xor_sync(~0u, top, o);
      best_of(top, at, w, __shfl_xor_sync(~0u, at, o));
    }
    m = run.m;
    s = run.s;
    hot = at < a.V ? at : 0;
  };
  for (int i = warp; i <= n; i += kVerifyThreads / 32) {
    float m, s;
    int hot;
    row_stats(i, m, s, hot);
    if (lane == 0 && i < kRows) rows[i] = make_float4(m, s, __int_as_float(hot), 0.f);
    if (i == n) break;
    const Draft d = i == warp ? mine : draft_of(i);
    float p = 0.f;
    if (d.in) p = greedy ? (d.tok == hot ? 1.f : 0.f) : fast_exp2((d.x - m) * k) / s;
    if (lane == 0 && !(d.u * d.q < p)) atomicMin(&first_no, i);
  }
  __syncthreads();
  const int i = first_no;
  if (i >= kRows) {  // very many drafts: the row's numbers again
    if (warp == 0) {
      float m, s;
      int hot;
      row_stats(i, m, s, hot);
      if (lane == 0) rows[0] = make_float4(m, s, __int_as_float(hot), 0.f);
    }
    __syncthreads();
  }
  const float4 st = rows[i < kRows ? i : 0];
  const int shot = __float_as_int(st.z);
  const float m = st.x, s = st.y;
  unsigned long long best = 0;
  if (!greedy) {
    const int64_t row = (int64_t)(begin + b + i) * a.xs0, qrow = (int64_t)(begin + i) * a.dp0;
    const bool with_q = i < n && a.dp;
    const int64_t drafted = i < n && !a.dp ? load_index(a.tok, a.tt, (int64_t)(begin + i) * a.tk0) : -1;
    const float is = 1.f / s;
    auto weight = [&](float x, float q, int v) { return fast_exp2((x - m) * k) * is - (v == drafted ? 1.f : q); };
    auto read = [&](int v) { return weight(V::one(a.x, row + v), with_q ? load_float(a.dp, a.dt, qrow + v) : 0.f, v); };
    auto divide = [&](int from, int to, int step) {
#pragma unroll 1
      for (int v = from; v < to; v += step) best = max(best, quotient_key(read(v), a.noise[nrow + v], v));
    };
    // w / e by an approximate reciprocal, good to 2^-22 as w itself; false where
    // that leaves float32's range and a division is due.
    float r = -1.f;
    int ri = 0x7fffffff;
    auto approximate = [&](float w, float e, int v) {
      float ie;
      asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(ie) : "f"(e));
      const float z = w * ie;
      const bool in = z >= 0x1p-126f && z <= 0x1p100f;
      if (in) rising(r, ri, z, v);
      return in || !(w > 0.f);
    };
    if (pl.y_vec) {
      for (int w0 = v0; w0 < v1; w0 += kPick * kVerifyThreads * N) {
        float x[kPick][N], y[kPick][N];
#pragma unroll
        for (int q = 0; q < kPick; ++q) {
          const int v = w0 + (tid + q * kVerifyThreads) * N;
          if (w0 != v0) load_noise<N>(a.noise + nrow, v, v1, e0[q]);
          if (v < v1) V::load(a.x, row + v, x[q]);
          load_probs<N>(a, with_q, qrow, v, v1, y[q]);
        }
#pragma unroll
        for (int q = 0; q < kPick; ++q) {
          const int v = w0 + (tid + q * kVerifyThreads) * N;
          if (v < v1) {
            bool odd = false;
#pragma unroll
            for (int h = 0; h < N; ++h) odd |= !approximate(weight(x[q][h], y[q][h], v + h), e0[q][h], v + h);
            if (odd) divide(v, v + N, 1);
          }
        }
      }
    } else {
      bool odd = false;
#pragma unroll 4
      for (int v = v0 + tid; v < v1; v += kVerifyThreads) odd |= !approximate(read(v), a.noise[nrow + v], v);
      if (odd) divide(v0 + tid, v1, kVerifyThreads);
    }
    if (ri < a.V) best = max(best, quotient_key(r, ri));
  }
  best = warp_max_key(best);
  if (lane == 0) {
    if (best) atomicMax(pl.best + b, best);
    __threadfence();
  }
  __syncthreads();
  __shared__ int last;
  if (tid == 0) last = atomicAdd(pl.done + b, 1) == (int)gridDim.x - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  unsigned long long key = *reinterpret_cast<volatile unsigned long long*>(pl.best + b);
  __syncthreads();  // every thread has read it before any raises it below
  if (!greedy && key == 0 && i < n) {
    // No residual anywhere: the target's own probabilities (this CTA alone; a
    // draft is rejected where q >= p throughout, which rounding alone allows).
    const int64_t row = (int64_t)(begin + b + i) * a.xs0;
    const float is = 1.f / s;
    best = 0;
    for (int v = tid; v < a.V; v += kVerifyThreads) {
      const float p = fast_exp2((V::one(a.x, row + v) - m) * k) * is;
      best = max(best, quotient_key(p, a.noise[nrow + v], v));
    }
    best = warp_max_key(best);
    if (lane == 0 && best) atomicMax(pl.best + b, best);
    __threadfence();
    __syncthreads();
    key = *reinterpret_cast<volatile unsigned long long*>(pl.best + b);
  }
  const int got = greedy ? shot : key ? token_of(key) : 0;
  for (int j = tid; j <= a.K; j += kVerifyThreads)
    a.out[b * a.o0 + j * a.o1] = j < i ? load_index(a.tok, a.tt, (int64_t)(begin + j) * a.tk0) : j == i ? got : -1;
  if (tid == 0) a.acc[b * a.a0] = i;
}

// Chunks so that a pass over `rows` rows is about `ctas` CTAs per SM, each of
// whole batches of `batch` elements (every thread's loads in flight together).
void cut(int64_t rows, int V, int ctas, int batch, int32_t* chunks, int32_t* span) {
  const int64_t want = std::max<int64_t>(1, ((int64_t)ctas * sm_count() + rows - 1) / rows);
  int64_t per = (V + want - 1) / want;
  per = (per + batch - 1) / batch * batch;
  if (rows * ((V + batch - 1) / batch) < 2 * sm_count()) per = batch / 4;  // few rows: as many CTAs as there are
  *span = (int32_t)std::min<int64_t>(per, (V + 31) / 32 * 32);
  *chunks = (V + *span - 1) / *span;
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The two-launch path: unit strides along the vocabulary.
bool make_plan(const VerifyArgs& a, int64_t rows, VerifyPlan* p, size_t* bytes) {
  if (a.xs1 != 1 || a.no1 != 1 || (a.dp && a.dp1 != 1) || rows > 65535 || a.B > 65535) return false;
  *p = VerifyPlan{};
  p->v = a;
  p->rows = (int32_t)rows;
  const int per_vec = a.xt == FA_F32 ? 4 : 8;
  cut(rows, a.V, kVerifyCtas, 4 * kVerifyThreads * per_vec, &p->chunks, &p->span);
  cut(a.B, a.V, kVerifyCtas, kPick * kVerifyThreads * per_vec, &p->pick_chunks, &p->pick_span);
  const int elt = elem_size(a.xt), qelt = a.dp ? elem_size(a.dt) : 0;
  auto al = [](const void* ptr, int64_t stride_bytes, int n) { return ((uintptr_t)ptr % n) == 0 && stride_bytes % n == 0; };
  p->x_vec = ((uintptr_t)a.x % elt) == 0;  // rows may begin anywhere
  const int per = elt == 4 ? 4 : 8;        // elements of a thread's vector
  p->y_vec = a.V % per == 0 && al(a.x, a.xs0 * elt, 16) && al(a.noise, a.no0 * 4, 16) &&
             (!a.dp || al(a.dp, a.dp0 * qelt, qelt == 4 ? 16 : 8));
  *bytes = up256((size_t)rows * p->chunks * sizeof(float4)) + up256((size_t)a.B * 8) + up256((size_t)a.B * 4);
  return true;
}

template <int DT>
int launch_verify(const VerifyPlan& p, cudaStream_t st) {
  verify_stats_kernel<DT><<<dim3((unsigned)p.chunks, (unsigned)p.rows), kVerifyThreads, 0, st>>>(p);
  note_launch();
  FAB_LAUNCH_CHECK("draft verification launch");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)p.pick_chunks, (unsigned)p.v.B);
  cfg.blockDim = dim3(kVerifyThreads);
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, verify_pick_kernel<DT>, p);
  if (e != cudaSuccess) return fail(FA_ERR_CUDA, "draft verification launch: %s", cudaGetErrorString(e));
  note_launch();
  return FA_OK;
}

int fill(const fa_verify_args* g, VerifyArgs* a) {
  FAB_CHECK_ARG(g != nullptr, "null arguments");
  FAB_CHECK_ARG(g->batch >= 1 && g->max_draft >= 0 && g->max_draft <= 1024, "batch must be positive, max_draft in 0..1024");
  const fa_tensor &x = g->logits, &tk = g->draft_tokens;
  FAB_CHECK_ARG(present(x) && x.ndim == 2 && is_float(x.dtype) && x.shape[1] >= 1 && x.shape[1] < (1LL << 30),
                "logits must be float [rows, vocabulary]");
  FAB_CHECK_ARG(present(tk) && tk.ndim == 1 && (tk.dtype == FA_I32 || tk.dtype == FA_I64) &&
                    x.shape[0] == tk.shape[0] + g->batch,
                "logits need one row per draft token and one more per request");
  const int64_t N = tk.shape[0], V = x.shape[1];
  FAB_CHECK_ARG(present(g->cu_drafts) && g->cu_drafts.dtype == FA_I32 && g->cu_drafts.ndim == 1 &&
                    g->cu_drafts.shape[0] == g->batch + 1,
                "cu_drafts must be int32 [batch + 1]");
  FAB_CHECK_ARG(present(g->uniform) && g->uniform.dtype == FA_F32 && g->uniform.ndim == 1 && g->uniform.shape[0] == N,
                "uniform must be float32 with one value per draft token");
  FAB_CHECK_ARG(present(g->noise) && g->noise.dtype == FA_F32 && g->noise.ndim == 2 && g->noise.shape[0] == g->batch &&
                    g->noise.shape[1] == V,
                "noise must be float32 [batch, vocabulary]");
  FAB_CHECK_ARG(!present(g->draft_probs) || (is_float(g->draft_probs.dtype) && g->draft_probs.ndim == 2 &&
                                             g->draft_probs.shape[0] == N && g->draft_probs.shape[1] == V),
                "draft_probs must be float [draft tokens, vocabulary]");
  FAB_CHECK_ARG(!present(g->temperature) || (g->temperature.dtype == FA_F32 && g->temperature.ndim == 1 &&
                                             g->temperature.shape[0] == g->batch),
                "temperature must be float32 [batch]");
  FAB_CHECK_ARG(present(g->tokens) && g->tokens.dtype == FA_I64 && g->tokens.ndim == 2 && g->tokens.shape[0] == g->batch &&
                    g->tokens.shape[1] == g->max_draft + 1,
                "tokens must be int64 [batch, max_draft + 1]");
  FAB_CHECK_ARG(present(g->accepted) && g->accepted.dtype == FA_I32 && g->accepted.ndim == 1 &&
                    g->accepted.shape[0] == g->batch,
                "accepted must be int32 [batch]");
  *a = VerifyArgs{};
  a->x = x.ptr; a->xt = x.dtype; a->xs0 = x.stride[0]; a->xs1 = x.stride[1];
  a->tok = tk.ptr; a->tt = tk.dtype; a->tk0 = tk.stride[0];
  a->cu = (const int32_t*)g->cu_drafts.ptr; a->cu0 = g->cu_drafts.stride[0];
  a->u = (const float*)g->uniform.ptr; a->u0 = g->uniform.stride[0];
  a->noise = (const float*)g->noise.ptr; a->no0 = g->noise.stride[0]; a->no1 = g->noise.stride[1];
  if (present(g->draft_probs)) {
    a->dp = g->draft_probs.ptr; a->dt = g->draft_probs.dtype;
    a->dp0 = g->draft_probs.stride[0]; a->dp1 = g->draft_probs.stride[1];
  }
  if (present(g->temperature)) { a->temp = (const float*)g->temperature.ptr; a->te0 = g->temperature.stride[0]; }
  a->out = (int64_t*)g->tokens.ptr; a->o0 = g->tokens.stride[0]; a->o1 = g->tokens.stride[1];
  a->acc = (int32_t*)g->accepted.ptr; a->a0 = g->accepted.stride[0];
  a->B = g->batch; a->V = (int32_t)V; a->K = g->max_draft;
  return FA_OK;
}

}  // namespace
}  // namespace fab

using namespace fab;

extern "C" int fa_verify_workspace_size(const fa_verify_args* g, size_t* bytes) {
  FAB_CHECK_ARG(bytes != nullptr, "bytes must not be null");
  *bytes = 0;
  VerifyArgs a;
  int rc = fill(g, &a);
  if (rc) return rc;
  VerifyPlan p;
  size_t need = 0;
  if (make_plan(a, g->logits.shape[0], &p, &need)) *bytes = need;
  return FA_OK;
}

extern "C" int fa_verify_draft_tokens(const fa_verify_args* g, void* stream) {
  VerifyArgs a;
  int rc = fill(g, &a);
  if (rc) return rc;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  VerifyPlan p;
  size_t need = 0;
  if (make_plan(a, g->logits.shape[0], &p, &need)) {
    FAB_CHECK_ARG(present(g->workspace) && g->workspace.ndim >= 1 &&
                      (size_t)g->workspace.shape[0] * elem_size(g->workspace.dtype) >= need &&
                      ((uintptr_t)g->workspace.ptr & 15u) == 0,
                  "workspace smaller than fa_verify_workspace_size, or not 16-byte aligned");
    uint8_t* ws = reinterpret_cast<uint8_t*>(g->workspace.ptr);
    p.stats = reinterpret_cast<float4*>(ws);
    ws += up256((size_t)p.rows * p.chunks * sizeof(float4));
    p.best = reinterpret_cast<unsigned long long*>(ws);
    p.done = reinterpret_cast<int32_t*>(ws + up256((size_t)a.B * 8));
    return a.xt == FA_BF16 ? launch_verify<FA_BF16>(p, st) : a.xt == FA_F16 ? launch_verify<FA_F16>(p, st)
                                                                           : launch_verify<FA_F32>(p, st);
  }
  verify_kernel<<<(unsigned)a.B, 1024, 0, st>>>(a);
  note_launch();
  FAB_LAUNCH_CHECK("draft verification launch");
  return FA_OK;
}
