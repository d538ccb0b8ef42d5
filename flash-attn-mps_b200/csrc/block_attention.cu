// Attention over a block-scaled E4M3 cache: argument checks, kernel choice and
// the kernel that takes every type, head dim and stride.
//
// With k_j = ks * c_j and v_j = vs * d_j (c, d the E4M3 codes, ks, vs the
// scales of key j's block), the kernels form
//   t_j = scale * log2e * ks_j * (q . c_j) + log2(vs_j),  p_j = 2^(t_j - m)
//   out = sum_j p_j d_j / sum_j p_j / vs_j,  lse = ln2 * (m + log2 sum_j p_j / vs_j)
// so both scales cost nothing per head dimension: one joins the factor of the
// score, the other its additive term and the factor of the row sum.
#include <algorithm>
#include <cmath>

#include "block_cache.cuh"
#include "prefill_common.cuh"
#include "ptx.cuh"

namespace fab {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// One CTA per (query row, head): each warp takes 32 keys at a time, a lane
// forms one key's score, then the lanes split the head dimension for P V.
// Types and head dims outside the tensor-core kernels only; not tuned.
__global__ void __launch_bounds__(128) block_attention_any_kernel(const BlockAttn p) {
  const int h = blockIdx.y, b = blockIdx.z;
  const int begin = p.cu_q[b * p.cq0], n = p.cu_q[(b + 1) * p.cq0] - begin;
  const int i = blockIdx.x;
  if (i >= n) return;
  const BlockCache& c = p.c;
  const int D = c.D, kh = h / (p.HQ / c.HK);
  const int len = p.used[b * p.u0];
  const int pos = len - n + i;
  const int hi = min(len, p.causal ? pos + 1 : len);           // keys [0, hi)
  const int lo = p.win >= 0 ? max(0, pos - p.win) : 0;         // window begins here
  const int nf = min(min(p.first, lo), max(hi, 0));            // first tokens before it
  const int keys = nf + max(0, hi - lo);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  __shared__ float qs[512];
  __shared__ float sm[4], sl[4];
  __shared__ float so[4][512];
  const int64_t t = (int64_t)begin + i;
  for (int d = threadIdx.x; d < D; d += blockDim.x)
    qs[d] = load_float(p.q, p.qt, t * p.qs0 + (int64_t)h * p.qs1 + d * p.qs2) * (p.scale * kLog2e);
  __syncthreads();
  float m = -INFINITY, l = 0.f;
  float o[16];
#pragma unroll
  for (int k = 0; k < 16; ++k) o[k] = 0.f;
  for (int k0 = warp * 32; k0 < keys; k0 += 128) {
    const int at = k0 + lane;
    const int j = at < nf ? at : at - nf + lo;
    float s = -INFINITY, vs = 1.f;
    const uint8_t* vrow = nullptr;
    if (at < keys) {
      const int pg = block_page(c, b, j);
      const int in = j & (c.page - 1);
      float dot = 0.f;
      if (pg >= 0) {
        const uint8_t* krow = c.k + (int64_t)pg * c.ks0 + (int64_t)in * c.ks1 + (int64_t)kh * c.ks2;
        vrow = c.v + (int64_t)pg * c.vs0 + (int64_t)in * c.vs1 + (int64_t)kh * c.vs2;
        for (int d = 0; d < D; ++d) dot = fmaf(qs[d], e4m3_to_float(krow[d]), dot);
        dot *= clamp_scale(c.ksc[(int64_t)pg * c.kc0 + (int64_t)(in >> c.block_shift) * c.kc1 + kh * c.kc2]);
        vs = clamp_scale(c.vsc[(int64_t)pg * c.vc0 + (int64_t)(in >> c.block_shift) * c.vc1 + kh * c.vc2]);
      }
      s = dot;
    }
    const float mt = fmaxf(m, warp_max(s));
    if (mt == -INFINITY && !__any_sync(0xffffffffu, s != s)) continue;
    const float f = exp2f(m - mt);  // m = -inf gives 0
    const float w = at < keys ? exp2f(s - mt) : 0.f;
    l = l * f + warp_sum(w);
    m = mt;
#pragma unroll
    for (int k = 0; k < 16; ++k) o[k] *= f;
    for (int r = 0; r < 32; ++r) {
      const float wr = __shfl_sync(0xffffffffu, w * vs, r);
      const uint8_t* row = reinterpret_cast<const uint8_t*>(__shfl_sync(0xffffffffu, (unsigned long long)vrow, r));
      if (row == nullptr) continue;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const int d = k * 32 + lane;
        if (d < D) o[k] = fmaf(wr, e4m3_to_float(row[d]), o[k]);
      }
    }
  }
  if (lane == 0) { sm[warp] = m; sl[warp] = l; }
#pragma unroll
  for (int k = 0; k < 16; ++k)
    if (k * 32 + lane < D) so[warp][k * 32 + lane] = o[k];
  __syncthreads();
  const float sink = p.sinks ? load_float(p.sinks, p.sink_t, h * p.si0) * kLog2e : -INFINITY;
  float mx = sink, lt = 0.f, wt[4];
  for (int w = 0; w < 4; ++w) mx = fmaxf(mx, sm[w]);
  for (int w = 0; w < 4; ++w) {
    wt[w] = sm[w] == -INFINITY && sl[w] == 0.f ? 0.f : exp2f(sm[w] - mx);
    lt += wt[w] * sl[w];
  }
  if (sink != -INFINITY) lt += exp2f(sink - mx);
  for (int d = threadIdx.x; d < D; d += blockDim.x) {
    float x = 0.f;
    for (int w = 0; w < 4; ++w) x += wt[w] * so[w][d];
    store_float(p.out, p.qt, t * p.os0 + (int64_t)h * p.os1 + d * p.os2, keys > 0 && lt != 0.f ? x / lt : 0.f);
  }
  if (threadIdx.x == 0)
    p.lse[(int64_t)h * p.ls0 + t * p.ls1] = lt != 0.f ? (mx + log2f(lt)) * kLn2 : -INFINITY;
}

// ---- many query rows: a 16-bit copy of the visible rows, then the tcgen05 prefill
//
// Every prefill row block and head reads its keys again, so decoding them once
// (1 byte read, 2 written per element: 29 us for 4 requests of 2500..8192 keys
// with 8 KV heads of 128, in front of 560 us of prefill at 980 TFLOP/s)
// turns the call into the 16-bit prefill's compute-bound work. As every 16-bit
// prefill of the library it rounds P to q's type before P V (2^-9 for bf16, 2^-12
// for f16; row sums keep float32): the tensor cores' 16-bit rate is what the
// copy is made for, and P in two parts would double its P V products. The error
// against 64 bits is 2.3e-3 of the output in bf16, 1.7e-3 of it from rounding
// the output itself. block_mode_kernel
// looks at the visible scales of every request and KV head first:
//   0: code * scale is exact in the 16-bit type (4 significant bits): powers of
//      two, in f16 up to 2^7 (448 * 2^7 = 57344) and K's from 2^-15 on. What
//      f16 cannot hold of smaller V is below half its least number, which
//      outputs are rounded to as well; scales below 2^-60 (a block of zeros has
//      2^-100) make values that add nothing to a score or output in f16.
//   1: anything else (an f16 element of 65504 is cached as 256 * 2^8): the copy
//      holds the codes alone and the prefill takes both scales as the formulas
//      above do, one factor and one addend per key.
// Rows in front of a window that share a tile with visible ones are written as
// zeros, rows in tiles that no query sees not at all. The modes cost 4 us, the
// launch over codes 3 where there is no head for it.
struct CopyArgs {
  BlockCache c;
  uint16_t* k; uint16_t* v;          // [requests * max_k, HK, D]
  const int32_t* cu_q; int64_t cq0;
  const int32_t* used; int64_t u0;
  int32_t* cu_out; int32_t* used_out;
  int32_t* mode;                                     // [requests * HK]
  float* kfac; int64_t kfac_stride;                  // mode 1: [requests * HK][3][stride] (AttnParams)
  int32_t* reset;                                    // the prefill launches' two work counters
  float per_log2;                                    // raw score units of one log2 unit
  int32_t b0, B, max_k, win, first;
};

template <bool BF16>
__device__ __forceinline__ uint32_t scaled_pair(uint32_t f16x2, float s) {
  const float2 f = unpack2<__half>(f16x2);
  if constexpr (BF16) return pack2<__nv_bfloat16>(f.x * s, f.y * s);
  else return pack2<__half>(f.x * s, f.y * s);
}

// First key that a window of the request shows (0 without one).
__device__ __forceinline__ int window_begin(const CopyArgs& a, int n, int len) {
  return a.win >= 0 ? max(0, len - n - a.win) : 0;
}

// Whether the 16-bit copy may hold code * scale (see above).
template <bool BF16>
__device__ __forceinline__ bool plain_scale(float s, bool key) {
  const bool two = (__float_as_uint(s) & 0x7fffffu) == 0;
  if constexpr (BF16) return two;
  else return s < 0x1p-60f || (two && s <= 0x1p7f && (!key || s >= 0x1p-15f));
}

// Mode of a (KV head, request); also clears the work counters.
template <bool BF16>
__global__ void __launch_bounds__(256) block_mode_kernel(const CopyArgs a) {
  const int h = blockIdx.x, lb = blockIdx.y, b = a.b0 + lb;
  if (h == 0 && lb == 0 && threadIdx.x < 2) a.reset[threadIdx.x] = 0;
  const BlockCache& c = a.c;
  const int n = a.cu_q[(b + 1) * a.cq0] - a.cu_q[b * a.cq0];
  const int len = min(a.used[b * a.u0], a.max_k), lo = window_begin(a, n, len);
  bool plain = true;
#pragma unroll 4
  for (int64_t t = (int64_t)threadIdx.x << c.block_shift; t < len; t += (int64_t)256 << c.block_shift) {
    const int pg = t + c.block > lo || t < a.first ? block_page(c, b, (int)t) : -1;
    if (pg < 0) continue;
    const int blk = ((int)t & (c.page - 1)) >> c.block_shift;
    plain &= plain_scale<BF16>(clamp_scale(__ldg(c.ksc + (int64_t)pg * c.kc0 + (int64_t)blk * c.kc1 + (int64_t)h * c.kc2)), true) &
             plain_scale<BF16>(clamp_scale(__ldg(c.vsc + (int64_t)pg * c.vc0 + (int64_t)blk * c.vc1 + (int64_t)h * c.vc2)), false);
  }
  plain = __syncthreads_and(plain);
  if (threadIdx.x == 0) a.mode[(int64_t)lb * c.HK + h] = !plain;
}

// One CTA: 16 tokens (of one page and scale block) of a request, all KV heads.
template <bool BF16>
__global__ void __launch_bounds__(256) block_copy_kernel(const CopyArgs a) {
  const int lb = blockIdx.y, b = a.b0 + lb, t0 = blockIdx.x * 16;
  const int n = a.cu_q[(b + 1) * a.cq0] - a.cu_q[b * a.cq0];
  const int len = min(a.used[b * a.u0], a.max_k);
  if (t0 == 0 && threadIdx.x == 0) {
    a.cu_out[lb] = lb * a.max_k;
    if (lb == a.B - 1) a.cu_out[a.B] = a.B * a.max_k;
    a.used_out[lb] = max(len, 0);
  }
  if (t0 >= (len + 127) / 128 * 128 || len <= 0 || n <= 0) return;
  const int lo = window_begin(a, n, len);
  if (a.win >= 0 && t0 >= (a.first + 127) / 128 * 128 && t0 + 16 <= lo / 128 * 128) return;
  const BlockCache& c = a.c;
  const int pg = block_page(c, b, t0);
  const int in = t0 & (c.page - 1), blk = in >> c.block_shift;
  const int per_head = c.D / 16, per_row = c.HK * per_head;
#pragma unroll 2
  for (int e = threadIdx.x; e < 16 * per_row; e += 256) {
    const int r = e / per_row, rem = e - r * per_row, h = rem / per_head, d = (rem - h * per_head) * 16;
    const int t = t0 + r;
    const bool codes = a.mode[(int64_t)lb * c.HK + h];
    if (t >= len && !codes) continue;  // another head's scales may still be due
    uint4 kv[2];
    float s[2];
    const bool seen = pg >= 0 && t < len && (t >= lo || t < a.first);
    if (seen) {
      kv[0] = __ldcs(reinterpret_cast<const uint4*>(c.k + (int64_t)pg * c.ks0 + (int64_t)(in + r) * c.ks1 + (int64_t)h * c.ks2 + d));
      kv[1] = __ldcs(reinterpret_cast<const uint4*>(c.v + (int64_t)pg * c.vs0 + (int64_t)(in + r) * c.vs1 + (int64_t)h * c.vs2 + d));
      s[0] = clamp_scale(__ldg(c.ksc + (int64_t)pg * c.kc0 + (int64_t)blk * c.kc1 + (int64_t)h * c.kc2));
      s[1] = clamp_scale(__ldg(c.vsc + (int64_t)pg * c.vc0 + (int64_t)blk * c.vc1 + (int64_t)h * c.vc2));
    } else {
      kv[0] = kv[1] = make_uint4(0, 0, 0, 0);
      s[0] = s[1] = 1.f;
    }
    if (codes) {
      if (d == 0) {  // also of the last tile's keys past the end, whose zero probabilities they meet
        float* f = a.kfac + 3 * ((int64_t)lb * c.HK + h) * a.kfac_stride + t;
        f[0] = s[0];
        f[a.kfac_stride] = log2f(s[1]) * a.per_log2;
        f[2 * a.kfac_stride] = pf::kSumUnit / s[1];
      }
      if (t >= len) continue;
      s[0] = s[1] = 1.f;
    }
    const int64_t off = (((int64_t)lb * a.max_k + t) * c.HK + h) * c.D + d;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t w[4] = {kv[i].x, kv[i].y, kv[i].z, kv[i].w};
      uint32_t o[8];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        uint32_t lo2, hi2;
        e4m3x4_to_f16x2x2(w[q], lo2, hi2);
        o[2 * q] = scaled_pair<BF16>(lo2, s[i]);
        o[2 * q + 1] = scaled_pair<BF16>(hi2, s[i]);
      }
      uint4* dst = reinterpret_cast<uint4*>((i ? a.v : a.k) + off);
      dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
      dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
    }
  }
}

constexpr int64_t kPrefillCopy = 1LL << 30;  // most bytes of a copy; larger batches go in several passes

enum Route { kAny = 0, kDecode = 1, kPrefill = 2 };

struct Plan {
  int route, splits, reqs;       // reqs: requests per prefill pass
  size_t bytes, kv_bytes, fac_bytes, len_bytes;  // workspace; one of its 16-bit copies, the keys' scales, offsets and lengths
};

size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// The prefill's view of `reqs` requests' copies.
AttnParams prefill_view(const BlockAttn& p, int reqs) {
  AttnParams v{};
  v.q = p.q; v.qt = v.kt = v.vt = v.ot = p.qt;
  v.qs0 = p.qs0; v.qs1 = p.qs1; v.qs2 = p.qs2;
  v.k = v.v = reinterpret_cast<const void*>(uintptr_t(256));  // until the workspace is there (alignment)
  v.ks1 = v.vs1 = (int64_t)p.c.HK * p.c.D;
  v.ks2 = v.vs2 = p.c.D;
  v.ks3 = v.vs3 = 1;
  v.k_rows = (int64_t)reqs * p.max_k;
  v.out = p.out; v.os0 = p.os0; v.os1 = p.os1; v.os2 = p.os2;
  v.lse = p.lse; v.ls0 = p.ls0; v.ls1 = p.ls1;
  v.cu_q = p.cu_q; v.cq0 = p.cq0;
  v.sinks = p.sinks; v.sink_t = p.sink_t; v.si0 = p.si0;
  v.T = p.T; v.B = reqs; v.HQ = p.HQ; v.HK = p.c.HK; v.DQ = v.DV = p.c.D;
  v.causal = p.causal; v.win_l = p.win; v.win_r = -1; v.first = p.first;
  v.max_q = p.max_q; v.max_k = p.max_k; v.splits = 1;
  v.scale = p.scale;
  v.kmode = reinterpret_cast<const int32_t*>(uintptr_t(256));
  return v;
}

bool prefill_supported(const BlockAttn& p) {
  if (!(p.qt == FA_F16 || p.qt == FA_BF16) || p.max_k < 1 || p.c.D % 16 || p.c.D > 256) return false;
  if (!(p.scale >= 0x1p-60f)) return false;  // the prefill takes maxima of raw scores
  if (((uintptr_t)p.c.k & 15u) || ((uintptr_t)p.c.v & 15u)) return false;
  for (int64_t s : {p.c.ks0, p.c.ks1, p.c.ks2, p.c.vs0, p.c.vs1, p.c.vs2})
    if (s <= 0 || s % 16) return false;
  return prefill_sm100_supported(prefill_view(p, 1));
}

// Keys of a (request, KV head) with scales: whole key tiles, so that a tile reads its 128.
int64_t kfac_stride(const BlockAttn& p) { return ((int64_t)p.max_k + 127) / 128 * 128; }

int launch_prefill(const BlockAttn& p, const Plan& plan, void* workspace, cudaStream_t st) {
  uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
  for (int b0 = 0; b0 < p.B; b0 += plan.reqs) {
    const int n = std::min(plan.reqs, p.B - b0);
    CopyArgs a{};
    a.c = p.c;
    a.k = reinterpret_cast<uint16_t*>(ws + 256);
    a.v = reinterpret_cast<uint16_t*>(ws + 256 + plan.kv_bytes);
    a.kfac = reinterpret_cast<float*>(ws + 256 + 2 * plan.kv_bytes);
    a.kfac_stride = kfac_stride(p);
    a.per_log2 = 1.f / (p.scale * kLog2e);
    a.cu_out = reinterpret_cast<int32_t*>(ws + 256 + 2 * plan.kv_bytes + plan.fac_bytes);
    a.used_out = a.cu_out + plan.reqs + 1;
    a.mode = reinterpret_cast<int32_t*>(ws + 256 + 2 * plan.kv_bytes + plan.fac_bytes + plan.len_bytes);
    a.reset = reinterpret_cast<int32_t*>(ws);
    a.cu_q = p.cu_q; a.cq0 = p.cq0;
    a.used = p.used; a.u0 = p.u0;
    a.b0 = b0; a.B = n; a.max_k = p.max_k; a.win = p.win; a.first = p.first;
    const dim3 grid((unsigned)(kfac_stride(p) / 16), (unsigned)n);  // whole key tiles
    const dim3 heads((unsigned)p.c.HK, (unsigned)n);
    if (p.qt == FA_BF16) block_mode_kernel<true><<<heads, 256, 0, st>>>(a);
    else block_mode_kernel<false><<<heads, 256, 0, st>>>(a);
    note_launch();
    FAB_LAUNCH_CHECK("block-scaled prefill scale launch");
    if (p.qt == FA_BF16) block_copy_kernel<true><<<grid, 256, 0, st>>>(a);
    else block_copy_kernel<false><<<grid, 256, 0, st>>>(a);
    note_launch();
    FAB_LAUNCH_CHECK("block-scaled prefill copy launch");
    AttnParams v = prefill_view(p, n);
    v.k = a.k; v.v = a.v;
    v.cu_k = a.cu_out; v.ck0 = 1;
    v.used = a.used_out; v.u0 = 1;
    v.cu_q = p.cu_q + (int64_t)b0 * p.cq0;
    v.scratch = ws;
    v.kmode = a.mode; v.kfac = a.kfac; v.kfac_stride = a.kfac_stride;
    for (int codes = 0; codes < 2; ++codes) {
      v.codes = codes;
      const int rc = launch_prefill_sm100(v, st);
      if (rc) return rc;
    }
  }
  return FA_OK;
}

int fill(const fa_block_attention_args* g, BlockAttn* p) {
  *p = BlockAttn{};
  FAB_CHECK_ARG(g != nullptr, "null arguments");
  FAB_CHECK_ARG(g->batch >= 1 && g->batch <= 65535, "batch must be 1..65535");
  int rc = parse_block_cache(g->cache, g->batch, &p->c);
  if (rc) return rc;
  FAB_CHECK_ARG(present(g->q) && g->q.ndim == 3 && is_float(g->q.dtype) && g->q.shape[2] == p->c.D &&
                    g->q.shape[0] < (1LL << 31),
                "q must be float [tokens, heads, dim] with the cache's head dim");
  FAB_CHECK_ARG(g->q.shape[1] >= 1 && g->q.shape[1] <= 65535 && g->q.shape[1] % p->c.HK == 0,
                "query heads must be a positive multiple of KV heads");
  FAB_CHECK_ARG(present(g->out) && g->out.ndim == 3 && g->out.dtype == g->q.dtype && g->out.shape[0] == g->q.shape[0] &&
                    g->out.shape[1] == g->q.shape[1] && g->out.shape[2] == g->q.shape[2],
                "out must have q's shape and dtype");
  FAB_CHECK_ARG(present(g->lse) && g->lse.ndim == 2 && g->lse.dtype == FA_F32 && g->lse.shape[0] == g->q.shape[1] &&
                    g->lse.shape[1] == g->q.shape[0],
                "lse must be float32 [heads, tokens]");
  FAB_CHECK_ARG(present(g->cu_seqlens_q) && g->cu_seqlens_q.dtype == FA_I32 && g->cu_seqlens_q.ndim == 1 &&
                    g->cu_seqlens_q.shape[0] == g->batch + 1,
                "cu_seqlens_q must be int32 [batch + 1]");
  FAB_CHECK_ARG(present(g->seqlens) && g->seqlens.dtype == FA_I32 && g->seqlens.ndim == 1 && g->seqlens.shape[0] == g->batch,
                "seqlens must be int32 [batch]");
  FAB_CHECK_ARG(!present(g->s_aux) || (is_float(g->s_aux.dtype) && g->s_aux.ndim == 1 && g->s_aux.shape[0] == g->q.shape[1]),
                "s_aux must have one value per query head");
  FAB_CHECK_ARG(g->max_seqlen_q >= 0 && g->max_seqlen_k >= 0, "sequence lengths must be nonnegative");
  FAB_CHECK_ARG(g->first_tokens >= 0 && g->num_splits >= 0 && g->num_splits <= 1024,
                "first_tokens must be nonnegative, num_splits in 0..1024");
  p->q = g->q.ptr; p->qt = g->q.dtype;
  p->qs0 = g->q.stride[0]; p->qs1 = g->q.stride[1]; p->qs2 = g->q.stride[2];
  p->out = g->out.ptr; p->os0 = g->out.stride[0]; p->os1 = g->out.stride[1]; p->os2 = g->out.stride[2];
  p->lse = (float*)g->lse.ptr; p->ls0 = g->lse.stride[0]; p->ls1 = g->lse.stride[1];
  p->cu_q = (const int32_t*)g->cu_seqlens_q.ptr; p->cq0 = g->cu_seqlens_q.stride[0];
  p->used = (const int32_t*)g->seqlens.ptr; p->u0 = g->seqlens.stride[0];
  if (present(g->s_aux)) { p->sinks = g->s_aux.ptr; p->sink_t = g->s_aux.dtype; p->si0 = g->s_aux.stride[0]; }
  p->T = (int32_t)g->q.shape[0]; p->B = g->batch; p->HQ = (int32_t)g->q.shape[1];
  // Bounds of any size up to 2^31 - 1 may be given: beyond the rows, the block
  // table and 2^30 keys they mean no more than these, and their sums and
  // differences stay within 32 bits.
  const int32_t capacity = std::min(p->c.bt_cols * p->c.page, 1 << 30);
  p->max_q = std::min(g->max_seqlen_q, p->T); p->max_k = std::min(g->max_seqlen_k, capacity);
  p->causal = g->causal != 0;
  p->win = g->window_left < 0 || g->window_left >= capacity ? -1 : g->window_left;
  p->first = p->win >= 0 ? std::min(g->first_tokens, capacity) : 0;
  p->splits = g->num_splits;
  p->scale = g->softmax_scale;
  return FA_OK;
}

// Whether the copy and the prefill take less time than the decode kernel, both
// in us per 128 keys of every request. A decode CTA spends 0.8 us on a tile
// with up to 8 columns, 1.0 with 16 and 1.8 with 24 or 32 (a third more above
// 128 dims); the prefill 2.35 us on a tile of one item (a row block of 128
// queries, of two heads where they pair), items in waves of one per SM, behind
// the copy's 3 bytes per element. 8 requests, 32/8 heads, 8192 keys, measured
// decode / copy and prefill: 16 queries 99 / 231 us, 32: 187 / 231, 48: 255 /
// 231, 128: 701 / 231; one request: 64 queries 58 / 163, 256: 185 / 163; head
// dim 256, 4 requests: 32 queries 131 / 219, 64: 234 / 219.
bool prefill_pays(const BlockAttn& p) {
  if (p.max_q < 16) return false;
  const int block = block_decode_columns(p), cols = p.max_q * (p.HQ / p.c.HK);
  const double tile = (block <= 8 ? 0.8 : block == 16 ? 1.0 : 1.8) * (p.c.D > 128 ? 1.33 : 1.0);
  const double decode = tile * p.B * p.c.HK * ((cols + block - 1) / block) / sm_count();
  const bool pairs = p.c.D <= 128 && (p.HQ / p.c.HK) % 2 == 0;
  const double items = (double)p.B * (pairs ? p.HQ / 2 : p.HQ) * ((p.max_q + 127) / 128);
  const double prefill = 2.35 * std::ceil(items / sm_count()) + (double)p.B * 128 * p.c.HK * 2 * p.c.D * 3 / 6.5e6;
  return prefill < decode;
}

void make_plan(const BlockAttn& p, Plan* plan) {
  *plan = Plan{kAny, 1, 0, 0, 0, 0, 0};
  // An explicit number of pieces is a decode plan.
  const bool decode = block_decode_supported(p);
  if (p.splits == 0 && prefill_supported(p) && (!decode || prefill_pays(p))) {
    plan->route = kPrefill;
    const int64_t one = (int64_t)p.max_k * p.c.HK * p.c.D * 2;
    const int64_t rows = (1LL << 30) / p.max_k - 1;
    plan->reqs = (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)p.B, kPrefillCopy / (2 * one), rows}));
    plan->kv_bytes = up256((size_t)plan->reqs * one);
    plan->fac_bytes = up256((size_t)plan->reqs * p.c.HK * 3 * kfac_stride(p) * sizeof(float));
    plan->len_bytes = up256((size_t)(2 * plan->reqs + 1) * 4);
    plan->bytes = 256 + 2 * plan->kv_bytes + plan->fac_bytes + plan->len_bytes + up256((size_t)plan->reqs * p.c.HK * 4);
  } else if (decode) {
    plan->route = kDecode;
    plan->splits = block_decode_splits(p);
    plan->bytes = block_decode_workspace(p, plan->splits);
  }
}

}  // namespace
}  // namespace fab

using namespace fab;

extern "C" int fa_block_attention_workspace_size(const fa_block_attention_args* g, size_t* bytes) {
  FAB_CHECK_ARG(bytes != nullptr, "bytes must not be null");
  *bytes = 0;
  BlockAttn p;
  int rc = fill(g, &p);
  if (rc || p.T == 0) return rc;
  Plan plan;
  make_plan(p, &plan);
  *bytes = plan.bytes;
  return FA_OK;
}

extern "C" int fa_block_attention_fwd(const fa_block_attention_args* g, void* stream) {
  BlockAttn p;
  int rc = fill(g, &p);
  if (rc || p.T == 0) return rc;
  FAB_CHECK_ARG(p.max_q >= 1, "nonempty q requires a positive max_seqlen_q");
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  Plan plan;
  make_plan(p, &plan);
  if (plan.bytes)
    FAB_CHECK_ARG(present(g->workspace) && g->workspace.ndim >= 1 &&
                      (size_t)g->workspace.shape[0] * elem_size(g->workspace.dtype) >= plan.bytes &&
                      ((uintptr_t)g->workspace.ptr & 255u) == 0,
                  "workspace smaller than fa_block_attention_workspace_size, or not 256-byte aligned");
  if (plan.route == kPrefill) return launch_prefill(p, plan, g->workspace.ptr, st);
  if (plan.route == kDecode) return launch_block_decode(p, plan.splits, g->workspace.ptr, st);
  block_attention_any_kernel<<<dim3((unsigned)p.max_q, (unsigned)p.HQ, (unsigned)p.B), 128, 0, st>>>(p);
  note_launch();
  FAB_LAUNCH_CHECK("block-scaled attention launch");
  return FA_OK;
}
