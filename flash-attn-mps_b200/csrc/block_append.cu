// Rotation + append to a block-scaled E4M3 cache.
//
// Unit of work: the new rows of one (request, scale block, KV head) of K or of
// V. Their largest finite magnitude gives the block's scale 2^k (the least k
// with amax <= 448 * 2^k: with a floating code a power of two costs no
// precision, only half a bit of range, and rounding older codes to a larger
// scale is exact but for subnormal codes). A block that already holds tokens
// keeps the larger of its scale and the new one and re-rounds its older codes
// when the scale grew.
//
// Bound by HBM (2 bytes read and 1 written per K/V element, 2 + 2 per Q element)
// and, for the units, by instructions: 40928 tokens, 32/8 heads of 128, take
// 105 us for Q (6.0 TB/s) and 95 for K and V (2.6 TB/s of 251 MB). One launch,
// or two from kApart tokens on (one: 260 us together). The bf16 units are at their
// cap of 128 registers and spill 4 bytes a thread.
#include <algorithm>
#include <type_traits>

#include "block_cache.cuh"
#include "ptx.cuh"

namespace fab {
namespace {

constexpr int kApart = 512;  // tokens from which the queries take a launch of their own
constexpr int kMinExp = -100, kMaxExp = 100;

struct AppendArgs {
  BlockCache c;
  const void* x[2]; int64_t xs0[2], xs1[2], xs2[2];   // key, value
  const void* q; int64_t qs0, qs1, qs2;
  void* qo; int64_t qo0, qo1, qo2;
  int32_t xt, qt;
  const int32_t* cu; int64_t cu0;
  const int32_t* lens; int64_t l0;
  const float* cos; const float* sin; int64_t cs0, cs1, sn0, sn1;
  const int32_t* pos; int64_t ps0, ps1;               // ps0: axis, ps1: row
  const int32_t* axes; int64_t ax0;
  int32_t B, T, HQ, half, rows, n_axes, interleaved, max_new, units_per_req;
  // Vector kernel: warps of a CTA and of a unit, CTAs of K and V units; query
  // rows' heads are taken q_heads at a time.
  int32_t warps, unit_warps, q_heads;
};

// Least k with amax <= 448 * 2^k (448 = 1.75 * 2^8), within the scale range.
__device__ __forceinline__ int scale_exponent(float amax) {
  const uint32_t u = __float_as_uint(amax);
  if (u < 0x00800000u) return kMinExp;
  const int k = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);
  return min(max(k, kMinExp), kMaxExp);
}
__device__ __forceinline__ float exp2_int(int k) { return __uint_as_float((uint32_t)(k + 127) << 23); }
__device__ __forceinline__ float finite_abs(float x) {
  const float a = fabsf(x);
  return a < INFINITY ? a : 0.f;  // infinities and NaN do not set a scale
}

// Whether a request's new tokens begin within its table row (what lies behind it is skipped).
__device__ __forceinline__ bool starts_inside(const BlockCache& c, int start) {
  return start >= 0 && start >> c.page_shift < c.bt_cols;
}

// cos/sin of pair i at a token row; positions are clamped to the tables.
__device__ __forceinline__ int row_position(const AppendArgs& a, int axis, int64_t t, int abs_pos) {
  int p = abs_pos;
  if (a.pos) p = a.pos[(int64_t)min(max(axis, 0), a.n_axes - 1) * a.ps0 + t * a.ps1];
  return min(max(p, 0), a.rows - 1);
}

// ---- any layout: one thread per element, two passes over a unit's rows
__device__ __forceinline__ float rotated(const AppendArgs& a, const void* base, int dt, int64_t off, int64_t sd, int d,
                                         int64_t t, int abs_pos) {
  const float x = load_float(base, dt, off + d * sd);
  if (d >= 2 * a.half) return x;
  const int i = a.interleaved ? d >> 1 : (d < a.half ? d : d - a.half);
  const bool second = a.interleaved ? d & 1 : d >= a.half;
  const int partner = a.interleaved ? d ^ 1 : (second ? d - a.half : d + a.half);
  const int p = row_position(a, a.axes ? a.axes[i * a.ax0] : 0, t, abs_pos);
  const float c = a.cos[(int64_t)p * a.cs0 + i * a.cs1], s = a.sin[(int64_t)p * a.sn0 + i * a.sn1];
  const float y = load_float(base, dt, off + partner * sd);
  return second ? __fadd_rn(__fmul_rn(x, c), __fmul_rn(y, s)) : __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
}

__global__ void __launch_bounds__(256) block_append_any_kernel(const AppendArgs a) {
  const int b = blockIdx.y;
  const int begin = a.cu[b * a.cu0], n = a.cu[(b + 1) * a.cu0] - begin;
  if (n <= 0) return;
  const int start = a.lens[b * a.l0];
  if (a.q && blockIdx.z == 2) {
    // Rotated queries of this request: a thread forms both elements of a pair
    // before it writes them (query_out may be query), the rest one by one.
    const int per_row = a.c.D - a.half;
    const int64_t total = (int64_t)n * a.HQ * per_row, step = (int64_t)gridDim.x * blockDim.x;
    for (int64_t e = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; e < total; e += step) {
      const int i = (int)(e % per_row);
      const int64_t r = e / per_row;
      const int h = (int)(r % a.HQ);
      const int j = (int)(r / a.HQ);
      const int64_t t = begin + j, src = t * a.qs0 + h * a.qs1, dst = t * a.qo0 + h * a.qo1;
      const int d0 = i >= a.half ? i + a.half : a.interleaved ? 2 * i : i, d1 = a.interleaved ? d0 + 1 : d0 + a.half;
      const float x0 = rotated(a, a.q, a.qt, src, a.qs2, d0, t, start + j);
      const float x1 = i < a.half ? rotated(a, a.q, a.qt, src, a.qs2, d1, t, start + j) : 0.f;
      store_float(a.qo, a.qt, dst + d0 * a.qo2, x0);
      if (i < a.half) store_float(a.qo, a.qt, dst + d1 * a.qo2, x1);
    }
    return;
  }
  const int side = blockIdx.z;
  const BlockCache& c = a.c;
  const int h = blockIdx.x % c.HK, u = blockIdx.x / c.HK;
  const int blk = (start >> c.block_shift) + u;
  const int base = blk << c.block_shift;
  if (!starts_inside(c, start) || base >= start + n) return;
  const int pg = block_page(c, b, base);
  if (pg < 0) return;
  const int r0 = max(start - base, 0), r1 = min(start + n - base, c.block);
  const int tok0 = base & (c.page - 1);
  const int64_t s0 = side ? c.vs0 : c.ks0, s1 = side ? c.vs1 : c.ks1, s2 = side ? c.vs2 : c.ks2;
  uint8_t* dst = (side ? c.v : c.k) + (int64_t)pg * s0 + (int64_t)tok0 * s1 + (int64_t)h * s2;
  float* scp = side ? c.vsc + (int64_t)pg * c.vc0 + (int64_t)(tok0 >> c.block_shift) * c.vc1 + h * c.vc2
                    : c.ksc + (int64_t)pg * c.kc0 + (int64_t)(tok0 >> c.block_shift) * c.kc1 + h * c.kc2;
  const int D = c.D;
  auto value = [&](int r, int d) {
    const int j = base + r - start;
    const int64_t t = begin + j;
    const int64_t off = t * a.xs0[side] + (int64_t)h * a.xs1[side];
    return side ? load_float(a.x[1], a.xt, off + d * a.xs2[1])
                : rotated(a, a.x[0], a.xt, off, a.xs2[0], d, t, start + j);
  };
  float amax = 0.f;
  for (int e = threadIdx.x; e < (r1 - r0) * D; e += blockDim.x) amax = fmaxf(amax, finite_abs(value(r0 + e / D, e % D)));
  __shared__ float red[8];
  amax = warp_max(amax);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = amax;
  const float old = r0 > 0 ? *scp : 0.f;
  __syncthreads();
  amax = red[0];
  for (int w = 1; w < 8; ++w) amax = fmaxf(amax, red[w]);
  const float need = exp2_int(scale_exponent(amax));
  const float scale = r0 > 0 ? fmaxf(old, need) : need;
  for (int e = threadIdx.x; e < (r1 - r0) * D; e += blockDim.x) {
    const int r = r0 + e / D, d = e % D;
    dst[r * s1 + d] = float_to_e4m3_sat(__fdiv_rn(value(r, d), scale));
  }
  if (r0 > 0 && scale > old) {
    const float f = __fdiv_rn(old, scale);
    for (int e = threadIdx.x; e < r0 * D; e += blockDim.x) {
      uint8_t* p = dst + (e / D) * s1 + e % D;
      *p = float_to_e4m3_sat(e4m3_to_float(*p) * f);
    }
  }
  if (threadIdx.x == 0) *scp = scale;
}

// ---- 16-bit rows with unit inner strides
//
// A row is D / 16 groups of 16 elements: in the rotated part of a split-half
// row 8 first and their 8 second elements, else 16 neighbours. A lane owns
// group (lane % groups) of every (32 / groups)'th row, 4 rows at a time, and
// keeps its 64 values in registers between the maximum and the codes, so every
// element is read once. The units are bound by instructions before memory, so
// products are packed (f32x2, each rounded as its scalar), a maximum
// that comes out infinite is the sign to look again for the finite one, and
// divisions by a power of two multiply.
constexpr int kPasses = 4;

struct Group { int o1, o2; bool rot, split; };  // element offsets of its two vectors of 8
__device__ __forceinline__ Group group_of(const AppendArgs& a, int g, bool rotary) {
  const bool rot = rotary && 16 * g < 2 * a.half;
  if (rot && !a.interleaved) return {8 * g, a.half + 8 * g, true, true};
  return {16 * g, 16 * g + 8, rot, false};
}

// Four floats of a table. Volatile keeps the passes' loads where they stand: the
// compiler otherwise lifts all four passes' angles to the front and spills.
__device__ __forceinline__ float4 table4(const float* p) {
  float4 v;
  asm volatile("ld.global.nc.v4.f32 {%0, %1, %2, %3}, [%4];\n" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "l"(p));
  return v;
}

// cos/sin of the 8 pairs of group g at token row t, a half (4 pairs) each.
struct Angles { float4 c, s; };
// at0: the row's position on axis 0.
__device__ __forceinline__ void angles_of(const AppendArgs& a, int g, int64_t t, int abs_pos, int at0, Angles (&r)[2]) {
  const int i0 = 8 * g;
  if (!a.axes) {
    const float* c = a.cos + (int64_t)at0 * a.cs0 + i0;
    const float* s = a.sin + (int64_t)at0 * a.sn0 + i0;
    r[0].c = table4(c); r[1].c = table4(c + 4);
    r[0].s = table4(s); r[1].s = table4(s + 4);
    return;
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int ax[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) ax[i] = __ldg(a.axes + (int64_t)(i0 + 4 * h + i) * a.ax0);
    if (ax[1] == ax[0] && ax[2] == ax[0] && ax[3] == ax[0]) {
      const int p = row_position(a, ax[0], t, abs_pos);
      r[h].c = table4(a.cos + (int64_t)p * a.cs0 + i0 + 4 * h);
      r[h].s = table4(a.sin + (int64_t)p * a.sn0 + i0 + 4 * h);
    } else {
      float c[4], s[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int q = row_position(a, ax[i], t, abs_pos);
        c[i] = __ldg(a.cos + (int64_t)q * a.cs0 + i0 + 4 * h + i);
        s[i] = __ldg(a.sin + (int64_t)q * a.sn0 + i0 + 4 * h + i);
      }
      r[h].c = make_float4(c[0], c[1], c[2], c[3]);
      r[h].s = make_float4(s[0], s[1], s[2], s[3]);
    }
  }
}

template <bool BF16>
__device__ __forceinline__ float2 two_of(uint32_t w) {
  if constexpr (BF16) return unpack2<__nv_bfloat16>(w);
  else return unpack2<__half>(w);
}
// Half h of a group (vectors v1, v2): words 2 h and 2 h + 1 of each vector, so of a
// split-half row 4 first elements and their 4 seconds.
template <bool BF16>
__device__ __forceinline__ void half_of(const uint4& v1, const uint4& v2, int h, float* x) {
  const uint32_t w[4] = {h ? v1.z : v1.x, h ? v1.w : v1.y, h ? v2.z : v2.x, h ? v2.w : v2.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = two_of<BF16>(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint64_t pair64(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void split64(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t mul64(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// Two pairs (u0, v0), (u1, v1) at once, products and sums rounded one by one.
// (Packed sums of packed products came out fused; the scalar ones do not.)
__device__ __forceinline__ void turn2(float& u0, float& u1, float& v0, float& v1, uint64_t c, uint64_t s) {
  const uint64_t u = pair64(u0, u1), v = pair64(v0, v1);
  float uc0, uc1, vs0, vs1, vc0, vc1, us0, us1;
  split64(mul64(u, c), uc0, uc1);
  split64(mul64(v, s), vs0, vs1);
  split64(mul64(v, c), vc0, vc1);
  split64(mul64(u, s), us0, us1);
  u0 = __fsub_rn(uc0, vs0); u1 = __fsub_rn(uc1, vs1);
  v0 = __fadd_rn(vc0, us0); v1 = __fadd_rn(vc1, us1);
}
// Rotates the 4 pairs of half h in place. Neighbouring pairs: two from each vector.
__device__ __forceinline__ void rotate_half(float* x, const Angles (&r)[2], int h, bool split) {
  if (split) {
    turn2(x[0], x[1], x[4], x[5], pair64(r[h].c.x, r[h].c.y), pair64(r[h].s.x, r[h].s.y));
    turn2(x[2], x[3], x[6], x[7], pair64(r[h].c.z, r[h].c.w), pair64(r[h].s.z, r[h].s.w));
  } else {
    auto two = [&](const float4& v) { return h ? pair64(v.z, v.w) : pair64(v.x, v.y); };
    turn2(x[0], x[2], x[1], x[3], two(r[0].c), two(r[0].s));
    turn2(x[4], x[6], x[5], x[7], two(r[1].c), two(r[1].s));
  }
}

__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {  // saturating, NaN kept
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | (uint32_t)hi << 16;
}

template <bool BF16>
__device__ void append_queries(const AppendArgs& a, int cta) {
  // One thread: one group of a token for q_heads heads, the angles read once.
  const int groups = a.c.D / 16, hsteps = a.HQ / a.q_heads;
  const int64_t e = (int64_t)cta * blockDim.x + threadIdx.x;
  const int g = (int)(e % groups);
  const int64_t r = e / groups;
  const int hs = (int)(r % hsteps);
  const int64_t t = r / hsteps;
  if (t >= a.T) return;
  const Group gr = group_of(a, g, true);
  const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + t * a.qs0 + (int64_t)hs * a.q_heads * a.qs1;
  uint16_t* dst = reinterpret_cast<uint16_t*>(a.qo) + t * a.qo0 + (int64_t)hs * a.q_heads * a.qo1;
  Angles an[2];
  const bool turn = gr.rot;
  uint4 v1[4], v2[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < a.q_heads) {
      v1[i] = __ldcs(reinterpret_cast<const uint4*>(src + i * a.qs1 + gr.o1));
      v2[i] = __ldcs(reinterpret_cast<const uint4*>(src + i * a.qs1 + gr.o2));
    }
  if (turn) {
    int abs_pos = 0;
    if (!a.pos) {  // the request of row t: last b with cu[b] <= t
      int lo = 0, hi = a.B;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if ((int64_t)__ldg(a.cu + mid * a.cu0) <= t) lo = mid;
        else hi = mid;
      }
      abs_pos = __ldg(a.lens + lo * a.l0) + (int)(t - __ldg(a.cu + lo * a.cu0));
    }
    angles_of(a, g, t, abs_pos, row_position(a, 0, t, abs_pos), an);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < a.q_heads) {
      if (turn) {
        uint32_t w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float x[8];
          half_of<BF16>(v1[i], v2[i], h, x);
          rotate_half(x, an, h, !a.interleaved);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (BF16) w[h][k] = pack2<__nv_bfloat16>(x[2 * k], x[2 * k + 1]);
            else w[h][k] = pack2<__half>(x[2 * k], x[2 * k + 1]);
          }
        }
        v1[i] = make_uint4(w[0][0], w[0][1], w[1][0], w[1][1]);
        v2[i] = make_uint4(w[0][2], w[0][3], w[1][2], w[1][3]);
      }
      *reinterpret_cast<uint4*>(dst + i * a.qo1 + gr.o1) = v1[i];
      *reinterpret_cast<uint4*>(dst + i * a.qo1 + gr.o2) = v2[i];
    }
}

// The queries by themselves: above a few hundred tokens their own launch, at a
// higher occupancy than the K and V units allow, outweighs its latency.
template <bool BF16>
__global__ void __launch_bounds__(256) block_rotate_kernel(const AppendArgs a) { append_queries<BF16>(a, blockIdx.x); }

template <bool BF16, int WARPS, bool QUERIES>
__global__ void __launch_bounds__(WARPS * 32, WARPS == 8 ? 2 : 1) block_append_vec_kernel(const AppendArgs a) {
  const int b = blockIdx.y;
  if constexpr (QUERIES) {
    if (b >= a.B) {
      append_queries<BF16>(a, (b - a.B) * gridDim.x + blockIdx.x);
      return;
    }
  }
  const BlockCache& c = a.c;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per_cta = a.warps / a.unit_warps;
  const int in_cta = warp / a.unit_warps, sub = warp - in_cta * a.unit_warps;
  const int begin = __ldg(a.cu + b * a.cu0), n = __ldg(a.cu + (b + 1) * a.cu0) - begin, start = __ldg(a.lens + b * a.l0);
  // Unit: heads fastest, then K and V, then blocks: a CTA's warps write neighbouring rows.
  const int id = blockIdx.x * per_cta + in_cta, hs = id / c.HK, h = id - hs * c.HK, side = hs & 1, u = hs >> 1;
  const int base = ((start >> c.block_shift) + u) << c.block_shift;
  bool live = in_cta < per_cta && u < a.units_per_req && n > 0 && starts_inside(c, start) && base < start + n;
  if (!__syncthreads_or(live)) return;
  const int r0 = max(start - base, 0), r1 = live ? min(start + n - base, c.block) : 0;
  const int tok0 = base & (c.page - 1);
  const int groups = c.D / 16, per = 32 / groups;         // rows of a pass
  const int lr = lane / groups, g = lane - lr * groups;
  const Group gr = group_of(a, g, side == 0);
  const uint16_t* src = reinterpret_cast<const uint16_t*>(a.x[side]) + (int64_t)h * a.xs1[side];
  const int row0 = r0 + sub * kPasses * per + lr;          // this lane's first row of the block
  const int rows = lr < per ? r1 : 0;
  uint4 v1[kPasses], v2[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = row0 + i * per;
    v1[i] = v2[i] = make_uint4(0, 0, 0, 0);
    if (r < rows) {
      const uint16_t* row = src + (int64_t)(begin + base + r - start) * a.xs0[side];
      v1[i] = __ldcs(reinterpret_cast<const uint4*>(row + gr.o1));
      v2[i] = __ldcs(reinterpret_cast<const uint4*>(row + gr.o2));
    }
  }
  int at[kPasses];  // positions ahead of the angles that hang on them
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = row0 + i * per, j = base + r - start;
    at[i] = gr.rot && !a.axes && r < rows ? row_position(a, 0, (int64_t)begin + j, start + j) : 0;
  }
  const int pg = live ? block_page(c, b, base) : -1;
  live = pg >= 0;
  const int64_t s1 = side ? c.vs1 : c.ks1;
  uint8_t* dst = (side ? c.v : c.k) + (int64_t)pg * (side ? c.vs0 : c.ks0) + (int64_t)tok0 * s1 + (int64_t)h * (side ? c.vs2 : c.ks2);
  float* scp = side ? c.vsc + (int64_t)pg * c.vc0 + (int64_t)(tok0 >> c.block_shift) * c.vc1 + h * c.vc2
                    : c.ksc + (int64_t)pg * c.kc0 + (int64_t)(tok0 >> c.block_shift) * c.kc1 + h * c.kc2;
  const float old = live && r0 > 0 ? *scp : 0.f;
  float x[kPasses][16];  // [pass][half][8]
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = row0 + i * per, j = base + r - start;
    half_of<BF16>(v1[i], v2[i], 0, x[i]);
    half_of<BF16>(v1[i], v2[i], 1, x[i] + 8);
    if (gr.rot && r < rows) {
      Angles an[2];
      angles_of(a, g, (int64_t)begin + j, start + j, at[i], an);
      rotate_half(x[i], an, 0, !a.interleaved);
      rotate_half(x[i] + 8, an, 1, !a.interleaved);
    }
  }
  float of_pass[kPasses];
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    of_pass[i] = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) of_pass[i] = fmaxf(of_pass[i], fabsf(x[i][k]));  // NaN is passed over
  }
  static_assert(kPasses == 4, "maximum");
  float amax = fmaxf(fmaxf(of_pass[0], of_pass[1]), fmaxf(of_pass[2], of_pass[3]));
  if (amax == INFINITY) {
    amax = 0.f;
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) amax = fmaxf(amax, finite_abs(x[i][k]));
  }
  amax = warp_max(amax);
  if (a.unit_warps > 1) {
    __shared__ float red[16];
    if (lane == 0) red[warp] = amax;
    __syncthreads();
    if (in_cta < per_cta)
      for (int w = 0; w < a.unit_warps; ++w) amax = fmaxf(amax, red[in_cta * a.unit_warps + w]);
  }
  if (!live) return;
  const float need = exp2_int(scale_exponent(amax));
  const float scale = r0 > 0 ? fmaxf(old, need) : need;
  // A power of two (all that this library writes) divides by multiplying.
  if ((__float_as_uint(scale) & 0x807fffffu) == 0 && scale >= 0x1p-126f && scale <= 0x1p126f) {
    const float f = 1.f / scale;
    const uint64_t inv = pair64(f, f);
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
#pragma unroll
      for (int k = 0; k < 16; k += 2) split64(mul64(pair64(x[i][k], x[i][k + 1]), inv), x[i][k], x[i][k + 1]);
  } else {
#pragma unroll
    for (int i = 0; i < kPasses; ++i)
#pragma unroll
      for (int k = 0; k < 16; ++k) x[i][k] = __fdiv_rn(x[i][k], scale);
  }
#pragma unroll
  for (int i = 0; i < kPasses; ++i) {
    const int r = row0 + i * per;
    if (r >= rows) continue;
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = e4m3x4(x[i][4 * k], x[i][4 * k + 1], x[i][4 * k + 2], x[i][4 * k + 3]);
    uint8_t* row = dst + (int64_t)r * s1;
    if (gr.split) {
      *reinterpret_cast<uint2*>(row + gr.o1) = make_uint2(w[0], w[2]);
      *reinterpret_cast<uint2*>(row + gr.o2) = make_uint2(w[1], w[3]);
    } else {
      *reinterpret_cast<uint4*>(row + gr.o1) = make_uint4(w[0], w[2], w[1], w[3]);
    }
  }
  if (r0 > 0 && scale > old) {
    // Older codes of the block, rounded to the larger scale.
    const float f = __fdiv_rn(old, scale);
    for (int e = sub * 32 + lane; e < r0 * groups; e += a.unit_warps * 32) {
      uint4* p = reinterpret_cast<uint4*>(dst + (int64_t)(e / groups) * s1 + (e % groups) * 16);
      uint32_t w[4] = {p->x, p->y, p->z, p->w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        uint32_t lo, hi;
        e4m3x4_to_f16x2x2(w[k], lo, hi);
        const float2 u0 = unpack2<__half>(lo), u1 = unpack2<__half>(hi);
        w[k] = e4m3x4(u0.x * f, u0.y * f, u1.x * f, u1.y * f);
      }
      *p = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
  if (sub == 0 && lane == 0) *scp = scale;
}

// The vector kernel's conditions: 16-byte vectors everywhere.
bool vector_rows(const AppendArgs& a) {
  auto al = [](const void* p, uintptr_t n) { return ((uintptr_t)p & (n - 1)) == 0; };
  if (a.xt != FA_F16 && a.xt != FA_BF16) return false;
  if (a.c.D % 16 || a.c.D > 256) return false;
  for (int i = 0; i < 2; ++i)
    if (a.xs2[i] != 1 || a.xs0[i] % 8 || a.xs1[i] % 8 || !al(a.x[i], 16)) return false;
  for (int64_t s : {a.c.ks0, a.c.ks1, a.c.ks2, a.c.vs0, a.c.vs1, a.c.vs2})
    if (s % 16) return false;
  if (!al(a.c.k, 16) || !al(a.c.v, 16)) return false;
  if (a.q && (a.qt != a.xt || a.qs2 != 1 || a.qo2 != 1 || a.qs0 % 8 || a.qs1 % 8 || a.qo0 % 8 || a.qo1 % 8 || !al(a.q, 16) ||
              !al(a.qo, 16)))
    return false;
  if (a.half && (a.half % 8 || a.cs1 != 1 || a.sn1 != 1 || a.cs0 % 4 || a.sn0 % 4 || !al(a.cos, 16) || !al(a.sin, 16)))
    return false;
  return true;
}

int check_rows(const fa_tensor& t, const char* name, int64_t T, int D, int dtype) {
  FAB_CHECK_ARG(present(t) && t.ndim == 3 && t.shape[0] == T && t.shape[2] == D && t.dtype == dtype,
                "%s must be [tokens, heads, dim] of one dtype", name);
  return FA_OK;
}

}  // namespace

int parse_block_cache(const fa_block_cache& c, int32_t batch, BlockCache* o) {
  *o = BlockCache{};
  FAB_CHECK_ARG(present(c.k) && present(c.v) && c.k.ndim == 4 && c.v.ndim == 4 && c.k.dtype == FA_E4M3 &&
                    c.v.dtype == FA_E4M3,
                "block-scaled caches must be float8_e4m3fn [pages, page, heads, dim]");
  for (int i = 0; i < 4; ++i)
    FAB_CHECK_ARG(c.k.shape[i] == c.v.shape[i], "block-scaled K and V caches must have one shape");
  const int64_t page = c.k.shape[1];
  FAB_CHECK_ARG(page >= 16 && page <= 65536 && (page & (page - 1)) == 0,
                "block-scaled caches need a power-of-two page size of 16..65536 tokens");
  FAB_CHECK_ARG(c.k.shape[0] >= 1 && c.k.shape[0] < (1LL << 31) && c.k.shape[2] >= 1 && c.k.shape[2] < (1 << 16),
                "block-scaled caches need pages and KV heads");
  FAB_CHECK_ARG(c.k.shape[3] >= 1 && c.k.shape[3] <= 512, "head dimension must be in 1..512");
  FAB_CHECK_ARG(c.k.stride[3] == 1 && c.v.stride[3] == 1, "block-scaled caches need a unit head-dim stride");
  const fa_tensor* sc[2] = {&c.k_scale, &c.v_scale};
  for (const fa_tensor* t : sc)
    FAB_CHECK_ARG(present(*t) && t->ndim == 3 && t->dtype == FA_F32 && t->shape[0] == c.k.shape[0] &&
                      t->shape[1] == c.k_scale.shape[1] && t->shape[2] == c.k.shape[2],
                  "block scales must be float32 [pages, page / block, heads]");
  const int64_t nb = c.k_scale.shape[1];
  FAB_CHECK_ARG(nb >= 1 && page % nb == 0, "block scales must divide the page into equal blocks");
  const int64_t block = page / nb;
  FAB_CHECK_ARG(block >= 16 && block <= 128 && (block & (block - 1)) == 0,
                "scale blocks must hold 16, 32, 64 or 128 tokens");
  FAB_CHECK_ARG(present(c.block_table) && c.block_table.ndim == 2 && c.block_table.dtype == FA_I32 &&
                    c.block_table.shape[0] == batch && c.block_table.shape[1] >= 1 &&
                    c.block_table.shape[1] < (1LL << 31) / page,
                "block_table must be int32 [batch, pages]");
  o->k = (uint8_t*)c.k.ptr; o->v = (uint8_t*)c.v.ptr;
  o->ks0 = c.k.stride[0]; o->ks1 = c.k.stride[1]; o->ks2 = c.k.stride[2];
  o->vs0 = c.v.stride[0]; o->vs1 = c.v.stride[1]; o->vs2 = c.v.stride[2];
  o->ksc = (float*)c.k_scale.ptr; o->vsc = (float*)c.v_scale.ptr;
  o->kc0 = c.k_scale.stride[0]; o->kc1 = c.k_scale.stride[1]; o->kc2 = c.k_scale.stride[2];
  o->vc0 = c.v_scale.stride[0]; o->vc1 = c.v_scale.stride[1]; o->vc2 = c.v_scale.stride[2];
  o->table = (const int32_t*)c.block_table.ptr;
  o->bt0 = c.block_table.stride[0]; o->bt1 = c.block_table.stride[1];
  o->bt_cols = (int32_t)c.block_table.shape[1];
  o->pages = c.k.shape[0];
  o->page = (int32_t)page; o->block = (int32_t)block;
  while ((1 << o->page_shift) < o->page) ++o->page_shift;
  while ((1 << o->block_shift) < o->block) ++o->block_shift;
  o->HK = (int32_t)c.k.shape[2]; o->D = (int32_t)c.k.shape[3];
  return FA_OK;
}

}  // namespace fab

using namespace fab;

extern "C" int fa_append_block_scaled(const fa_block_append_args* g, void* stream) {
  FAB_CHECK_ARG(g != nullptr, "null arguments");
  FAB_CHECK_ARG(g->batch >= 1 && g->batch <= 65535 && g->max_seqlen >= 0, "batch must be 1..65535, max_seqlen nonnegative");
  AppendArgs a{};
  int rc = parse_block_cache(g->cache, g->batch, &a.c);
  if (rc) return rc;
  FAB_CHECK_ARG(present(g->key) && g->key.ndim == 3 && is_float(g->key.dtype), "key must be float [tokens, heads, dim]");
  const int64_t T = g->key.shape[0];
  FAB_CHECK_ARG(T < (1LL << 31), "too many tokens");
  if ((rc = check_rows(g->key, "key", T, a.c.D, g->key.dtype))) return rc;
  if ((rc = check_rows(g->value, "value", T, a.c.D, g->key.dtype))) return rc;
  FAB_CHECK_ARG(g->key.shape[1] == a.c.HK && g->value.shape[1] == a.c.HK, "key/value heads must match the cache");
  FAB_CHECK_ARG(present(g->cu_seqlens) && g->cu_seqlens.dtype == FA_I32 && g->cu_seqlens.ndim == 1 &&
                    g->cu_seqlens.shape[0] == g->batch + 1,
                "cu_seqlens must be int32 [batch + 1]");
  FAB_CHECK_ARG(present(g->seqlens) && g->seqlens.dtype == FA_I32 && g->seqlens.ndim == 1 && g->seqlens.shape[0] == g->batch,
                "seqlens must be int32 [batch]");
  a.B = g->batch; a.T = (int32_t)T; a.max_new = std::min(g->max_seqlen, a.T);  // any upper bound may be given
  a.x[0] = g->key.ptr; a.x[1] = g->value.ptr; a.xt = g->key.dtype;
  const fa_tensor* xs[2] = {&g->key, &g->value};
  for (int i = 0; i < 2; ++i) { a.xs0[i] = xs[i]->stride[0]; a.xs1[i] = xs[i]->stride[1]; a.xs2[i] = xs[i]->stride[2]; }
  if (present(g->query)) {
    FAB_CHECK_ARG(is_float(g->query.dtype), "query must be float");
    FAB_CHECK_ARG(g->query.ndim == 3 && g->query.shape[1] >= 1, "query must have heads");
    if ((rc = check_rows(g->query, "query", T, a.c.D, g->query.dtype))) return rc;
    if ((rc = check_rows(g->query_out, "query_out", T, a.c.D, g->query.dtype))) return rc;
    FAB_CHECK_ARG(g->query_out.shape[1] == g->query.shape[1], "query_out must have the query's shape");
    a.q = g->query.ptr; a.qs0 = g->query.stride[0]; a.qs1 = g->query.stride[1]; a.qs2 = g->query.stride[2];
    a.qo = g->query_out.ptr; a.qo0 = g->query_out.stride[0]; a.qo1 = g->query_out.stride[1]; a.qo2 = g->query_out.stride[2];
    a.qt = g->query.dtype; a.HQ = (int32_t)g->query.shape[1];
  }
  a.cu = (const int32_t*)g->cu_seqlens.ptr; a.cu0 = g->cu_seqlens.stride[0];
  a.lens = (const int32_t*)g->seqlens.ptr; a.l0 = g->seqlens.stride[0];
  FAB_CHECK_ARG(present(g->cos) == present(g->sin), "rotary cosine and sine go together");
  if (present(g->cos)) {
    FAB_CHECK_ARG(g->cos.dtype == FA_F32 && g->sin.dtype == FA_F32 && g->cos.ndim == 2 && g->sin.ndim == 2 &&
                      g->cos.shape[0] == g->sin.shape[0] && g->cos.shape[1] == g->sin.shape[1] && g->cos.shape[0] >= 1 &&
                      g->cos.shape[0] < (1LL << 31) && 2 * g->cos.shape[1] <= a.c.D,
                  "rotary cosine/sine must be float32 [positions, rotary_dim/2]");
    a.cos = (const float*)g->cos.ptr; a.sin = (const float*)g->sin.ptr;
    a.cs0 = g->cos.stride[0]; a.cs1 = g->cos.stride[1]; a.sn0 = g->sin.stride[0]; a.sn1 = g->sin.stride[1];
    a.half = (int32_t)g->cos.shape[1]; a.rows = (int32_t)g->cos.shape[0];
    a.interleaved = g->interleaved != 0;
  }
  if (present(g->positions)) {
    FAB_CHECK_ARG(g->positions.dtype == FA_I32 && (g->positions.ndim == 1 || g->positions.ndim == 2) &&
                      g->positions.shape[g->positions.ndim - 1] == T,
                  "positions must be int32 [tokens] or [axes, tokens]");
    a.pos = (const int32_t*)g->positions.ptr;
    FAB_CHECK_ARG(g->positions.ndim == 1 || (g->positions.shape[0] >= 1 && g->positions.shape[0] < (1 << 16)),
                  "positions must have at least one axis");
    a.n_axes = g->positions.ndim == 2 ? (int32_t)g->positions.shape[0] : 1;
    a.ps0 = g->positions.ndim == 2 ? g->positions.stride[0] : 0;
    a.ps1 = g->positions.stride[g->positions.ndim - 1];
  }
  if (present(g->rotary_axes)) {
    FAB_CHECK_ARG(g->rotary_axes.dtype == FA_I32 && g->rotary_axes.ndim == 1 && g->rotary_axes.shape[0] == a.half,
                  "rotary_axes must be int32 [rotary_dim/2]");
    a.axes = (const int32_t*)g->rotary_axes.ptr; a.ax0 = g->rotary_axes.stride[0];
  }
  if (T == 0 || g->max_seqlen == 0) return FA_OK;
  a.units_per_req = (int32_t)(((int64_t)a.max_new + a.c.block - 2) / a.c.block + 1);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (vector_rows(a)) {
    const int groups = a.c.D / 16, rows = kPasses * (32 / groups);
    a.unit_warps = (std::min(a.c.block, a.max_new) + rows - 1) / rows;
    a.warps = a.unit_warps > 8 ? 16 : 8;
    const int per_cta = a.warps / a.unit_warps;
    const int64_t kv = ((int64_t)a.units_per_req * 2 * a.c.HK + per_cta - 1) / per_cta;  // CTAs of a request
    int64_t q_ctas = 0;
    const bool apart = a.q && T >= kApart;
    if (a.q) {
      a.q_heads = a.HQ % 4 == 0 ? 4 : a.HQ % 2 == 0 ? 2 : 1;
      const int threads = apart ? 256 : a.warps * 32;
      q_ctas = ((int64_t)T * (a.HQ / a.q_heads) * groups + threads - 1) / threads;
    }
    FAB_CHECK_ARG(kv < (1LL << 31) && q_ctas < (1LL << 31), "too many tokens for one append");
    const bool bf16 = a.xt == FA_BF16;
    if (apart) {
      (bf16 ? block_rotate_kernel<true> : block_rotate_kernel<false>)<<<(unsigned)q_ctas, 256, 0, st>>>(a);
      note_launch();
      FAB_LAUNCH_CHECK("block-scaled rotation launch");
      q_ctas = 0;
    }
    const int64_t q_rows = (q_ctas + kv - 1) / kv;  // grid rows behind the requests'
    FAB_CHECK_ARG(a.B + q_rows <= 65535, "too many requests for one append");
    auto pick = [&](auto with_q) {
      constexpr bool Q = decltype(with_q)::value;
      return a.warps == 8 ? (bf16 ? block_append_vec_kernel<true, 8, Q> : block_append_vec_kernel<false, 8, Q>)
                          : (bf16 ? block_append_vec_kernel<true, 16, Q> : block_append_vec_kernel<false, 16, Q>);
    };
    auto kernel = q_ctas ? pick(std::true_type{}) : pick(std::false_type{});
    kernel<<<dim3((unsigned)kv, (unsigned)(a.B + q_rows)), a.warps * 32, 0, st>>>(a);
    note_launch();
    FAB_LAUNCH_CHECK("block-scaled append launch");
    return FA_OK;
  }
  FAB_CHECK_ARG((int64_t)a.units_per_req * a.c.HK < (1LL << 31), "too many tokens for one append");
  const dim3 grid((unsigned)(a.units_per_req * a.c.HK), (unsigned)a.B, a.q ? 3u : 2u);
  block_append_any_kernel<<<grid, 256, 0, st>>>(a);
  note_launch();
  FAB_LAUNCH_CHECK("block-scaled append launch");
  return FA_OK;
}
