// Decode over a block-scaled E4M3 cache on the 5th-generation tensor cores.
//
// A column is one query row of a request and one head of a KV head's group; a
// CTA works on one KV head and up to C columns, so a few drafted tokens share
// every K/V byte. Per tile of 128 keys
//   S^T [128 keys x N] = K [128 x D] Q^T          (A = K tile, K-major)
//   O^T [D x N]        = V^T [D x 128] P^T        (A = V tile, MN-major)
// as tcgen05.mma kind::f8f6f4 straight from the codes in shared memory: no
// code is converted in registers, which bounds a decode that unpacks E4M3 for
// 16-bit products.
//   * Q becomes a sum of E4M3 parts, part i scaled by 2^(4 i): 2 parts hold 8
//     bits of a query (bf16), 3 parts 12 (f16), for elements down to 2^-14 of
//     the row's largest; smaller ones to 2^-22 (2^-26) of it. The parts are extra
//     columns of the same MMA (N = 16 is its least width).
//   * P becomes a sum of E5M2 parts, part i scaled by 2^(3 i): 3 parts for bf16
//     hold a probability to 2^-9, as the 16-bit type itself would, 4 for f16 to
//     2^-12, down to 2^-29 of the tile's largest (20 nats; of p vs, which is what
//     the tile's maximum is taken of); below that the error
//     stays under 2^-38 (2^-41) of the largest. The wide exponent matters where
//     the largest keys add nothing to an output (an attention sink's V row is
//     close to zero): E4M3 parts, which hold 2^-14, lost such rows.
//   * Thread t owns key t of the tile: the block scales are one factor and one
//     addend per thread, t_j = s_j * ks_j + log2(vs_j); the row sum takes
//     p_j / vs_j (see block_attention.cu).
//   * P is scaled by the tile's own maximum and O^T read back per tile and
//     summed in registers (N values per thread): relative to the tile rather
//     than to the running maximum no long tail is lost behind one dominant key.
//
// Persistent and balanced: the visible tiles of all requests form one list;
// group g of the G groups takes tiles [g T / G, (g+1) T / G) of it, for each
// KV head (and block of columns) one CTA, so neighbouring CTAs read
// neighbouring heads of the same pages and ragged batches end together. A
// request that lies within one group is written directly, else its pieces
// (at most two unfinished ones per group) go to the workspace and
// block_merge_kernel joins them. Short requests and windows take a CTA each
// instead (by_request; block_decode_splits): a few tiles one after another cost
// less than the second launch.
//
// Warps 0..4 WG-1: softmax and accumulation (thread = key of S^T, then head
// dim of O^T; WG warpgroups of CT columns each: up to 16 columns one warpgroup,
// with 3 CTAs per SM for 4 columns and 2 above, then 8 columns a thread with one
// CTA); then one warp that gathers K
// pages by TMA and writes scales and unit records, one that issues MMAs, one
// that splits queries, one that gathers V pages (a second issuer of page boxes:
// 16-token pages make 16 boxes a tile, and one warp issued them at 4.2 TB/s).
// Rings decouple them, so the gathers run on into the next request.
// HBM-bound: D bytes of K and of V per key and KV head, once for all columns.
// 32 requests x 32768 tokens, 32/8 heads of 128, 16-token pages: 348 us, 6.2 TB/s
// of K and V (page 64: 330, 6.5); the library's mma.sync decode of a cache with one
// descale per head takes 428. More columns are bound by the softmax warps: 8192
// tokens, 4 / 8 / 16 / 24 / 32 columns a KV head 96 / 110 / 133 / 183 / 198 us
// (bf16; f16 with its fourth part 96 / 109 / 138 / 185 / 203) one call behind
// another. Their arithmetic goes two columns to an instruction (f32x2; column
// by column 6 % slower at 16 to 32 columns). Prompts of 32-column blocks alone
// are 5 to 9 % slower than with two E4M3 parts. Of the shapes bf16 rows of 256
// with 32 columns spill 16 bytes.
//
// Every wait is bounded; on a timeout the CTA records a flag, drains its own
// copies and MMAs, frees tensor memory and returns.
#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <cstring>

#include "block_cache.cuh"
#include "prefill_common.cuh"
#include "ptx.cuh"
#include "sm100.cuh"

namespace fab {
namespace {

using namespace sm100;
using pf::fadd2;
using pf::ffma2;
using pf::fmul2;
using pf::f2pack;
using pf::f2unpack;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kBias = 15.f;         // probabilities up to 2^15 (E5M2 ends at 57344)
constexpr float kUnbias = 0x1p-15f;   // 2^-kBias: row sums are kept without it
constexpr int kKeys = 128;            // keys per tile
constexpr int kUnitRing = 4;          // unit records in shared memory

__device__ int g_block_decode_timeout;

// NP: parts of a query; a probability has one more.
template <int NP, int C, int DH>
struct Shape {
  static constexpr int N = (NP * C + 15) / 16 * 16;         // columns of S^T
  static constexpr int NV = ((NP + 1) * C + 15) / 16 * 16;  // columns of O^T
  static constexpr int CT = C < 8 || C == 16 ? C : 8;     // columns per softmax thread
  static constexpr int WG = C / CT;                       // softmax warpgroups
  static constexpr int kThreads = WG * 128 + 128;
  static constexpr int kItem = kKeys * 128 * DH;          // bytes of a K or V tile
  // P^T of a tile. With 4 columns K-major rows of 128 keys (least space), else
  // MN-major: a key's N codes side by side, so that a thread stores its own in
  // 8- or 16-byte pieces instead of byte by byte (f16, 32 columns: 1720 -> 900
  // cycles a tile); rows of 32, 64 or 128 bytes, swizzled as wide.
  static constexpr bool kPmn = C >= 8;
  static constexpr int PW = NV <= 32 ? 32 : NV <= 64 ? 64 : 128;
  static constexpr int kQ = N * 128 * DH, kP = kPmn ? kKeys * PW : NV * 128;
  // CTAs per SM that the shape asks for, and tiles whose scales are kept: a K
  // slot of tile t + kRing comes free only after tile t's scales are read when
  // kRing >= K slots + 2.
  static constexpr int kMany = C > 16 || DH > 1 ? 1 : C > 4 ? 2 : 3;
  static constexpr int kRing = kMany > 2 ? 4 : 8;
  // Tables behind the tiles (byte offsets).
  static constexpr int kHolder = 384, kRec = 400, kCol = 592, kScale = kCol + 16 * C;
  static constexpr int kWmax = kScale + kRing * 8 * 16, kSum = kWmax + 32 * C, kMrow = kSum + 32 * C, kFac = (kMrow + 8 * C + 15) / 16 * 16;
  static constexpr int kMisc = (kFac + (CT >= 8 ? 96 * CT * WG : 0) + 255) / 256 * 256;
  static constexpr uint32_t cols() {
    uint32_t got = 32;
    while (got < 2 * N + 2 * NV * DH) got *= 2;
    return got;
  }
  static constexpr uint32_t kCols = cols();               // tensor memory: S^T and O^T, two buffers each
  // Ring slots of one K or V tile each: even ones K, odd ones V (so that the
  // two gather warps each see every phase of the barriers that they wait on).
  static constexpr int kFixed = 1024 + kMisc + 2 * kQ + 2 * kP;
  static constexpr int fit(int ctas) { return (232448 / ctas - 1024 - kFixed) / kItem / 2 * 2; }
  static constexpr int kCtas = fit(kMany) >= 4 && kCols * kMany <= 512 ? kMany : 1;
  static constexpr int kMost = 2 * (kRing - 2);
  static constexpr int NSLOT = fit(kCtas) > kMost ? kMost : fit(kCtas) > 8 ? 8 : fit(kCtas);
  static constexpr int kSmem = kFixed + NSLOT * kItem;
  static_assert(NSLOT >= 4 && NSLOT % 2 == 0 && kRing >= NSLOT / 2 + 2, "ring");
  // Never more resident CTAs than tensor memory holds.
  static_assert(kCols * (232448 / (kSmem + 1024)) <= 512, "tensor memory");
  static constexpr int B_FULL = 0, B_EMPTY = 8, B_S = 16, B_P = 18, B_O = 20, B_QF = 22, B_QE = 24, B_UF = 26,
                       B_UE = B_UF + kUnitRing, B_X = B_UE + kUnitRing, B_FIN = B_X + 4, B_Q0 = B_FIN + 1, B_COUNT = B_Q0 + 1;
  static_assert(B_COUNT * 8 <= kHolder, "barriers");
};

__device__ __forceinline__ void mma_f8_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n"
      " tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
// E4M3 x E4M3 (b_e5m2: x E5M2) -> f32; a_mn, b_mn: operand stored MN-major.
__host__ __device__ constexpr uint32_t f8_idesc(int M, int N, int a_mn, int b_mn, int b_e5m2) {
  return (1u << 4) | ((uint32_t)b_e5m2 << 10) | ((uint32_t)a_mn << 15) | ((uint32_t)b_mn << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}
// Descriptor of an MN-major tile with rows of W bytes, swizzled over W bytes;
// the stride of 8-row groups along K is 8 W.
template <int W>
__device__ __forceinline__ uint64_t mn_desc(uint32_t saddr) {
  constexpr uint64_t kSwizzle = W == 128 ? 2 : W == 64 ? 4 : 6;
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | (uint64_t)1 << 16 | (uint64_t)(8 * W >> 4) << 32 | (uint64_t)1 << 46 | kSwizzle << 61;
}
template <int W>
__device__ __forceinline__ void tmem_ld(uint32_t taddr, uint32_t (&u)[W]) {
  static_assert(W == 4 || W == 8 || W == 16, "width");
  if constexpr (W == 4)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3])
                 : "r"(taddr));
  else if constexpr (W == 16)
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr));
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7])
                 : "r"(taddr));
}
// The parts of CT columns of a TMEM row (parts C columns apart, each 2^STEP
// times the one behind it) as one value each, two columns to a register pair.
template <int NP, int STEP, int C, int CT>
__device__ __forceinline__ void load_columns(uint32_t taddr, uint64_t (&x)[CT / 2]) {
  uint32_t r[NP][CT];
#pragma unroll
  for (int part = 0; part < NP; ++part) tmem_ld<CT>(taddr + part * C, r[part]);
  tmem_wait_ld();
  constexpr float kStep = 1.f / (1 << STEP);
  const uint64_t step = f2pack(kStep, kStep);
  auto two = [&](int part, int c) { return f2pack(__uint_as_float(r[part][c]), __uint_as_float(r[part][c + 1])); };
#pragma unroll
  for (int c = 0; c < CT; c += 2) {
    uint64_t s = two(NP - 1, c);
#pragma unroll
    for (int part = NP - 2; part >= 0; --part) s = ffma2(s, step, two(part, c));
    x[c / 2] = s;
  }
}

__device__ __forceinline__ float redux_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;\n" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t e4m3x2(float lo, float hi) {  // saturating, NaN kept
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float2 from_e4m3x2(uint32_t two) {
  const uint32_t h = e4m3x2_to_f16x2(two);
  return unpack2<__half>(h);
}
__device__ __forceinline__ uint32_t e5m2x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;\n" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
// An E5M2 code is the upper byte of the same value in f16.
__device__ __forceinline__ float2 from_e5m2x2(uint32_t two) { return unpack2<__half>(__byte_perm(two, 0, 0x1404)); }
__device__ __forceinline__ bool wait_all(uint32_t bar, uint32_t parity) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, &g_block_decode_timeout));
}

struct DecodeArgs {
  BlockAttn p;
  int32_t box_tok, cblocks, group, groups;  // group: query heads per KV head; groups: pieces of the tile list
  int32_t by_request;                       // group g is request g, whole
  int32_t q_vec;                            // query rows can be read 8 bytes at a time
  int4* info;                               // [B][cblocks] {first group, last group, begins a group, -}
};

// Tiles of a request that the columns from col0 on see: the first tokens'
// tiles, then those of [lo, len).
struct Extent {
  int n, len, first, lo, tiles;  // query rows, keys; first-token tiles, first tile behind them, all
  int lo_key;
};
__device__ __forceinline__ Extent extent_of(const BlockAttn& p, int n, int len, int col0, int group) {
  Extent e;
  e.n = n;
  e.len = len;
  e.lo_key = p.win >= 0 ? max(0, len - n + col0 / group - p.win) : 0;
  e.lo = e.lo_key / kKeys;
  e.first = min((p.first + kKeys - 1) / kKeys, e.lo);
  const int hi = len > 0 ? (len + kKeys - 1) / kKeys : 0;
  // A request without keys still has rows to write: one (masked) tile.
  e.tiles = n * group <= col0 ? 0 : max(1, e.first + max(0, hi - e.lo));
  return e;
}

// Sum of a warp's values and the exclusive sum up to each lane.
__device__ __forceinline__ int warp_scan(int v, int lane, int& total) {
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  total = __shfl_sync(0xffffffffu, x, 31);
  return x - v;
}

enum { R_B = 0, R_N, R_LEN, R_QB, R_FIRST, R_LO, R_LOKEY, R_I0, R_IT, R_SLOT, R_WORDS = 12 };

template <int NP, int C, int DH>
__global__ void __launch_bounds__(Shape<NP, C, DH>::kThreads, Shape<NP, C, DH>::kCtas)
    block_decode_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                        const DecodeArgs a) {
  using Sh = Shape<NP, C, DH>;
  constexpr int N = Sh::N, NV = Sh::NV, NPV = NP + 1, NSLOT = Sh::NSLOT, CT = Sh::CT, WG = Sh::WG;
  const BlockAttn& p = a.p;
  const int piece = blockIdx.y;                                   // group of the tile list
  const int kh = blockIdx.x / a.cblocks, cb = blockIdx.x - kh * a.cblocks;
  const int col0 = cb * C;

  extern __shared__ uint8_t smem_raw[];
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  uint8_t* gbase = smem_raw + (base - raw);
  constexpr int kOffQ = NSLOT * Sh::kItem, kOffP = kOffQ + 2 * Sh::kQ, kOffMisc = kOffP + 2 * Sh::kP;
  auto bar = [&](int i) { return base + kOffMisc + 8u * (uint32_t)i; };
  uint8_t* misc = gbase + kOffMisc;
  volatile uint32_t* holder = reinterpret_cast<volatile uint32_t*>(misc + Sh::kHolder);
  volatile int* rec = reinterpret_cast<volatile int*>(misc + Sh::kRec);      // [kUnitRing][R_WORDS]
  float* colfac = reinterpret_cast<float*>(misc + Sh::kCol);                 // [2][C] scale * log2e * 2^e of the query
  int* col_pos = reinterpret_cast<int*>(misc + Sh::kCol + 8 * C);            // [2][C] query position
  float4* scales = reinterpret_cast<float4*>(misc + Sh::kScale);             // [kRing][8] {ks, log2 vs, 2^-kBias / vs}
  float* wmax = reinterpret_cast<float*>(misc + Sh::kWmax);                  // [WG][2][4][CT]
  float* sums = reinterpret_cast<float*>(misc + Sh::kSum);                   // [2 units][WG][4][CT]
  float* mrow = reinterpret_cast<float*>(misc + Sh::kMrow);                  // [2 units][C]
  float* fac = reinterpret_cast<float*>(misc + Sh::kFac);                    // [4 WG warps][2][3][CT], CT >= 8 only
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  if (tid == 0) {
    for (int s = 0; s < NSLOT; ++s) {
      mbar_init(bar(Sh::B_FULL + s), 2);              // the copies, and what the gather warp writes beside them
      mbar_init(bar(Sh::B_EMPTY + s), 1);
    }
    for (int s = 0; s < 2; ++s) {
      mbar_init(bar(Sh::B_S + s), 2);                 // MMA commit + the issuing thread (orders the scales)
      mbar_init(bar(Sh::B_P + s), 128 * WG);
      mbar_init(bar(Sh::B_O + s), 1);
      mbar_init(bar(Sh::B_QF + s), 32);
      mbar_init(bar(Sh::B_QE + s), 1 + 4 * WG);
    }
    for (int s = 0; s < kUnitRing; ++s) {
      mbar_init(bar(Sh::B_UF + s), 1);
      mbar_init(bar(Sh::B_UE + s), 3 + 4 * WG);       // MMA, V gather, query and softmax warps
    }
    for (int w = 0; w < WG; ++w) mbar_init(bar(Sh::B_X + w), 128);
    mbar_init(bar(Sh::B_FIN), 1);
    mbar_init(bar(Sh::B_Q0), 128 * WG);
    mbar_fence_init();
  }
  // Sequence offsets and lengths of the requests (the K gather warp's lanes).
  auto request = [&](int b, int& q_begin) {
    const bool in = b < p.B && (!a.by_request || b == piece);
    q_begin = in ? p.cu_q[b * p.cq0] : 0;
    const int n = in ? p.cu_q[(b + 1) * p.cq0] - q_begin : 0;
    return extent_of(p, n, in ? p.used[b * p.u0] : 0, col0, a.group);
  };
  const int b_first = a.by_request ? piece / 32 * 32 : 0, b_last = a.by_request ? b_first + 32 : p.B;
  int total = 0;  // tiles of all requests; read while the barriers are set up
  if (warp == 4 * WG) {
#pragma unroll 4
    for (int b0 = b_first; b0 < b_last; b0 += 32) {
      int q;
      total += request(b0 + lane, q).tiles;
    }
    total = __reduce_add_sync(0xffffffffu, total);
  }
  if (warp == 4 * WG + 1) {
    tmem_alloc(smem_addr(const_cast<uint32_t*>(holder)), Sh::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *holder;
  asm volatile("griddepcontrol.launch_dependents;\n" ::: "memory");  // the merge waits for this grid's end itself

  // Unit u of this CTA, once the gather warp has published it (false: no more, or a timeout).
  auto next_unit = [&](int u) {
    if (!wait_all(bar(Sh::B_UF + u % kUnitRing), (u / kUnitRing) & 1)) return false;
    return rec[(u % kUnitRing) * R_WORDS + R_B] >= 0;
  };
  auto unit_done = [&](int u) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(Sh::B_UE + u % kUnitRing));
  };

  // Parts of column c's query for a unit of parity par, by one warp: rows
  // part * C + c of the B operand of S^T, K-major, 128-byte swizzle.
  auto split_query = [&](int par, int c, int n, int len, int q_begin) {
    const int cols = min(C, n * a.group - col0);
    uint8_t* qs = gbase + kOffQ + par * Sh::kQ;
    const bool real = c < cols;
    const int qi = (col0 + c) / a.group, h = kh * a.group + (col0 + c) - qi * a.group;
    float x[DH][4];
    float amax = 0.f;
    bool odd = false;
    const int64_t row = (int64_t)(q_begin + qi) * p.qs0 + (int64_t)h * p.qs1;
#pragma unroll
    for (int hf = 0; hf < DH; ++hf) {
      const int d0 = hf * 128 + lane * 4;
      x[hf][0] = x[hf][1] = x[hf][2] = x[hf][3] = 0.f;
      if (real && d0 < p.c.D) {
        if (a.q_vec) {  // D is a multiple of 16: the four dims are there together
          const uint2 w = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p.q) + row + d0));
          const float2 lo = p.qt == FA_BF16 ? unpack2<__nv_bfloat16>(w.x) : unpack2<__half>(w.x);
          const float2 hi = p.qt == FA_BF16 ? unpack2<__nv_bfloat16>(w.y) : unpack2<__half>(w.y);
          x[hf][0] = lo.x; x[hf][1] = lo.y; x[hf][2] = hi.x; x[hf][3] = hi.y;
        } else {
#pragma unroll
          for (int i = 0; i < 4; ++i) x[hf][i] = load_float(p.q, p.qt, row + (d0 + i) * p.qs2);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        amax = fmaxf(amax, fabsf(x[hf][i]));
        odd |= !(fabsf(x[hf][i]) < INFINITY);
      }
    }
    amax = redux_max(amax);
    odd = __any_sync(0xffffffffu, odd);
    // 2^e with amax * 2^-e in [128, 256), e within the exponents of a float.
    const int e = min(max((int)(__float_as_uint(amax) >> 23) - 127 - 7, -118), 119);
    const float down = __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
    for (int hf = 0; hf < DH; ++hf) {
      float y[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) y[i] = x[hf][i] * down;
#pragma unroll
      for (int part = 0; part < NP; ++part) {
        const uint32_t lo = e4m3x2(y[0], y[1]), hi = e4m3x2(y[2], y[3]);
        const int row = part * C + c;
        *reinterpret_cast<uint32_t*>(qs + hf * N * 128 + (row >> 3) * 1024 + (row & 7) * 128 +
                                     (((lane >> 2) ^ (row & 7)) << 4) + (lane & 3) * 4) = lo | (hi << 16);
        const float2 f0 = from_e4m3x2(lo), f1 = from_e4m3x2(hi);
        y[0] = (y[0] - f0.x) * 16.f; y[1] = (y[1] - f0.y) * 16.f;
        y[2] = (y[2] - f1.x) * 16.f; y[3] = (y[3] - f1.y) * 16.f;
      }
    }
    if (lane == 0) {
      // A query with an infinity or NaN has no finite score.
      colfac[par * C + c] = !real ? 0.f : odd ? __uint_as_float(0x7fc00000u)
                                                  : p.scale * kLog2e * __uint_as_float((uint32_t)(127 + e) << 23);
      col_pos[par * C + c] = real ? len - n + qi : -1;
    }
  };

  // Query parts of unit u are there: the first unit's by all softmax threads,
  // then each parity's by the query warp.
  auto wait_queries = [&](int u) {
    if (u == 0) return wait_all(bar(Sh::B_Q0), 0);
    return wait_all(bar(Sh::B_QF + (u & 1)), ((u >> 1) - (u & 1 ? 0 : 1)) & 1);
  };

  if (warp == 4 * WG) {
    // ------------------------------------------- units, page gathers and scales
    if (lane == 0) {
      tma_prefetch_desc(&tmk);
      tma_prefetch_desc(&tmv);
    }
    // Every group that takes part has a tile.
    const int groups = a.by_request ? 1 : min(a.groups, total), g = a.by_request ? 0 : piece;
    const int t0 = g < groups ? (int)((int64_t)g * total / groups) : 0;
    const int t1 = g < groups ? (int)((int64_t)(g + 1) * total / groups) : 0;
    const int nbox = kKeys / a.box_tok, boxes = DH * nbox;
    const int half = lane / nbox, bx = lane - half * nbox;
    const int nblk = kKeys >> p.c.block_shift;
    // Lanes below 16: one box each; lanes 16..23: one scale block each.
    const bool is_box = lane < boxes, is_blk = lane >= 16 && lane - 16 < nblk;
    const int lane_off = is_box ? bx * a.box_tok : (lane - 16) << p.c.block_shift;
    int gt = 0, u = 0, pre = 0;
    bool ok = true;
    for (int b0 = b_first; ok && b0 < b_last && pre < t1; b0 += 32) {
      int q_lane, sum;
      const Extent e_lane = request(b0 + lane, q_lane);
      const int pre_lane = pre + warp_scan(e_lane.tiles, lane, sum);
      if (a.info && kh == 0 && e_lane.tiles > 0 && pre_lane >= t0 && pre_lane < t1) {
        // The group that holds a request's first tile says which groups hold it.
        const int last = (int)(((int64_t)(pre_lane + e_lane.tiles) * groups - 1) / total);
        a.info[(b0 + lane) * a.cblocks + cb] = make_int4(piece, last, pre_lane == t0, 0);
      }
      pre += sum;
      // Records go out one unit ahead of the copies, so that the next unit's
      // queries are split while this one's tiles arrive.
      auto publish = [&](int src) {
        if (u >= kUnitRing && !wait_all(bar(Sh::B_UE + u % kUnitRing), ((u / kUnitRing) - 1) & 1)) return false;
        if (lane == src) {
          const int i0 = max(t0 - pre_lane, 0), n_it = min(t1 - pre_lane, e_lane.tiles) - i0;
          volatile int* r = rec + (u % kUnitRing) * R_WORDS;
          r[R_B] = b0 + src; r[R_N] = e_lane.n; r[R_LEN] = e_lane.len; r[R_QB] = q_lane; r[R_FIRST] = e_lane.first;
          r[R_LO] = e_lane.lo; r[R_LOKEY] = e_lane.lo_key; r[R_I0] = i0; r[R_IT] = n_it;
          r[R_SLOT] = n_it == e_lane.tiles ? -1 : 2 * piece + (pre_lane > t0 ? 1 : 0);
          mbar_arrive(bar(Sh::B_UF + u % kUnitRing));
        }
        ++u;
        return true;
      };
      uint32_t m = __ballot_sync(0xffffffffu, e_lane.tiles > 0 && pre_lane < t1 && pre_lane + e_lane.tiles > t0);
      if (m) ok = publish(__ffs(m) - 1);
      for (; ok && m; m &= m - 1) {
        const int src = __ffs(m) - 1, b = b0 + src;
        if ((m & (m - 1)) && !(ok = publish(__ffs(m & (m - 1)) - 1))) break;
        auto get = [&](int x) { return __shfl_sync(0xffffffffu, x, src); };
        const int len = get(e_lane.len), t_first = get(e_lane.first), t_lo = get(e_lane.lo), tiles = get(e_lane.tiles);
        const int begin = get(pre_lane);
        const int i0 = max(t0 - begin, 0), n_it = min(t1 - begin, tiles) - i0;
        auto tile_of = [&](int i) { return i < t_first ? i : i - t_first + t_lo; };
        // Table entry of this lane's box or block, as it stands in the table.
        auto lookup = [&](int it) {
          const int pos = tile_of(i0 + it) * kKeys + lane_off;
          const int col = pos >> p.c.page_shift;
          return it < n_it && (is_box || is_blk) && pos < len && col < p.c.bt_cols
                     ? __ldg(p.c.table + (int64_t)b * p.c.bt0 + (int64_t)col * p.c.bt1) : -1;
        };
        auto load_scales = [&](int pg, int it, float& ks, float& vs) {
          ks = vs = 1.f;
          if (is_blk && pg >= 0 && (int64_t)pg < p.c.pages) {
            const int blk = ((tile_of(i0 + it) * kKeys + lane_off) & (p.c.page - 1)) >> p.c.block_shift;
            ks = __ldg(p.c.ksc + (int64_t)pg * p.c.kc0 + (int64_t)blk * p.c.kc1 + (int64_t)kh * p.c.kc2);
            vs = __ldg(p.c.vsc + (int64_t)pg * p.c.vc0 + (int64_t)blk * p.c.vc1 + (int64_t)kh * p.c.vc2);
          }
        };
        // Table entries are read three tiles ahead, scales one tile ahead of
        // the copies: neither latency is waited for tile by tile.
        int pg0 = lookup(0), pg1 = lookup(1), pg2 = lookup(2);
        float ks0, vs0, ks1, vs1;
        load_scales(pg0, 0, ks0, vs0);
        load_scales(pg1, 1, ks1, vs1);
        for (int it = 0; it < n_it; ++it, ++gt) {
          const int pg3 = lookup(it + 3);
          const int pos = tile_of(i0 + it) * kKeys + lane_off;
          const int page = pg0 >= 0 && (int64_t)pg0 < p.c.pages ? pg0 : -1;  // -1: zero fill
          const int item = 2 * gt, slot = item % NSLOT;
          if (item >= NSLOT && !(ok = wait_all(bar(Sh::B_EMPTY + slot), ((item / NSLOT) - 1) & 1))) break;
          if (lane == 0) mbar_expect_tx(bar(Sh::B_FULL + slot), Sh::kItem);
          __syncwarp();
          if (is_box)
            tma_load_4d(base + slot * Sh::kItem + half * (kKeys * 128) + bx * a.box_tok * 128, &tmk,
                        bar(Sh::B_FULL + slot), half * 128, kh, pos & (p.c.page - 1), page);
          // The tile that used this entry 8 tiles ago is done: its K slot came free since.
          if (is_blk) {
            const float s = clamp_scale(vs0);
            scales[(gt % Sh::kRing) * 8 + lane - 16] = make_float4(clamp_scale(ks0), log2f(s), kUnbias / s, 0.f);
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(bar(Sh::B_FULL + slot));
          ks0 = ks1; vs0 = vs1;
          load_scales(pg2, it + 2, ks1, vs1);
          pg0 = pg1; pg1 = pg2; pg2 = pg3;
        }
      }
    }
    if (ok && (u < kUnitRing || wait_all(bar(Sh::B_UE + u % kUnitRing), ((u / kUnitRing) - 1) & 1)) && lane == 0) {
      rec[(u % kUnitRing) * R_WORDS + R_B] = -1;
      mbar_arrive(bar(Sh::B_UF + u % kUnitRing));
    }
    // Every issued copy lands before the CTA leaves, after a time-out too.
    for (int i = max(0, 2 * gt - NSLOT); i < 2 * gt; ++i)
      if (i % 2 == 0) wait_all(bar(Sh::B_FULL + i % NSLOT), (i / NSLOT) & 1);
  } else if (warp == 4 * WG + 3) {
    // ----------------------------------------------------------- V page gathers
    const int nbox = kKeys / a.box_tok, boxes = DH * nbox;
    const int half = lane / nbox, bx = lane - half * nbox;
    int gt = 0;
    bool ok = true;
    for (int u = 0; ok && next_unit(u); ++u) {
      const volatile int* r = rec + (u % kUnitRing) * R_WORDS;
      const int b = r[R_B], len = r[R_LEN], t_first = r[R_FIRST], t_lo = r[R_LO], i0 = r[R_I0], n_it = r[R_IT];
      unit_done(u);
      auto position = [&](int it) {
        const int i = i0 + it;
        return (i < t_first ? i : i - t_first + t_lo) * kKeys + bx * a.box_tok;
      };
      auto lookup = [&](int it) {
        const int pos = position(it), col = pos >> p.c.page_shift;
        return it < n_it && lane < boxes && pos < len && col < p.c.bt_cols
                   ? __ldg(p.c.table + (int64_t)b * p.c.bt0 + (int64_t)col * p.c.bt1) : -1;
      };
      int pg0 = lookup(0), pg1 = lookup(1);
      for (int it = 0; it < n_it; ++it, ++gt) {
        const int pg2 = lookup(it + 2);
        const int item = 2 * gt + 1, slot = item % NSLOT;
        const int page = pg0 >= 0 && (int64_t)pg0 < p.c.pages ? pg0 : -1;
        if (item >= NSLOT && !(ok = wait_all(bar(Sh::B_EMPTY + slot), ((item / NSLOT) - 1) & 1))) break;
        if (lane == 0) {
          mbar_expect_tx(bar(Sh::B_FULL + slot), Sh::kItem);
          mbar_arrive(bar(Sh::B_FULL + slot));
        }
        __syncwarp();
        if (lane < boxes)
          tma_load_4d(base + slot * Sh::kItem + half * (kKeys * 128) + bx * a.box_tok * 128, &tmv, bar(Sh::B_FULL + slot),
                      half * 128, kh, position(it) & (p.c.page - 1), page);
        pg0 = pg1; pg1 = pg2;
      }
    }
    for (int i = max(0, 2 * gt - NSLOT); i < 2 * gt; ++i)
      if (i % 2 == 1) wait_all(bar(Sh::B_FULL + i % NSLOT), (i / NSLOT) & 1);
  } else if (warp == 4 * WG + 1) {
    // --------------------------------------------------------------------- MMA
    constexpr uint32_t kQk = f8_idesc(128, N, 0, 0, 0), kPv = f8_idesc(128, NV, 1, Sh::kPmn, 1);
    int gt = 0;
    bool ok = true;
    auto pv = [&](int t) {
      const int item = 2 * t + 1, slot = item % NSLOT;
      if (!wait_all(bar(Sh::B_FULL + slot), (item / NSLOT) & 1)) return false;
      if (!wait_all(bar(Sh::B_P + (t & 1)), (t >> 1) & 1)) return false;
      tc_fence_after();
      if (lane == 0) {
#pragma unroll
        for (int hf = 0; hf < DH; ++hf)
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            mma_f8_ss(tmem + 2 * N + (t & 1) * (NV * DH) + hf * NV,
                      sw128_desc(base + slot * Sh::kItem + hf * (kKeys * 128) + kk * 4096, 16, 1024),
                      Sh::kPmn ? mn_desc<Sh::PW>(base + kOffP + (t & 1) * Sh::kP + kk * 32 * Sh::PW)
                               : sw128_desc(base + kOffP + (t & 1) * Sh::kP + kk * 32, 16, 1024),
                      kPv, kk > 0);
        mma_commit(bar(Sh::B_O + (t & 1)));
        mma_commit(bar(Sh::B_EMPTY + slot));
      }
      __syncwarp();
      return true;
    };
    for (int u = 0; ok && next_unit(u); ++u) {
      const int n_it = rec[(u % kUnitRing) * R_WORDS + R_IT];
      unit_done(u);
      if (!(ok = wait_queries(u))) break;
      for (int it = 0; it < n_it; ++it, ++gt) {
        const int item = 2 * gt, slot = item % NSLOT;
        if (!(ok = wait_all(bar(Sh::B_FULL + slot), (item / NSLOT) & 1))) break;
        tc_fence_after();
        if (lane == 0) {
#pragma unroll
          for (int hf = 0; hf < DH; ++hf)
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              mma_f8_ss(tmem + (gt & 1) * N, sw128_desc(base + slot * Sh::kItem + hf * (kKeys * 128) + kk * 32, 16, 1024),
                        sw128_desc(base + kOffQ + (u & 1) * Sh::kQ + hf * (N * 128) + kk * 32, 16, 1024), kQk, (hf | kk) > 0);
          mma_commit(bar(Sh::B_S + (gt & 1)));
          mbar_arrive(bar(Sh::B_S + (gt & 1)));
          mma_commit(bar(Sh::B_EMPTY + slot));
          if (it + 1 == n_it) mma_commit(bar(Sh::B_QE + (u & 1)));
        }
        __syncwarp();
        if (it > 0 && !(ok = pv(gt - 1))) break;
      }
      if (ok) ok = pv(gt - 1);  // not behind the next unit's queries
    }
    // No MMA is in flight when tensor memory is released.
    if (lane == 0) mma_commit(bar(Sh::B_FIN));
    __syncwarp();
    wait_all(bar(Sh::B_FIN), 0);
  } else if (warp >= 4 * WG) {
    // ----------------------------------------------------------- query parts
    // Every unit's but the first, which the softmax warps split at the start.
    bool ok = true;
    for (int u = 0; ok && next_unit(u); ++u) {
      const volatile int* r = rec + (u % kUnitRing) * R_WORDS;
      const int n = r[R_N], len = r[R_LEN], q_begin = r[R_QB];
      unit_done(u);
      if (u == 0) continue;
      if (u >= 2 && !(ok = wait_all(bar(Sh::B_QE + (u & 1)), ((u >> 1) - 1) & 1))) break;
#pragma unroll 4
      for (int c = 0; c < C; ++c) split_query(u & 1, c, n, len, q_begin);
      fence_proxy_async_smem();
      mbar_arrive(bar(Sh::B_QF + (u & 1)));
    }
  } else {
    // ----------------------------------------------------------------- softmax
    const int wg = warp >> 2, wq = warp & 3, key_i = tid & 127;
    const uint32_t lane_off = (uint32_t)(wq * 32) << 16;
    const int c0 = wg * CT;                        // this warpgroup's columns [c0, c0 + CT)
    // Factors of tile t: minus the reference, the old sums' factor, the tile's.
    auto myfac = [&](int t, int k) { return fac + ((warp * 2 + (t & 1)) * 3 + k) * CT; };
    auto pair_at = [&](const float* v, int c) { return *reinterpret_cast<const uint64_t*>(v + c); };
    int gt = 0, xs = 0;                            // tiles, exchanges so far
    bool ok = true;
    for (int u = 0; ok && next_unit(u); ++u) {
      const volatile int* r_ = rec + (u % kUnitRing) * R_WORDS;
      const int n = r_[R_N], len = r_[R_LEN], q_begin = r_[R_QB], t_first = r_[R_FIRST], t_lo = r_[R_LO];
      const int lo_key = r_[R_LOKEY], i0 = r_[R_I0], n_it = r_[R_IT], part_slot = r_[R_SLOT];
      unit_done(u);
      const int cols = min(C, n * a.group - col0);
      const int first_pos = len - n + col0 / a.group, last_pos = len - n + (col0 + cols - 1) / a.group;
      const int hi_all = p.causal ? min(len, first_pos + 1) : len;      // keys that every column sees (but for windows)
      const int lo_all = p.win >= 0 ? last_pos - p.win : 0;
      if (u == 0) {
        for (int c = warp; c < C; c += 4 * WG) split_query(0, c, n, len, q_begin);
        fence_proxy_async_smem();
        mbar_arrive(bar(Sh::B_Q0));
      }
      if (!(ok = wait_queries(u))) break;
      const float* cf = colfac + (u & 1) * C + c0;
      const int* cp = col_pos + (u & 1) * C + c0;
      uint64_t o[DH][CT / 2], l[CT / 2];           // two columns each
#pragma unroll
      for (int c = 0; c < CT / 2; ++c) {
        l[c] = 0;
#pragma unroll
        for (int hf = 0; hf < DH; ++hf) o[hf][c] = 0;
      }
      float m_run[CT < 8 ? CT : 1];               // per column; from 8 columns on lane c holds column c's
#pragma unroll
      for (int c = 0; c < (CT < 8 ? CT : 1); ++c) m_run[c] = -INFINITY;
      float f_old[CT < 8 ? CT : 1], f_new[CT < 8 ? CT : 1];
      float g_old[CT < 8 ? CT : 1], g_new[CT < 8 ? CT : 1];
      // O^T of tile t: o = o * f + tile * g.
      auto take = [&](int t, const float* f, const float* g) {
        if (!wait_all(bar(Sh::B_O + (t & 1)), (t >> 1) & 1)) return false;
        tc_fence_after();
#pragma unroll
        for (int hf = 0; hf < DH; ++hf) {
          uint64_t x[CT / 2];
          load_columns<NPV, 3, C, CT>(tmem + 2 * N + (t & 1) * (NV * DH) + hf * NV + lane_off + c0, x);
#pragma unroll
          for (int c = 0; c < CT; c += 2) {
            uint64_t kf, kg;
            if constexpr (CT < 8) {
              kf = f2pack(f[c], f[c + 1]); kg = f2pack(g[c], g[c + 1]);
            } else {
              kf = pair_at(myfac(t, 1), c); kg = pair_at(myfac(t, 2), c);
            }
            o[hf][c / 2] = ffma2(o[hf][c / 2], kf, fmul2(x[c / 2], kg));
          }
        }
        return true;
      };
      for (int it = 0; it < n_it; ++it, ++gt) {
        const int ti = i0 + it, tile0 = (ti < t_first ? ti : ti - t_first + t_lo) * kKeys, key = tile0 + key_i;
        if (!(ok = wait_all(bar(Sh::B_S + (gt & 1)), (gt >> 1) & 1))) break;
        tc_fence_after();
        const float4 sc = scales[(gt % Sh::kRing) * 8 + (key_i >> p.c.block_shift)];
        float x[CT];
        {
          uint64_t s[CT / 2];
          load_columns<NP, 4, C, CT>(tmem + (gt & 1) * N + lane_off + c0, s);
          const uint64_t ks = f2pack(sc.x, sc.x), add = f2pack(sc.y, sc.y);
#pragma unroll
          for (int c = 0; c < CT; c += 2) f2unpack(ffma2(s[c / 2], fmul2(ks, pair_at(cf, c)), add), x[c], x[c + 1]);
        }
        // Tiles that some column does not see whole: keys past the end, past a
        // drafted token's own position, before its window.
        if (!(tile0 + kKeys <= hi_all && (tile0 >= lo_all || tile0 + kKeys <= p.first))) {
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const int pos = cp[c];
            const bool seen = key < len && (!p.causal || key <= pos) && (p.win < 0 || key >= pos - p.win || key < p.first);
            x[c] = seen ? x[c] : -INFINITY;
          }
          // V rows that no column sees may hold anything: zero them, so that
          // nothing but zeros meets their zero probabilities.
          if (wg == 0 && (key >= len || (key < lo_key && key >= p.first))) {
            const int item = 2 * gt + 1, slot = item % NSLOT;
            if (mbar_wait(bar(Sh::B_FULL + slot), (item / NSLOT) & 1, &g_block_decode_timeout)) {
#pragma unroll
              for (int hf = 0; hf < DH; ++hf)
#pragma unroll
                for (int q4 = 0; q4 < 8; ++q4)
                  *reinterpret_cast<uint4*>(gbase + slot * Sh::kItem + hf * (kKeys * 128) + key_i * 128 + q4 * 16) =
                      make_uint4(0, 0, 0, 0);
            }
          }
          __syncwarp();
        }
        // The tile's maximum per column over the four warps.
        float mine = -INFINITY;
#pragma unroll
        for (int c = 0; c < CT; ++c) {
          const float m = redux_max(x[c]);
          if (lane == c) mine = m;
        }
        float* wm = wmax + (wg * 2 + (gt & 1)) * 4 * CT;
        if (lane < CT) wm[wq * CT + lane] = mine;
        mbar_arrive(bar(Sh::B_X + wg));
        if (!(ok = wait_all(bar(Sh::B_X + wg), xs & 1))) break;
        ++xs;
        float ref[CT < 8 ? CT : 1];
        if constexpr (CT < 8) {
#pragma unroll
          for (int c = 0; c < CT; ++c) { g_old[c] = f_old[c]; g_new[c] = f_new[c]; }
#pragma unroll
          for (int c = 0; c < CT; ++c) {
            const float mt = fmaxf(fmaxf(wm[c], wm[CT + c]), fmaxf(wm[2 * CT + c], wm[3 * CT + c]));
            const float m_new = fmaxf(m_run[c], mt);
            const float safe = m_new == -INFINITY ? 0.f : m_new;
            ref[c] = kBias - (mt == -INFINITY ? 0.f : mt);
            f_old[c] = fast_exp2(m_run[c] - safe);
            f_new[c] = fast_exp2(mt - safe);
            m_run[c] = m_new;
          }
        } else {
          if (lane < CT) {
            const float mt = fmaxf(fmaxf(wm[lane], wm[CT + lane]), fmaxf(wm[2 * CT + lane], wm[3 * CT + lane]));
            const float m_new = fmaxf(m_run[0], mt);
            const float safe = m_new == -INFINITY ? 0.f : m_new;
            myfac(gt, 0)[lane] = kBias - (mt == -INFINITY ? 0.f : mt);
            myfac(gt, 1)[lane] = fast_exp2(m_run[0] - safe);
            myfac(gt, 2)[lane] = fast_exp2(mt - safe);
            m_run[0] = m_new;
          }
          __syncwarp();
        }
        // Probabilities: row sums in f32, E5M2 parts into the P^T tile.
        uint32_t codes[NPV][CT / 2];                 // two columns each
        const uint64_t per_v = f2pack(sc.z, sc.z), eight = f2pack(8.f, 8.f), minus = f2pack(-1.f, -1.f);
#pragma unroll
        for (int c = 0; c < CT; c += 2) {
          uint64_t r, f, g;
          if constexpr (CT < 8) {
            r = f2pack(ref[c], ref[c + 1]); f = f2pack(f_old[c], f_old[c + 1]); g = f2pack(f_new[c], f_new[c + 1]);
          } else {
            r = pair_at(myfac(gt, 0), c); f = pair_at(myfac(gt, 1), c); g = pair_at(myfac(gt, 2), c);
          }
          float p0, p1;
          f2unpack(fadd2(f2pack(x[c], x[c + 1]), r), p0, p1);
          p0 = fast_exp2(p0); p1 = fast_exp2(p1);
          uint64_t pp = f2pack(p0, p1);
          l[c / 2] = ffma2(l[c / 2], f, fmul2(pp, fmul2(per_v, g)));
#pragma unroll
          for (int part = 0; part < NPV; ++part) {
            f2unpack(pp, p0, p1);
            const uint32_t code = e5m2x2(p0, p1);
            codes[part][c / 2] = code;
            if (part + 1 < NPV) {  // 8 (p - code), exact
              const float2 d = from_e5m2x2(code);
              pp = fmul2(ffma2(f2pack(d.x, d.y), minus, pp), eight);
            }
          }
        }
        uint8_t* pt = gbase + kOffP + (gt & 1) * Sh::kP;
        if constexpr (Sh::kPmn) {
          // Swizzle over PW bytes: chunk (address bits 4..) XOR address bits 7.., PW / 16 of them.
          constexpr int kChunks = Sh::PW / 16;
          const uint32_t xr = (uint32_t)(key_i / (8 / kChunks)) & (kChunks - 1);
#pragma unroll
          for (int part = 0; part < NPV; ++part) {
            const uint32_t at = part * C + c0;
            uint8_t* d = pt + key_i * Sh::PW + (((at >> 4) ^ xr) << 4) + (at & 15);
            uint32_t w[CT / 4];
#pragma unroll
            for (int i = 0; i < CT / 4; ++i) w[i] = codes[part][2 * i] | codes[part][2 * i + 1] << 16;
            if constexpr (CT == 8) *reinterpret_cast<uint2*>(d) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint4*>(d) = make_uint4(w[0], w[1], w[CT / 4 - 2], w[CT / 4 - 1]);
          }
        } else {
          const uint32_t col = ((uint32_t)(key_i >> 4) << 4) + (key_i & 15);
#pragma unroll
          for (int part = 0; part < NPV; ++part)
#pragma unroll
            for (int c = 0; c < CT; ++c) {
              const int n0 = part * C + c;
              pt[(col ^ ((n0 & 7) << 4)) + (n0 >> 3) * 1024 + (n0 & 7) * 128] = (uint8_t)(codes[part][c / 2] >> (8 * (c & 1)));
            }
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(bar(Sh::B_P + (gt & 1)));
        if (it > 0 && !(ok = take(gt - 1, g_old, g_new))) break;
      }
      if (!ok) break;
      if (!(ok = take(gt - 1, f_old, f_new))) break;
      // ---- the unit's sums over the keys' threads, then its rows: thread = head
      // dim. Two units' sums take turns, so one exchange per unit is enough.
      float* ws = sums + ((u & 1) * WG + wg) * 4 * CT;
      float* ms = mrow + (u & 1) * C + c0;
#pragma unroll
      for (int c = 0; c < CT; c += 2) {
        float s0, s1;
        f2unpack(l[c / 2], s0, s1);
        s0 = warp_sum(s0);
        s1 = warp_sum(s1);
        if (lane == 0) { ws[wq * CT + c] = s0; ws[wq * CT + c + 1] = s1; }
      }
      if (wq == 0) {
        if constexpr (CT < 8) {
#pragma unroll
          for (int c = 0; c < CT; ++c)
            if (lane == c) ms[c] = m_run[c];
        } else {
          if (lane < CT) ms[lane] = m_run[0];
        }
      }
      mbar_arrive(bar(Sh::B_X + wg));
      if (!(ok = wait_all(bar(Sh::B_X + wg), xs & 1))) break;
      ++xs;
      if (lane == 0) mbar_arrive(bar(Sh::B_QE + (u & 1)));  // the unit's query tables have been read
      const bool sink = p.sinks != nullptr && i0 == 0;
      int qi = (col0 + c0) / a.group, hg = col0 + c0 - qi * a.group;  // query row, head of the group
#pragma unroll
      for (int c = 0; c < CT; ++c) {
        if (c0 + c >= cols) break;
        const int h = kh * a.group + hg;
        const int64_t t = (int64_t)q_begin + qi;
        if (++hg == a.group) { hg = 0; ++qi; }
        float total = (ws[c] + ws[CT + c]) + (ws[2 * CT + c] + ws[3 * CT + c]);
        float m = ms[c], f = 1.f;
        if (sink) {
          const float s = load_float(p.sinks, p.sink_t, h * p.si0) * kLog2e;
          const float mx = fmaxf(m, s);
          if (mx != -INFINITY) {
            f = m == -INFINITY ? 0.f : fast_exp2(m - mx);
            total = total * f + fast_exp2(s - mx);
            m = mx;
          }
        }
        const bool none = total == 0.f;
        const float inv = none ? 0.f : f * kUnbias / total;
        const float lse = none ? -INFINITY : (m + log2f(total)) * kLn2;
        const int64_t prow_ = (((int64_t)part_slot * p.c.HK + kh) * a.cblocks + cb) * C + c0 + c;
#pragma unroll
        for (int hf = 0; hf < DH; ++hf) {
          const int d = hf * 128 + key_i;
          if (d >= p.c.D) break;
          float o0, o1;
          f2unpack(o[hf][c / 2], o0, o1);
          const float y = (c & 1 ? o1 : o0) * inv;
          if (part_slot >= 0) p.part[prow_ * p.c.D + d] = y;
          else store_float(p.out, p.qt, t * p.os0 + (int64_t)h * p.os1 + d * p.os2, y);
        }
        if (key_i == 0) {
          if (part_slot >= 0) p.part_lse[prow_] = lse;
          else p.lse[(int64_t)h * p.ls0 + t * p.ls1] = lse;
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 4 * WG + 1) {
    tc_fence_after();
    tmem_dealloc(tmem, Sh::kCols);
  }
}

// Joins the pieces of requests that several groups share: one warp per column.
__global__ void __launch_bounds__(128) block_merge_kernel(const DecodeArgs a, const int C) {
  const BlockAttn& p = a.p;
  const int lane = threadIdx.x & 31, b = blockIdx.z, kh = blockIdx.y;
  const int col = blockIdx.x * 4 + (threadIdx.x >> 5);
  const int q_begin = p.cu_q[b * p.cq0], n = p.cu_q[(b + 1) * p.cq0] - q_begin;
  const int cb = col / C, qi = col / a.group, h = kh * a.group + col - qi * a.group;
  asm volatile("griddepcontrol.wait;\n" ::: "memory");
  if (col >= n * a.group) return;
  const int4 in = a.info[b * a.cblocks + cb];
  if (in.y <= in.x) return;  // one group holds the request: written already
  // A decode that gave up on a wait may have left no such numbers.
  if (in.x < 0 || in.y >= a.groups) return;
  const int D = p.c.D, pieces = in.y - in.x + 1;
  auto row_of = [&](int k) {
    const int64_t slot = 2 * (int64_t)(in.x + k) + (k == 0 && !in.z ? 1 : 0);
    return ((slot * p.c.HK + kh) * a.cblocks + cb) * C + (col - cb * C);
  };
  // The first rows come beside their LSEs (most requests have two or three pieces).
  constexpr int kAhead = 3;
  float ahead[kAhead][8];
#pragma unroll
  for (int k = 0; k < kAhead; ++k)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      ahead[k][i] = k < pieces && i * 32 + lane < D ? p.part[row_of(k) * D + i * 32 + lane] : 0.f;
  float m = -INFINITY;
  bool nan = false;
  for (int k = lane; k < pieces; k += 32) {
    const float x = p.part_lse[row_of(k)];
    m = fmaxf(m, x);
    nan |= x != x;
  }
  m = warp_max(m);
  nan = __any_sync(0xffffffffu, nan);
  float sum = 0.f;
  for (int k = lane; k < pieces; k += 32) {
    const float x = p.part_lse[row_of(k)];
    if (x != -INFINITY) sum += fast_exp2((x - m) * kLog2e);
  }
  sum = warp_sum(sum);
  const int64_t t = (int64_t)q_begin + qi;
  const bool none = m == -INFINITY && !nan;
  const float inv = none ? 0.f : 1.f / sum;
  float acc[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
  for (int k = 0; k < kAhead; ++k) {
    const float x = k < pieces ? p.part_lse[row_of(k)] : -INFINITY;
    if (x == -INFINITY) continue;
    const float w = fast_exp2((x - m) * kLog2e) * inv;
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = fmaf(w, ahead[k][i], acc[i]);
  }
  for (int k = kAhead; k < pieces; ++k) {
    const int64_t r = row_of(k);
    const float x = p.part_lse[r];
    if (x == -INFINITY) continue;
    const float w = fast_exp2((x - m) * kLog2e) * inv;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i * 32 + lane < D) acc[i] = fmaf(w, p.part[r * D + i * 32 + lane], acc[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (i * 32 + lane < D) store_float(p.out, p.qt, t * p.os0 + (int64_t)h * p.os1 + (i * 32 + lane) * p.os2, acc[i]);
  if (lane == 0) p.lse[(int64_t)h * p.ls0 + t * p.ls1] = none ? -INFINITY : m + log2f(sum) * kLn2;
}

int columns(const BlockAttn& p) { return p.max_q * (p.HQ / p.c.HK); }

// Columns per CTA of the kernel variant that takes these columns.
int column_block(const BlockAttn& p) {
  const int cols = columns(p), most = p.qt == FA_F16 && p.c.D > 128 ? 16 : 32;
  return std::min(cols <= 4 ? 4 : cols <= 8 ? 8 : cols <= 16 ? 16 : cols <= 24 ? 24 : 32, most);
}
int column_blocks(const BlockAttn& p) { return (columns(p) + column_block(p) - 1) / column_block(p); }

// Most tiles that a request's columns see.
int64_t visible_tiles(const BlockAttn& p) {
  const int64_t all = std::max<int64_t>(1, ((int64_t)p.max_k + kKeys - 1) / kKeys);
  if (p.win < 0) return all;
  const int64_t some = ((int64_t)p.win + p.max_q + 2 * kKeys - 2) / kKeys + (p.first + kKeys - 1) / kKeys;
  return std::max<int64_t>(1, std::min(all, some));
}

int make_map(CUtensorMap* map, const uint8_t* ptr, const BlockCache& c, int64_t s0, int64_t s1, int64_t s2, int box_tok) {
  const uint64_t dims[4] = {(uint64_t)c.D, (uint64_t)c.HK, (uint64_t)c.page, (uint64_t)c.pages};
  const uint64_t strides[3] = {(uint64_t)s2, (uint64_t)s1, (uint64_t)s0};
  const uint32_t box[4] = {128u, 1u, (uint32_t)box_tok, 1u};
  return encode_tensor_map(map, FA_E4M3, 4, ptr, dims, strides, box, true);
}

// Calls f with the kernel shape (parts, columns, halves) of a call.
template <int NP, int DH, typename F>
auto with_columns(int block, F f) {
  if (block == 4) return f(Shape<NP, 4, DH>{}, block_decode_kernel<NP, 4, DH>);
  if (block == 8) return f(Shape<NP, 8, DH>{}, block_decode_kernel<NP, 8, DH>);
  if constexpr (!(NP == 3 && DH == 2))
    if (block == 24) return f(Shape<NP, 24, DH>{}, block_decode_kernel<NP, 24, DH>);
  if constexpr (!(NP == 3 && DH == 2))
    if (block == 32) return f(Shape<NP, 32, DH>{}, block_decode_kernel<NP, 32, DH>);
  return f(Shape<NP, 16, DH>{}, block_decode_kernel<NP, 16, DH>);
}
template <typename F>
auto with_shape(const BlockAttn& p, F f) {
  const int block = column_block(p);
  if (p.qt == FA_BF16) return p.c.D > 128 ? with_columns<2, 2>(block, f) : with_columns<2, 1>(block, f);
  return p.c.D > 128 ? with_columns<3, 2>(block, f) : with_columns<3, 1>(block, f);
}

size_t up256(size_t x) { return (x + 255) / 256 * 256; }
size_t part_rows(const BlockAttn& p, int groups) {
  return (size_t)2 * groups * p.c.HK * column_blocks(p) * column_block(p);
}

}  // namespace

bool block_decode_supported(const BlockAttn& p) {
  if (!(p.qt == FA_F16 || p.qt == FA_BF16) || p.c.D > 256 || p.c.D % 16) return false;
  if (((uintptr_t)p.c.k & 15u) || ((uintptr_t)p.c.v & 15u)) return false;
  for (int64_t s : {p.c.ks0, p.c.ks1, p.c.ks2, p.c.vs0, p.c.vs1, p.c.vs2})
    if (s <= 0 || s % 16 || s >= ((int64_t)1 << 40)) return false;
  if (p.B * visible_tiles(p) >= (1LL << 31)) return false;
  return tensor_map_available();
}

// Groups that the tile list is cut into: one wave of resident CTAs over the KV
// heads and column blocks, 3 tiles each at least (one request, 16 tiles: 18.3 us
// in 16 pieces, 14.6 in 8; 4 requests: 23.4 in 55, 19.4 in 27).
//
// Negative: a group per request (-B). That saves the merge and the change from
// one request to the next (about 9 us) and loses what the shorter requests leave
// idle, at most half of a request's time if lengths spread evenly -- nothing
// where a window cuts most requests to one length; a CTA takes 0.65 us a tile
// alone on its SM, and 0.75 us for each CTA there at HBM's rate. 32 requests, 8
// KV heads, 4 / 8 / 16 tiles: 13.2 / 16.8 / 35 us against 22.5 / 25.6 / 41 split;
// 48 requests of 32 tiles: 73 against 79, of 8..32 tiles 62 against 56; 48
// windows of 34 tiles: 79 against 86. Few CTAs: up to 8 tiles (one request: 13.7
// against 13.9). More CTAs than fit at once start as others end, where an SM has
// two or three of them: requests of 4 tiles, 96 / 128 of them, 31 / 46 us against
// 36 / 47 split (1..4 tiles: 27 / 35 against 36 / 41), 96 of 6 tiles 42 against 44
// (1..6: 33 against 42), but 512 of 4 tiles 147 against 131, 128 of 8 68 against
// 60, and with one CTA per SM (rows of 256) 128 of 4 tiles 98 against 74.
int block_decode_splits(const BlockAttn& p) {
  if (p.splits > 0) return p.splits;
  const int64_t ctas = with_shape(p, [](auto shape, auto) { return decltype(shape)::kCtas; });
  const int64_t resident = ctas * sm_count(), per_request = (int64_t)p.c.HK * column_blocks(p);
  const int64_t most = visible_tiles(p), tiles = p.B * most, units = p.B * per_request;
  const double tile = std::max(0.65, 0.75 * units / sm_count());
  const bool even = p.win >= 0 && 2 * most * kKeys <= p.max_k;
  if (units <= resident && (even || most * tile <= 32) && (most <= 8 || units >= 128)) return -p.B;
  if (ctas > 1 && most <= 6 && most * units <= 16 * resident) return -p.B;
  return (int)std::max<int64_t>(1, std::min(resident / per_request, (tiles + 2) / 3));
}

int block_decode_columns(const BlockAttn& p) { return column_block(p); }

size_t block_decode_workspace(const BlockAttn& p, int groups) {
  if (groups <= 1) return 0;
  const size_t rows = part_rows(p, groups);
  return up256(rows * p.c.D * sizeof(float)) + up256(rows * sizeof(float)) +
         up256((size_t)p.B * column_blocks(p) * sizeof(int4));
}

int block_decode_timeout_flag(bool clear) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_block_decode_timeout, sizeof(int)) != cudaSuccess) return -1;
  if (clear && v) {
    const int zero = 0;
    if (cudaMemcpyToSymbol(g_block_decode_timeout, &zero, sizeof(int)) != cudaSuccess) return -1;
  }
  return v;
}

int launch_block_decode(const BlockAttn& p, int groups, void* workspace, cudaStream_t stream) {
  DecodeArgs a{};
  a.p = p;
  a.group = p.HQ / p.c.HK;
  a.cblocks = column_blocks(p);
  a.by_request = groups < 0;
  a.groups = groups = std::abs(groups);
  a.box_tok = std::min(p.c.page, kKeys);
  a.q_vec = p.qs2 == 1 && p.qs0 % 4 == 0 && p.qs1 % 4 == 0 && ((uintptr_t)p.q & 7u) == 0;
  if (groups > 1 && !a.by_request) {
    uint8_t* ws = reinterpret_cast<uint8_t*>(workspace);
    const size_t rows = part_rows(p, groups);
    a.p.part = reinterpret_cast<float*>(ws);
    ws += up256(rows * p.c.D * sizeof(float));
    a.p.part_lse = reinterpret_cast<float*>(ws);
    a.info = reinterpret_cast<int4*>(ws + up256(rows * sizeof(float)));
  }
  CUtensorMap mk, mv;
  std::memset(&mk, 0, sizeof(mk));
  std::memset(&mv, 0, sizeof(mv));
  int rc = make_map(&mk, p.c.k, p.c, p.c.ks0, p.c.ks1, p.c.ks2, a.box_tok);
  if (rc == FA_OK) rc = make_map(&mv, p.c.v, p.c, p.c.vs0, p.c.vs1, p.c.vs2, a.box_tok);
  if (rc != FA_OK) return rc;
  rc = with_shape(p, [&](auto shape, auto kernel) -> int {
    using Sh = decltype(shape);
    static std::atomic<uint64_t> ready{0};  // devices whose kernel has its shared-memory limit
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && (dev >= 64 || !(ready.load(std::memory_order_relaxed) >> dev & 1))) {
      e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
      if (e == cudaSuccess && dev < 64) ready.fetch_or(1ull << dev, std::memory_order_relaxed);
    }
    if (e != cudaSuccess) return fail(FA_ERR_CUDA, "block decode smem attribute: %s", cudaGetErrorString(e));
    kernel<<<dim3((unsigned)(p.c.HK * a.cblocks), (unsigned)groups), Sh::kThreads, Sh::kSmem, stream>>>(mk, mv, a);
    note_launch();
    FAB_LAUNCH_CHECK("block-scaled decode launch");
    return FA_OK;
  });
  if (rc != FA_OK || groups <= 1 || a.by_request) return rc;
  // The merge may start before the decode's end and waits for it on the device.
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((columns(p) + 3) / 4), (unsigned)p.c.HK, (unsigned)p.B);
  cfg.blockDim = dim3(128);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, block_merge_kernel, a, column_block(p));
  if (e != cudaSuccess) return fail(FA_ERR_CUDA, "block-scaled merge launch: %s", cudaGetErrorString(e));
  note_launch();
  return FA_OK;
}

}  // namespace fab
