// Products of a few rows with weights of 4 bits, and the weights' rounding.
#include "iris_kernels.h"
#include "lm_device.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

namespace {

// ------------------------------------------------------------------ products
//   y[r][n] = sum over groups g of  s[n][g] sum over k in g of (q[n][k] - z[n][g]) x[r][k]   (+ add[r][n])
// Should be bound by the weights' bytes; instructions are.  151936 x 2560 in groups of 32,
// one row: 65 us, 34 for the bytes, 27 instructions for a word of eight weights, 65 % of the issue slots, the pipe of shifts and logic
// 58 % active; 6144 x 2560 in groups of 128: 5.5 us, of which 1.3 for the bytes (one round, latency).  The products are mma m16n8k16 with 16 rows of the
// weights as m and 8 rows of x as n.  q - z is a whole number of at most 8 bits,
// exact in bf16, and so is x; the scale multiplies a group's f32 sum.
// A 32-bit word holds eight columns k .. k + 7 of a row; its halves' nibble j give
// the pair (k + j, k + j + 4) by one shift and one mask-and-or onto bf16 128 =
// 0x4300, whose last bits count in ones.  The order of the columns within the
// product is free as long as x has the same: lane (g, i4) takes word i4 of 32
// columns of row g and g + 8, and the same eight columns of x, paired alike.
// A warp takes 16 rows of the weights and goes along k by chunks of 128 columns,
// through a ring of cp.async stages.
constexpr int L4_WARPS = 8, L4_THREADS = 32 * L4_WARPS, L4_CHUNK = 128;
constexpr int L4_STAGE = 16 * L4_CHUNK / 2;  // bytes of a warp's chunk

__device__ __forceinline__ uint32_t minus2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// Numbers that the compiler does not see through, for the two below.
struct Constants4 {
  uint32_t mask, magic;
  __device__ Constants4() {
    asm volatile("mov.b32 %0, 0x000F000F;" : "=r"(mask));
    asm volatile("mov.b32 %0, 0x43004300;" : "=r"(magic));
  }
};
// Pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word's nibbles, less the zero (128 + z twice).  The busiest pipe is that of
// shifts and logic: mask and magic are in registers, so that one instruction does both (constants would take two: the head's
// 151936 x 2560 74 us, 66 so; the shifts as high halves of products, on another pipe, 79).
__device__ __forceinline__ void nibbles(uint32_t w, uint32_t zero, const Constants4& k, uint32_t p[4]) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    uint32_t x;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(x) : "r"(w >> 4 * j), "r"(k.mask), "r"(k.magic));  // and, or
    p[j] = minus2(x, zero);
  }
}

// A warp's 16 MT rows of the weights from n0 on; what does not change from chunk to chunk is worked out once.  GS: parts of 32
// columns of a chunk that share a group, 1, 2 or 4.  ZERO: zeros are given.
template <int MT, int GS, bool ZERO>
struct Weights {
  const IrisLinear4& a;
  Constants4 constants;
  const uint8_t* q[2 * MT];    // rows 8 j + g, at this lane's 16 bytes of a chunk
  const uint8_t* scale[2 * MT];
  const uint8_t* zero[2 * MT];
  int bytes[2 * MT];           // 16, or 0 where there is no row

  __device__ Weights(const IrisLinear4& a, int n0) : a(a) {
    const int g = threadIdx.x % 32 / 4, i4 = threadIdx.x % 4;
#pragma unroll
    for (int j = 0; j < 2 * MT; j++) {
      const int row = n0 + j * 8 + g;
      bytes[j] = row < a.n ? 16 : 0;
      const int64_t r = row < a.n ? row : 0;
      q[j] = a.q + r * a.ldq + i4 * 16;
      scale[j] = (const uint8_t*)a.scale + r * a.lds * (a.scale_f32 ? 4 : 2);
      if (ZERO) zero[j] = a.zero + r * a.ldz;
    }
  }
  // chunk c into shared memory at `to`: part s of 32 columns of row r is at place s ^ (r >> 1 & 3)
  __device__ void load(uint32_t to, int c) const {
    const int g = threadIdx.x % 32 / 4, i4 = threadIdx.x % 4;
    const bool in = c * (L4_CHUNK / 2) + i4 * 16 < a.k / 2;
#pragma unroll
    for (int j = 0; j < 2 * MT; j++)
      cp_async16(to + (j * 8 + g) * 64 + ((i4 ^ (g >> 1 & 3)) << 4), q[j] + (in ? c * (L4_CHUNK / 2) : 0), in ? bytes[j] : 0);
  }
  // Scales and zeros of a chunk as they are in memory (work on them here would wait for them); lane i4 has those of the group
  // of part i4.
  struct Group {
    uint32_t scale[2 * MT], zero[2 * MT];
  };
  __device__ void load(Group& v, int c) const {
    const int i4 = threadIdx.x % 4, group = GS == 4 ? iris_paged_block(a.div, c) : c * (4 / GS) + i4 / GS;
    const bool in = c * L4_CHUNK + i4 * 32 < a.k;
#pragma unroll
    for (int j = 0; j < 2 * MT; j++) {
      v.scale[j] = 0;
      if (!in || !bytes[j]) continue;
      v.scale[j] = a.scale_f32 ? __ldg((const uint32_t*)scale[j] + group) : __ldg((const uint16_t*)scale[j] + group);
      if (ZERO) v.zero[j] = __ldg(zero[j] + group);
    }
  }
  // One chunk: acc of each 8 rows of x; x(s, t) gives part s's eight columns of row g of x's rows 8 t ..
  template <int NT, typename X>
  __device__ void products(uint32_t base, const Group& v, X x, float acc[MT][NT][4]) const {
    const int g = threadIdx.x % 32 / 4, i4 = threadIdx.x % 4;
    float sc[2 * MT];
    uint32_t z[2 * MT];
#pragma unroll
    for (int j = 0; j < 2 * MT; j++) {
      sc[j] = __uint_as_float(a.scale_f32 ? v.scale[j] : v.scale[j] << 16);
      z[j] = ZERO ? 0x43004300u + (v.zero[j] & 127) * 0x10001u : 0x43084308u;
    }
    float sum[MT][NT][4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
      uint32_t p[2 * MT][4];
      const uint32_t word = base + g * 64 + ((s ^ (g >> 1 & 3)) << 4) + i4 * 4;
#pragma unroll
      for (int j = 0; j < 2 * MT; j++) {
        uint32_t w;
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(word + j * 512));
        nibbles(w, GS == 4 || !ZERO ? z[j] : __shfl_sync(0xffffffffu, z[j], g * 4 + s), constants, p[j]);
      }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const uint4 u = x(s, t);
        const uint32_t x0 = __byte_perm(u.x, u.z, 0x5410), x1 = __byte_perm(u.x, u.z, 0x7632);
        const uint32_t x2 = __byte_perm(u.y, u.w, 0x5410), x3 = __byte_perm(u.y, u.w, 0x7632);
#pragma unroll
        for (int m = 0; m < MT; m++) {
          if (s % GS == 0) mma_bf16_first(sum[m][t], p[2 * m][0], p[2 * m + 1][0], p[2 * m][1], p[2 * m + 1][1], x0, x1);
          else mma_bf16(sum[m][t], p[2 * m][0], p[2 * m + 1][0], p[2 * m][1], p[2 * m + 1][1], x0, x1);
          mma_bf16(sum[m][t], p[2 * m][2], p[2 * m + 1][2], p[2 * m][3], p[2 * m + 1][3], x2, x3);
        }
      }
      if (s % GS == GS - 1) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
          const float s0 = GS == 4 ? sc[2 * m] : __shfl_sync(0xffffffffu, sc[2 * m], g * 4 + s);
          const float s1 = GS == 4 ? sc[2 * m + 1] : __shfl_sync(0xffffffffu, sc[2 * m + 1], g * 4 + s);
#pragma unroll
          for (int t = 0; t < NT; t++) {
            acc[m][t][0] += s0 * sum[m][t][0], acc[m][t][1] += s0 * sum[m][t][1];
            acc[m][t][2] += s1 * sum[m][t][2], acc[m][t][3] += s1 * sum[m][t][3];
          }
        }
      }
    }
  }
};

__device__ __forceinline__ void store4(const IrisLinear4& a, int r, int n, float y) {
  if (r >= a.rows || n >= a.n) return;
  if (a.f32) {
    if (a.add) y += ((const float*)a.add)[r * a.ldadd + n];
    ((float*)a.out)[r * a.ldo + n] = y;
  } else {
    if (a.add) y += __bfloat162float(((const __nv_bfloat16*)a.add)[r * a.ldadd + n]);
    ((__nv_bfloat16*)a.out)[r * a.ldo + n] = __float2bfloat16_rn(y);
  }
}

// Up to 8 rows of x.  WK warps share 16 MT rows of the weights and take chunks in turn (and a.parts blocks, a cluster): all of
// them where the weights have few rows, so that their bytes are asked for at once; where they have many, two, and two
// sixteens of rows to a warp, which share what is done for x.  x comes through registers, a chunk ahead.
constexpr int L4_RING = 4;
template <int MT, int WK, int GS, bool ZERO>
__global__ void __launch_bounds__(L4_THREADS, MT == 1 ? 3 : 2) linear4_kernel(const __grid_constant__ IrisLinear4 a) {
  constexpr int STRIPS = L4_WARPS / WK, LD = MT * 16 + 4;  // LD: of a row of x in the sums: no bank conflicts
  constexpr int STAGE = MT * L4_STAGE, PER = 8 * LD, OUT = STRIPS * MT * 128;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid / 32, g = tid % 32 / 4, i4 = tid % 4;
  const int part = blockIdx.x % a.parts, b0 = blockIdx.x / a.parts * (STRIPS * MT * 16), strip = warp / WK;
  const int chunks = (a.k + L4_CHUNK - 1) / L4_CHUNK, step = a.parts * WK, c0 = part * WK + warp % WK;
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const Weights<MT, GS, ZERO> weights(a, b0 + strip * (MT * 16));
  const uint32_t base = iris::smem_u32(smem) + warp * (L4_RING * STAGE);
  int ld = c0;
  auto issue = [&](int stage) {
    if (ld < chunks) weights.load(base + stage * STAGE, ld);
    ld += step;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < L4_RING - 1; s++) issue(s);
  const __nv_bfloat16* xr = (const __nv_bfloat16*)a.x + (int64_t)(g < a.rows ? g : 0) * a.ldx + i4 * 8;
  const bool live = g < a.rows;
  auto load_x = [&](uint4 v[4], int c) {  // (the lanes of a row that is not there keep their zeros)
    const __nv_bfloat16* from = xr + (int64_t)c * L4_CHUNK;
    if ((c + 1) * L4_CHUNK <= a.k) {
      if (live) {
#pragma unroll
        for (int s = 0; s < 4; s++) v[s] = __ldg(reinterpret_cast<const uint4*>(from + s * 32));
      }
    } else {
#pragma unroll
      for (int s = 0; s < 4; s++)
        v[s] = live && c * L4_CHUNK + s * 32 < a.k ? __ldg(reinterpret_cast<const uint4*>(from + s * 32)) : make_uint4(0u, 0u, 0u, 0u);
    }
  };
  uint4 x[2][4] = {};
  typename Weights<MT, GS, ZERO>::Group v[2];
  if (c0 < chunks) {
    load_x(x[0], c0);
    weights.load(v[0], c0);
  }
  float acc[MT][1][4] = {};
  int stage = 0;
  auto chunk = [&](int c, uint4 now[4], typename Weights<MT, GS, ZERO>::Group& v_now, uint4 next[4],
                   typename Weights<MT, GS, ZERO>::Group& v_next) {
    issue(stage == 0 ? L4_RING - 1 : stage - 1);
    if (c + step < chunks) {
      load_x(next, c + step);
      weights.load(v_next, c + step);
    }
    asm volatile("cp.async.wait_group %0;" ::"n"(L4_RING - 1) : "memory");
    __syncwarp();
    weights.template products<1>(base + stage * STAGE, v_now, [&](int s, int) { return now[s]; }, acc);
    __syncwarp();  // this stage is filled again by the next chunk's issue
    stage = stage == L4_RING - 1 ? 0 : stage + 1;
  };
  for (int c = c0; c < chunks; c += 2 * step) {
    chunk(c, x[0], v[0], x[1], v[1]);
    if (c + step < chunks) chunk(c + step, x[1], v[1], x[0], v[0]);
  }
  // the warps' sums, then the parts' of a cluster, always in the same order
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int m = 0; m < MT; m++) {
    float* to = red + warp * PER + 2 * i4 * LD + m * 16 + g;
    const float* y = acc[m][0];
    to[0] = y[0], to[LD] = y[1], to[8] = y[2], to[LD + 8] = y[3];
  }
  __syncthreads();
  constexpr int R = MT * 16;  // rows of the weights of a strip
  auto place = [&](int e) { return red + e / (8 * R) * WK * PER + e % (8 * R) / R * LD + e % R; };
  auto out = [&](int e, float y) { store4(a, e % (8 * R) / R, b0 + e / (8 * R) * R + e % R, y); };
  for (int e = tid; e < OUT; e += L4_THREADS) {
    if (e % (8 * R) / R >= a.rows) continue;
    float* at = place(e);
    float y = at[0];
#pragma unroll
    for (int w = 1; w < WK; w++) y += at[w * PER];
    if (a.parts == 1) out(e, y);
    else at[0] = y;  // this thread alone reads and writes these places
  }
  if (a.parts == 1) return;
  __syncwarp();
  iris::cluster_sync();
  for (int e = part * L4_THREADS + tid; e < OUT; e += a.parts * L4_THREADS) {
    if (e % (8 * R) / R >= a.rows) continue;
    float* at = place(e);
    float y = 0.f;
    for (int p = 0; p < a.parts; p++) y += *iris::cluster_map(at, p);
    out(e, y);
  }
  __syncwarp();
  iris::cluster_sync();  // the others have read this block's sums
}

// More rows: WK warps share 16 rows of the weights, and the block loads the columns of x of a stage's WK chunks together (8 NT
// rows of x; with a chunk to each warp x would cross L2 that much more often).  k in parts, a block of a cluster each.
template <int NT, int WK>
struct L4Rows {
  static constexpr int kStages = NT * WK > 4 ? 3 : 4;
  static constexpr int kX = NT * 8 * L4_CHUNK * 2;             // bytes of x of a chunk
  static constexpr int kStage = L4_WARPS * L4_STAGE + WK * kX;
  static constexpr int kRows = L4_WARPS / WK * 16;             // of the weights, a block's
  static constexpr int kLd = kRows + 4;                        // of a row of x in the sums: no bank conflicts
  static constexpr int kRed = WK * NT * 8 * kLd * 4;
  static constexpr int kSmem = kStages * kStage > kRed ? kStages * kStage : kRed;
};
template <int NT, int WK, int GS, bool ZERO>
__global__ void __launch_bounds__(L4_THREADS, 2) linear4_rows_kernel(const __grid_constant__ IrisLinear4 a) {
  using Sh = L4Rows<NT, WK>;
  constexpr int D = Sh::kStages, ROWS = Sh::kRows;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid / 32, g = tid % 32 / 4, i4 = tid % 4, sub = warp % WK;
  const int part = blockIdx.x % a.parts, b0 = blockIdx.x / a.parts * ROWS, r0 = blockIdx.y * (NT * 8);
  const int steps = ((a.k + L4_CHUNK - 1) / L4_CHUNK + WK - 1) / WK;  // of WK chunks
  const int first = (int)((int64_t)steps * part / a.parts), end = (int)((int64_t)steps * (part + 1) / a.parts);
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const Weights<1, GS, ZERO> weights(a, b0 + warp / WK * 16);
  const uint32_t ring = iris::smem_u32(smem);
  auto issue = [&](int c, int stage) {
    if (c < end) {
      const uint32_t to = ring + stage * Sh::kStage;
      weights.load(to + warp * L4_STAGE, c * WK + sub);
#pragma unroll
      for (int i = tid; i < WK * NT * 8 * 16; i += L4_THREADS) {  // 16 bytes each: row i / 16, place (i % 16) ^ (row & 1) << 2
        const int row = i / 16 % (NT * 8), ch = i % 16, k = (c * WK + i / (NT * 128)) * L4_CHUNK + ch * 8;
        const bool has = r0 + row < a.rows && k < a.k;
        cp_async16(to + L4_WARPS * L4_STAGE + i / 16 * 256 + ((ch ^ (row & 1) << 2) << 4),
                   (const __nv_bfloat16*)a.x + (has ? (int64_t)(r0 + row) * a.ldx + k : 0), has ? 16 : 0);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < D - 1; s++) issue(first + s, s);
  typename Weights<1, GS, ZERO>::Group v, v_next;
  weights.load(v_next, first * WK + sub);
  float acc[1][NT][4] = {};
  int stage = 0;
  for (int c = first; c < end; c++) {
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
    __syncthreads();  // this stage has come, and the one before it is done with
    issue(c + D - 1, stage == 0 ? D - 1 : stage - 1);
    v = v_next;
    if (c + 1 < end) weights.load(v_next, (c + 1) * WK + sub);
    const uint32_t base = ring + stage * Sh::kStage, xs = base + L4_WARPS * L4_STAGE + sub * Sh::kX;
    weights.template products<NT>(base + warp * L4_STAGE, v, [&](int s, int t) {
      uint4 u;
      asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w)
                   : "r"(xs + (t * 8 + g) * 256 + (((s * 4 + i4) ^ (g & 1) << 2) << 4)));
      return u;
    }, acc);
    stage = stage == D - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  constexpr int LD = Sh::kLd, PER = NT * 8 * LD, OUT = NT * 8 * ROWS;
#pragma unroll
  for (int t = 0; t < NT; t++) {
    float* to = red + sub * PER + (t * 8 + 2 * i4) * LD + warp / WK * 16 + g;
    const float* y = acc[0][t];
    to[0] = y[0], to[LD] = y[1], to[8] = y[2], to[LD + 8] = y[3];
  }
  if (a.parts > 1) {
    __syncwarp();
    iris::cluster_sync();
  } else {
    __syncthreads();
  }
  for (int e = part * L4_THREADS + tid; e < OUT; e += a.parts * L4_THREADS) {
    float* at = red + e / ROWS * LD + e % ROWS;
    float y = 0.f;
    for (int p = 0; p < a.parts; p++) {
      const float* from = a.parts > 1 ? iris::cluster_map(at, p) : at;
#pragma unroll
      for (int w = 0; w < WK; w++) y += from[w * PER];
    }
    store4(a, r0 + e / ROWS, b0 + e % ROWS, y);
  }
  if (a.parts > 1) {
    __syncwarp();
    iris::cluster_sync();  // the others have read this block's sums
  }
}

// ------------------------------------------------------------------ rounding to 4 bits
// Lanes of 8 values each take a group (up to 256 columns in registers between the
// two passes): its largest magnitude / 7, rounded to the scale's type, is the scale s;
// q = round(w / s) + 8, ties to even.  A group that holds an infinity or NaN gets the
// scale NaN.  Bound by the divisions, which decide the ties: bf16 151936 x 2560 516 us,
// 156 for the bytes (572 with values read twice and converted; through 1 / s with the
// division only next to ties 686, since some lane of a warp mostly has to).  It runs
// once for a model's weights.
template <typename In>
__device__ __forceinline__ void eight(const In* p, float x[8]) {
  if constexpr (sizeof(In) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
  } else {
    vec_values<__nv_bfloat16>(*reinterpret_cast<const uint4*>(p), x);
  }
}

template <typename In>
__global__ void __launch_bounds__(256) quantize4_kernel(const __grid_constant__ IrisQuantize4 a) {
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const int lanes = a.group >= 256 ? 32 : a.group / 8;  // 4, 8, 16 or 32 of a group
  const int in = threadIdx.x % lanes, groups = a.k / a.group;
  const int64_t first = ((int64_t)blockIdx.x * 256 + threadIdx.x) / lanes, step = (int64_t)gridDim.x * 256 / lanes;
  const int64_t all = (int64_t)a.n * groups;
  for (int64_t i0 = first - threadIdx.x % 32 / lanes; i0 < all; i0 += step) {  // i0: the warp's first group
    const int64_t i = i0 + threadIdx.x % 32 / lanes;
    const bool has = i < all;
    const int64_t row = !has ? 0 : all >> 31 ? i / groups : (uint32_t)i / (uint32_t)groups, group = has ? i - row * groups : 0;
    const In* w = (const In*)a.w + row * a.ldw + group * a.group;
    uint32_t top = 0;  // of the magnitudes' bits: an infinity or NaN is above all others
    float x[8] = {};
    for (int c = in * 8; has && c < a.group; c += lanes * 8) {
      eight(w + c, x);
#pragma unroll
      for (int j = 0; j < 8; j++) top = max(top, __float_as_uint(x[j]) & 0x7FFFFFFFu);
    }
    for (int o = lanes / 2; o; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (!has) continue;
    float s = top >= 0x7F800000u ? __uint_as_float(0x7FC00000u) : __uint_as_float(top) / 7.0f;
    if (!a.scale_f32) s = __bfloat162float(__float2bfloat16_rn(s));
    if (in == 0) {
      if (a.scale_f32) ((float*)a.scale)[row * a.lds + group] = s;
      else ((__nv_bfloat16*)a.scale)[row * a.lds + group] = __float2bfloat16_rn(s);
    }
    for (int c = in * 8; c < a.group; c += lanes * 8) {
      if (a.group > 256) eight(w + c, x);
      uint32_t q = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        // the last bits of 1.5 * 2^23 + 8 + v are those of 8 + v, rounded ties to even
        const float v = s > 0.f ? fminf(fmaxf(x[j] / s, -8.f), 7.f) : 0.f;
        q |= (__float_as_uint(v + (0x1.8p23f + 8.f)) & 15u) << 4 * j;
      }
      *reinterpret_cast<uint32_t*>(a.q + row * a.ldq + (group * a.group + c) / 2) = q;
    }
  }
}

template <typename Kernel>
cudaError_t go(Kernel kernel, dim3 grid, size_t smem, cudaStream_t stream, const IrisLinear4& a) {
  grid.x *= a.parts;
  if (a.parts == 1) return iris::launch_overlapped(kernel, grid, dim3(L4_THREADS), smem, stream, a);
  return iris::launch_cluster_overlapped(kernel, grid, dim3(L4_THREADS), smem, a.parts, stream, a);
}

// Parts of k for blocks of 128 / wk rows of the weights and 8 nt of x: as many as let all blocks be on the device at once, two an
// SM, of which clusters reach seven eighths (16 rows of 9728 -> 2560 28 -> 11 us, of 4096 -> 2560 13 -> 6.8)
int rows_parts(const IrisLinear4* a, int nt, int wk, int num_sms, int64_t* blocks) {
  const int64_t base = (int64_t)((a->n + 128 / wk - 1) / (128 / wk)) * ((a->rows + nt * 8 - 1) / (nt * 8));
  const int steps = ((a->k + L4_CHUNK - 1) / L4_CHUNK + wk - 1) / wk;
  int64_t parts = num_sms * 2 * 7 / 8 / base;
  if (parts > 8) parts = 8;
  if (parts > steps / 2) parts = steps / 2;
  if (parts < 1) parts = 1;
  *blocks = base * parts;
  return (int)parts;
}

template <int NT, int WK, int GS, bool ZERO>
cudaError_t go_rows(IrisLinear4* a, int parts, cudaStream_t stream) {
  using Sh = L4Rows<NT, WK>;
  a->parts = parts;
  const dim3 grid((unsigned)((a->n + Sh::kRows - 1) / Sh::kRows), (a->rows + NT * 8 - 1) / (NT * 8));
  return go(linear4_rows_kernel<NT, WK, GS, ZERO>, grid, Sh::kSmem, stream, *a);
}

// Warps that share 16 rows of the weights: one where the weights have many rows (16 rows of x, n 75776 of k 2560 46 us, 51 with
// two; 151936 97 and 103) or where that lets more blocks be on the device at once (n 6144 8.0 and 8.8, 9728 11.4 and 13.2); else
// two (n 38912 33 us, 36 with one; 25600 21 and 23; 2560 of k 9728 11 and 13).
template <int NT, int GS, bool ZERO>
cudaError_t rows_variant(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  int64_t one, two;
  const int parts1 = rows_parts(a, NT, 1, num_sms, &one), parts2 = rows_parts(a, NT, 2, num_sms, &two);
  if (a->n >= 4 * 128 * num_sms || one > two) return go_rows<NT, 1, GS, ZERO>(a, parts1, stream);
  return go_rows<NT, 2, GS, ZERO>(a, parts2, stream);
}

// parts: while that adds blocks for which there is room (one row of 9728 -> 2560 11.0 -> 9.6 us)
template <int MT, int WK, int GS, bool ZERO>
cudaError_t go_few(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  constexpr int rows = L4_WARPS / WK * MT * 16;
  const int strips = (a->n + rows - 1) / rows, chunks = (a->k + L4_CHUNK - 1) / L4_CHUNK;
  a->parts = 1;
  while (a->parts < 8 && (int64_t)strips * a->parts * 2 <= 3 * num_sms && a->parts * WK < chunks) a->parts *= 2;
  return go(linear4_kernel<MT, WK, GS, ZERO>, dim3((unsigned)strips), L4_WARPS * L4_RING * MT * L4_STAGE, stream, *a);
}

// Up to 8 rows: all of a block's warps on 16 rows of the weights (one row of x, n 9728 of k 2560 8.1 us, 11.8 with two; 38912 22.5
// and 24.8), or, of many rows, two on 32 (75776 32 us, 41 with all; 151936 63 and 79).
template <int GS, bool ZERO>
cudaError_t variant(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  if (a->rows > 16) return rows_variant<4, GS, ZERO>(a, num_sms, stream);
  if (a->rows > 8) return rows_variant<2, GS, ZERO>(a, num_sms, stream);
  return a->n >= 4 * 128 * num_sms ? go_few<2, 2, GS, ZERO>(a, num_sms, stream) : go_few<1, 8, GS, ZERO>(a, num_sms, stream);
}

template <int GS, bool ZERO>
cudaError_t shared_limits() {
  const struct { const void* f; int bytes; } k[] = {
      {(const void*)linear4_kernel<1, 8, GS, ZERO>, L4_WARPS * L4_RING * L4_STAGE},
      {(const void*)linear4_kernel<2, 2, GS, ZERO>, L4_WARPS * L4_RING * 2 * L4_STAGE},
      {(const void*)linear4_rows_kernel<2, 1, GS, ZERO>, L4Rows<2, 1>::kSmem},
      {(const void*)linear4_rows_kernel<2, 2, GS, ZERO>, L4Rows<2, 2>::kSmem},
      {(const void*)linear4_rows_kernel<4, 1, GS, ZERO>, L4Rows<4, 1>::kSmem},
      {(const void*)linear4_rows_kernel<4, 2, GS, ZERO>, L4Rows<4, 2>::kSmem}};
  for (const auto& x : k) {
    const cudaError_t e = cudaFuncSetAttribute(x.f, cudaFuncAttributeMaxDynamicSharedMemorySize, x.bytes);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

extern "C" cudaError_t iris_linear4_init(void) {
  const cudaError_t e[] = {shared_limits<1, false>(), shared_limits<1, true>(),  shared_limits<2, false>(),
                           shared_limits<2, true>(),  shared_limits<4, false>(), shared_limits<4, true>()};
  for (cudaError_t x : e)
    if (x != cudaSuccess) return x;
  return cudaSuccess;
}

extern "C" cudaError_t iris_launch_linear4(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  a->div = iris_paged_div(a->group >= L4_CHUNK ? a->group / L4_CHUNK : 1);
  if (a->group == 32) return a->zero ? variant<1, true>(a, num_sms, stream) : variant<1, false>(a, num_sms, stream);
  if (a->group == 64) return a->zero ? variant<2, true>(a, num_sms, stream) : variant<2, false>(a, num_sms, stream);
  return a->zero ? variant<4, true>(a, num_sms, stream) : variant<4, false>(a, num_sms, stream);
}

extern "C" cudaError_t iris_launch_quantize4(const IrisQuantize4* a, int f32, int num_sms, cudaStream_t stream) {
  const int lanes = a->group >= 256 ? 32 : a->group / 8;
  const int64_t blocks = ((int64_t)a->n * (a->k / a->group) * lanes + 255) / 256;
  const int64_t most = (int64_t)num_sms * 64;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (f32) return iris::launch_overlapped(quantize4_kernel<float>, grid, dim3(256), 0, stream, *a);
  return iris::launch_overlapped(quantize4_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, *a);
}
