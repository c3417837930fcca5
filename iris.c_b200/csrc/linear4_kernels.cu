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
// Bound by the weights' bytes.  A block takes 16 (or 32) rows of the weights and
// all of k, or a part of it (a cluster then adds up the parts); its warps take
// chunks of 128 columns in turn, each through a ring of cp.async stages of its
// own.  The products are mma m16n8k16 with the weights' rows as m and the rows of
// x as n.  q - z is a whole number of at most 8 bits, exact in bf16, and so is x;
// the scale multiplies a group's f32 sum.
// A 32-bit word holds eight columns k .. k + 7 of a row; its halves' nibble j give
// the pair (k + j, k + j + 4) by one shift and one mask-and-or onto bf16 128 =
// 0x4300, whose last bits count in ones.  The order of the columns within the
// product is free as long as x has the same: lane (g, i4) takes word i4 of 32
// columns of row g and g + 8, and the same eight columns of x, paired alike.
constexpr int L4_WARPS = 8, L4_THREADS = 32 * L4_WARPS, L4_CHUNK = 128;

// MT: 16 rows of weights each, NT: 8 rows of x each
template <int MT, int NT>
struct L4Shape {
  static constexpr int kStages = MT == 1 ? 4 : 3;
  static constexpr int kStage = MT * 16 * L4_CHUNK / 2;  // bytes
  static constexpr int kRing = kStages * kStage;         // of a warp
  static constexpr int kLd = MT * 16 + 4;                // of a row of x in the sums: no bank conflicts
  static constexpr int kRed = L4_WARPS * NT * 8 * kLd * 4;
  static constexpr int kSmem = L4_WARPS * kRing > kRed ? L4_WARPS * kRing : kRed;
};

__device__ __forceinline__ uint32_t minus2(uint32_t a, uint32_t b) {
  const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
  return *reinterpret_cast<const uint32_t*>(&d);
}

// pairs (0, 4), (1, 5), (2, 6), (3, 7) of a word's nibbles, less the zero (128 + z twice)
__device__ __forceinline__ void nibbles(uint32_t w, uint32_t zero, uint32_t p[4]) {
#pragma unroll
  for (int j = 0; j < 4; j++) p[j] = minus2((w >> 4 * j & 0x000F000Fu) | 0x43004300u, zero);
}

// GS: parts of 32 columns of a chunk that share a group, 1, 2 or 4
template <int MT, int NT, int GS>
__global__ void __launch_bounds__(L4_THREADS, MT * NT <= 2 ? 4 : 2) linear4_kernel(const __grid_constant__ IrisLinear4 a) {
  using Sh = L4Shape<MT, NT>;
  constexpr int D = Sh::kStages;
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, i4 = lane % 4;
  const int part = blockIdx.x % a.parts, n0 = blockIdx.x / a.parts * (MT * 16), r0 = blockIdx.y * (NT * 8);
  const int chunks = (a.k + L4_CHUNK - 1) / L4_CHUNK, step = a.parts * L4_WARPS;
  iris::grid_dep_wait();
  iris::grid_dep_launch();

  const uint32_t ring = iris::smem_u32(smem) + warp * Sh::kRing;
  int ld = part * L4_WARPS + warp;  // the next chunk to load
  auto issue = [&](int stage) {
    if (ld < chunks) {
#pragma unroll
      for (int j = 0; j < 2 * MT; j++) {
        const int row = j * 8 + g, at = ld * (L4_CHUNK / 2) + i4 * 16;
        const bool has = n0 + row < a.n && at < a.k / 2;
        cp_async16(ring + stage * Sh::kStage + row * 64 + ((i4 ^ (row >> 1 & 3)) << 4),
                   a.q + (has ? (int64_t)(n0 + row) * a.ldq + at : 0), has ? 16 : 0);
      }
      ld += step;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < D - 1; s++) issue(s);

  float acc[MT][NT][4];
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int t = 0; t < NT; t++) acc[m][t][0] = acc[m][t][1] = acc[m][t][2] = acc[m][t][3] = 0.f;
  int stage = 0;
  for (int c = part * L4_WARPS + warp; c < chunks; c += step) {
    issue(stage == 0 ? D - 1 : stage - 1);
    const int k0 = c * L4_CHUNK;
    // x of the chunk: columns 8 i4 .. of each 32, row g of each 8
    uint4 xv[4][NT];
#pragma unroll
    for (int s = 0; s < 4; s++)
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const bool has = r0 + t * 8 + g < a.rows && k0 + s * 32 < a.k;
        xv[s][t] = has ? __ldg(reinterpret_cast<const uint4*>((const __nv_bfloat16*)a.x + (int64_t)(r0 + t * 8 + g) * a.ldx +
                                                              k0 + s * 32 + i4 * 8))
                       : make_uint4(0u, 0u, 0u, 0u);
      }
    // lane i4: scale and zero of the group of part i4
    float scale[MT][2];
    uint32_t zero[MT][2];
#pragma unroll
    for (int m = 0; m < MT; m++)
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const int row = n0 + m * 16 + h * 8 + g;
        const int64_t group = GS == 4 ? iris_paged_block(a.div, c) : c * (4 / GS) + i4 / GS;
        const bool has = row < a.n && k0 + i4 * 32 < a.k;
        scale[m][h] = 0.f;
        zero[m][h] = 0x43084308u;
        if (has) {
          const int64_t at = row * a.lds + group;
          scale[m][h] = a.scale_f32 ? __ldg((const float*)a.scale + at)
                                    : __uint_as_float((uint32_t)__ldg((const uint16_t*)a.scale + at) << 16);
          if (a.zero) zero[m][h] = 0x43004300u + (__ldg(a.zero + row * a.ldz + group) & 127) * 0x10001u;
        }
      }
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    __syncwarp();
    const uint32_t base = ring + stage * Sh::kStage;
    float sum[MT][NT][4];
#pragma unroll
    for (int s = 0; s < 4; s++) {
      if (s % GS == 0) {
#pragma unroll
        for (int m = 0; m < MT; m++)
#pragma unroll
          for (int t = 0; t < NT; t++) sum[m][t][0] = sum[m][t][1] = sum[m][t][2] = sum[m][t][3] = 0.f;
      }
      uint32_t p[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; m++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t w;
          asm volatile("ld.shared.u32 %0, [%1];"
                       : "=r"(w)
                       : "r"(base + (m * 16 + h * 8 + g) * 64 + ((s ^ (g >> 1 & 3)) << 4) + i4 * 4));
          const uint32_t z = GS == 4 || !a.zero ? zero[m][h] : __shfl_sync(0xffffffffu, zero[m][h], g * 4 + s);
          nibbles(w, z, p[m][h]);
        }
#pragma unroll
      for (int t = 0; t < NT; t++) {
        const uint4 x = xv[s][t];
        const uint32_t x0 = __byte_perm(x.x, x.z, 0x5410), x1 = __byte_perm(x.x, x.z, 0x7632);
        const uint32_t x2 = __byte_perm(x.y, x.w, 0x5410), x3 = __byte_perm(x.y, x.w, 0x7632);
#pragma unroll
        for (int m = 0; m < MT; m++) {
          mma_bf16(sum[m][t], p[m][0][0], p[m][1][0], p[m][0][1], p[m][1][1], x0, x1);
          mma_bf16(sum[m][t], p[m][0][2], p[m][1][2], p[m][0][3], p[m][1][3], x2, x3);
        }
      }
      if (s % GS == GS - 1) {
#pragma unroll
        for (int m = 0; m < MT; m++) {
          const float s0 = GS == 4 ? scale[m][0] : __shfl_sync(0xffffffffu, scale[m][0], g * 4 + s);
          const float s1 = GS == 4 ? scale[m][1] : __shfl_sync(0xffffffffu, scale[m][1], g * 4 + s);
#pragma unroll
          for (int t = 0; t < NT; t++) {
            acc[m][t][0] += s0 * sum[m][t][0], acc[m][t][1] += s0 * sum[m][t][1];
            acc[m][t][2] += s1 * sum[m][t][2], acc[m][t][3] += s1 * sum[m][t][3];
          }
        }
      }
    }
    __syncwarp();  // this stage is filled again by the next iteration's issue
    stage = stage == D - 1 ? 0 : stage + 1;
  }

  // ---- the warps' sums, then the parts' of a cluster, always in the same order
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);
  constexpr int LD = Sh::kLd, PER = NT * 8 * LD;
#pragma unroll
  for (int m = 0; m < MT; m++)
#pragma unroll
    for (int t = 0; t < NT; t++) {
      float* to = red + warp * PER + (t * 8 + 2 * i4) * LD + m * 16 + g;
      to[0] = acc[m][t][0], to[LD] = acc[m][t][1], to[8] = acc[m][t][2], to[LD + 8] = acc[m][t][3];
    }
  __syncthreads();
  constexpr int OUT = NT * 8 * MT * 16;
  auto store = [&](int e, float y) {
    const int r = r0 + e / (MT * 16), n = n0 + e % (MT * 16);
    if (r >= a.rows || n >= a.n) return;
    if (a.f32) {
      if (a.add) y += ((const float*)a.add)[r * a.ldadd + n];
      ((float*)a.out)[r * a.ldo + n] = y;
    } else {
      if (a.add) y += __bfloat162float(((const __nv_bfloat16*)a.add)[r * a.ldadd + n]);
      ((__nv_bfloat16*)a.out)[r * a.ldo + n] = __float2bfloat16_rn(y);
    }
  };
  for (int e = tid; e < OUT; e += L4_THREADS) {
    float* at = red + e / (MT * 16) * LD + e % (MT * 16);
    float y = at[0];
#pragma unroll
    for (int w = 1; w < L4_WARPS; w++) y += at[w * PER];
    if (a.parts == 1) store(e, y);
    else at[0] = y;  // this thread alone reads and writes these places
  }
  if (a.parts == 1) return;
  __syncwarp();
  iris::cluster_sync();
  for (int e = part * L4_THREADS + tid; e < OUT; e += a.parts * L4_THREADS) {
    float* at = red + e / (MT * 16) * LD + e % (MT * 16);
    float y = 0.f;
    for (int p = 0; p < a.parts; p++) y += *iris::cluster_map(at, p);
    store(e, y);
  }
  __syncwarp();
  iris::cluster_sync();  // the others have read this block's sums
}

// ------------------------------------------------------------------ rounding to 4 bits
// Bound by the bytes of the weights.  Lanes of 8 values each take a group: its
// largest magnitude / 7, rounded to the scale's type, is the scale s; q = round(w /
// s) + 8, ties to even.  A group that holds an infinity or NaN gets the scale NaN.
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
    const int64_t row = has ? i / groups : 0, group = has ? i - row * groups : 0;
    const In* w = (const In*)a.w + row * a.ldw + group * a.group;
    uint32_t top = 0;  // of the magnitudes' bits: an infinity or NaN is above all others
    for (int c = in * 8; has && c < a.group; c += lanes * 8) {
      float x[8];
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
      float x[8];
      eight(w + c, x);
      uint32_t q = 0;
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float v = s > 0.f ? fminf(fmaxf(rintf(x[j] / s), -8.f), 7.f) : 0.f;
        q |= (uint32_t)((int)v + 8) << 4 * j;
      }
      *reinterpret_cast<uint32_t*>(a.q + row * a.ldq + (group * a.group + c) / 2) = q;
    }
  }
}

template <int MT, int NT, int GS>
cudaError_t go(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  using Sh = L4Shape<MT, NT>;
  const int strips = (a->n + MT * 16 - 1) / (MT * 16), blocks = (a->rows + NT * 8 - 1) / (NT * 8);
  const int chunks = (a->k + L4_CHUNK - 1) / L4_CHUNK;
  a->parts = 1;
  while (a->parts < 8 && (int64_t)strips * blocks * a->parts * 2 <= 4 * num_sms && a->parts * L4_WARPS < chunks) a->parts *= 2;
  const dim3 grid((unsigned)strips * a->parts, blocks);
  if (a->parts == 1) return iris::launch_overlapped(linear4_kernel<MT, NT, GS>, grid, dim3(L4_THREADS), Sh::kSmem, stream, *a);
  return iris::launch_cluster_overlapped(linear4_kernel<MT, NT, GS>, grid, dim3(L4_THREADS), Sh::kSmem, a->parts, stream, *a);
}

template <int GS>
cudaError_t rows_variant(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  if (a->rows <= 8) return go<1, 1, GS>(a, num_sms, stream);
  if (a->rows <= 16) return go<1, 2, GS>(a, num_sms, stream);
  return go<2, 4, GS>(a, num_sms, stream);
}

template <int MT, int NT>
cudaError_t shared_limit() {
  const void* k[] = {(const void*)linear4_kernel<MT, NT, 1>, (const void*)linear4_kernel<MT, NT, 2>,
                     (const void*)linear4_kernel<MT, NT, 4>};
  for (const void* f : k) {
    const cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, L4Shape<MT, NT>::kSmem);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

extern "C" cudaError_t iris_linear4_init(void) {
  const cudaError_t e[] = {shared_limit<1, 1>(), shared_limit<1, 2>(), shared_limit<2, 4>()};
  for (cudaError_t x : e)
    if (x != cudaSuccess) return x;
  return cudaSuccess;
}

extern "C" cudaError_t iris_launch_linear4(IrisLinear4* a, int num_sms, cudaStream_t stream) {
  a->div = iris_paged_div(a->group >= L4_CHUNK ? a->group / L4_CHUNK : 1);
  if (a->group == 32) return rows_variant<1>(a, num_sms, stream);
  if (a->group == 64) return rows_variant<2>(a, num_sms, stream);
  return rows_variant<4>(a, num_sms, stream);
}

extern "C" cudaError_t iris_launch_quantize4(const IrisQuantize4* a, int f32, int num_sms, cudaStream_t stream) {
  const int lanes = a->group >= 256 ? 32 : a->group / 8;
  const int64_t blocks = ((int64_t)a->n * (a->k / a->group) * lanes + 255) / 256;
  const int64_t most = (int64_t)num_sms * 64;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (f32) return iris::launch_overlapped(quantize4_kernel<float>, grid, dim3(256), 0, stream, *a);
  return iris::launch_overlapped(quantize4_kernel<__nv_bfloat16>, grid, dim3(256), 0, stream, *a);
}
