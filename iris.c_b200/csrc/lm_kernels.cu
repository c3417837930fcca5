// Language-model operators: rotary positions written into a paged key-value
// cache, attention over the cache, and token log probabilities with entropy
// and the best alternatives.  Sums, softmax statistics and rotations are f32;
// bf16 appears where the tensors have it, rounded once on the way out.
#include "iris_kernels.h"
#include "paged.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <math.h>
#include <stdint.h>

namespace {

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

__device__ __forceinline__ float2 unpack2(uint32_t u) {
  return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xFFFF0000u));
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float x[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const float2 a = unpack2(u.x), b = unpack2(u.y), c = unpack2(u.z), d = unpack2(u.w);
  x[0] = a.x, x[1] = a.y, x[2] = b.x, x[3] = b.y, x[4] = c.x, x[5] = c.y, x[6] = d.x, x[7] = d.y;
}

__device__ __forceinline__ void load8(const float* p, float x[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
}

// ------------------------------------------------------------------ rotary positions into the cache
// One block per token and slice of its heads.  The angles of a token are the
// same for all its heads, so the block evaluates them once: pair i turns by
// pos * turns[i] (64-bit, wrapping at a whole turn), whose top 32 bits as a
// signed fraction of a half turn go to sincospi.  Then HD / 8 lanes take a
// head, 8 columns each: norm by a shuffle reduction over them, the half
// layout's partner columns by one shuffle (rot_dim / 2 is a multiple of 8).
template <typename In, int HD>
__global__ void __launch_bounds__(256) rope_append_kernel(const __grid_constant__ IrisRopeAppend a) {
  constexpr int LPH = HD / 8, GROUPS = 256 / LPH;
  __shared__ __align__(16) float cs[128], sn[128];
  const int t = blockIdx.x;
  const int seq = a.seq[t], pos = a.pos[t];
  if (seq < 0 || seq >= a.cache.num_seqs || pos < 0) return;
  const int rd = a.rope.rot_dim;
  for (int i = threadIdx.x; i < rd / 2; i += 256) {
    const uint64_t turn = (uint64_t)pos * a.rope.turns[i];
    float s, c;
    sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
    cs[i] = c * a.rope.amplitude;
    sn[i] = s * a.rope.amplitude;
  }
  __syncthreads();
  const int nh = a.heads, nkv = a.cache.kv_heads, total = nh + 2 * nkv;
  const int lane = threadIdx.x % LPH, c0 = lane * 8;
  const int page = iris_paged_page(&a.cache, seq, pos);
  const int64_t slot = page < 0 ? -1 : iris_paged_offset(&a.cache, page, pos);
  for (int h0 = blockIdx.y * GROUPS; h0 < total; h0 += gridDim.y * GROUPS) {
    const int h = h0 + threadIdx.x / LPH;
    const bool live = h < total, is_q = h < nh, is_k = !is_q && h < nh + nkv;
    float x[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (live) {
      const In* src = is_q ? (const In*)a.q + (int64_t)t * a.ldq + h * HD
                           : is_k ? (const In*)a.k + (int64_t)t * a.ldk + (h - nh) * HD
                                  : (const In*)a.v + (int64_t)t * a.ldv + (h - nh - nkv) * HD;
      load8(src + c0, x);
    }
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) ss += x[i] * x[i];
#pragma unroll
    for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    const float* w = is_q ? a.q_norm : is_k ? a.k_norm : nullptr;
    if (live && w) {
      const float r = 1.0f / sqrtf(ss * (1.0f / HD) + a.eps);
      float wv[8];
      load8(w + c0, wv);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] = x[i] * r * wv[i];
    }
    if (rd) {
      const bool turned = c0 < rd && (is_q || is_k);
      if (a.rope.layout == IRIS_ROPE_INTERLEAVED) {
        if (turned) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const float c = cs[c0 / 2 + i], s = sn[c0 / 2 + i], u = x[2 * i], v = x[2 * i + 1];
            x[2 * i] = u * c - v * s;
            x[2 * i + 1] = u * s + v * c;
          }
        }
      } else {
        const bool upper = c0 >= rd / 2;
        const int from = c0 >= rd ? lane : upper ? lane - rd / 16 : lane + rd / 16;
        const int i0 = upper ? c0 - rd / 2 : c0;
#pragma unroll
        for (int i = 0; i < 8; i++) {
          const float y = __shfl_sync(0xffffffffu, x[i], from, LPH);
          if (turned) x[i] = upper ? y * sn[i0 + i] + x[i] * cs[i0 + i] : x[i] * cs[i0 + i] - y * sn[i0 + i];
        }
      }
    }
    if (!live || (!is_q && slot < 0)) continue;
    __nv_bfloat16* dst;
    if (is_q)
      dst = (__nv_bfloat16*)a.q_out + (int64_t)t * a.ldq_out + h * HD;
    else if (is_k)
      dst = (__nv_bfloat16*)a.cache.k + slot + (int64_t)(h - nh) * a.cache.head_stride;
    else
      dst = (__nv_bfloat16*)a.cache.v + slot + (int64_t)(h - nh - nkv) * a.cache.head_stride;
    *reinterpret_cast<uint4*>(dst + c0) =
        make_uint4(pack2(x[0], x[1]), pack2(x[2], x[3]), pack2(x[4], x[5]), pack2(x[6], x[7]));
  }
}

// ------------------------------------------------------------------ attention over the cache
// Bound by the cache's bytes (4 flops a byte and query head): the kernel is a
// stream of key and value rows.  Every CTA gets an equal share of all key tiles
// (paged.h), so sequences of any mix of lengths, one long one included, keep
// every SM loading to the end.  Each warp takes 16 keys of a tile through its
// own ring of cp.async stages (no barriers in the loop; page numbers are read a
// stage ahead, so the loads run on across rows and units), and keeps its own
// running maximum m, sum l and output o:
//   s = q k^T      mma m16n8k16, rows = up to 8 query heads of the head's group
//   p = 2^(s c - m), c = scale log2(e);  l = l 2^(m_old - m) + sum p
//   o = o 2^(m_old - m) + p v
// The 8 unused rows of the second product carry what p loses to bf16: row g
// holds bf16(p), row g + 8 holds bf16(p - bf16(p)), and the two halves of o are
// added at the end, so that weights count with 16 bits at no extra instruction
// (with 8 bits the result would be off by sqrt(2) of its own rounding).
// At a unit's end the four warps' sums are joined in shared memory and written,
// or, where a share's border cuts the unit, left for the join kernel.

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void ldsm4(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldsm4t(uint32_t r[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void mma_bf16(float d[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// 16 bytes, or zeros where `bytes` is 0 (nothing is read then)
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}

template <int HD>
struct PagedShape {
  static constexpr int kStages = HD == 64 ? 6 : 3;
  static constexpr int kCtas = HD == 256 ? 1 : 2;                // resident per SM
  static constexpr int kStageBytes = 16 * HD * 2;                // 16 rows of K or of V
  static constexpr int kRing = kStages * 2 * kStageBytes;        // per warp
  static constexpr int kSlot = IRIS_PAGED_HEADS * (HD + 2);      // floats of a piece: m, l, then o
  static constexpr int kSmem = 4 * kRing + 4 * kSlot * 4;
};

// Offset of the first slot in the workspace (floats), after the joins
// {row, unit, later pieces, -} of every share
__host__ __device__ __forceinline__ size_t paged_slots_at(int ctas) { return (size_t)ctas * 4; }

template <int HD>
__global__ void __launch_bounds__(128, PagedShape<HD>::kCtas)
paged_attention_kernel(const __grid_constant__ IrisPagedAttention a) {
  using Sh = PagedShape<HD>;
  constexpr int D = Sh::kStages, CH = HD / 8;  // CH: 16-byte chunks of a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int64_t scan[5];
  __shared__ int64_t found_prefix;
  __shared__ int found_row;
  __shared__ uint32_t seen[4][D];  // per warp and stage: which of its 16 keys exist
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, i4 = lane % 4;
  const iris_gpu_kv_cache_t& cache = a.cache;
  const int units = iris_paged_units(&cache, a.heads), group = a.heads / cache.kv_heads;
  iris::grid_dep_wait();
  iris::grid_dep_launch();

  // rows that see nothing give zeros
  for (int t = blockIdx.x; t < a.rows; t += gridDim.x)
    if (iris_paged_seq(&cache, a.seq, t) >= 0 && a.pos[t] < 0) {
      uint4* o = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (int64_t)t * a.ldo);
      for (int c = tid; c < a.heads * CH; c += 128) o[c] = make_uint4(0u, 0u, 0u, 0u);
    }

  // this share's first tile: prefix sums over the rows, a run of rows per thread
  const int run = (a.rows + 127) / 128, r0 = min(a.rows, tid * run), r1 = min(a.rows, r0 + run);
  int64_t mine = 0;
  for (int t = r0; t < r1; t++) mine += iris_paged_row_tiles(&cache, a.seq, a.pos, t);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  int64_t before = incl - mine, total = 0;
  for (int w = 0; w < 4; w++) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  total *= units;
  const int64_t share = iris_paged_share(total, gridDim.x), start = blockIdx.x * share;
  int4* joins = reinterpret_cast<int4*>(a.ws);
  if (start >= total) {
    if (tid == 0) joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    return;
  }
  {
    const int64_t x = start / units;  // before * units <= start < (before + mine) * units
    if (before <= x && x < before + mine) {
      int t = r0;
      int64_t p = before;
      for (;; t++) {
        const int n = iris_paged_row_tiles(&cache, a.seq, a.pos, t);
        if (x < p + n) break;
        p += n;
      }
      found_row = t;
      found_prefix = p;
    }
  }
  __syncthreads();
  iris_paged_at_t at;
  at.t = found_row;
  iris_paged_row(&at, &cache, a.seq, a.pos);
  {
    const int64_t rest = start - found_prefix * units;
    at.u = (int)(rest / at.n);
    at.i = (int)(rest - (int64_t)at.u * at.n);
  }
  const int64_t count = min(share, total - start);
  if (tid == 0) joins[blockIdx.x] = make_int4(at.t, at.u, iris_paged_join(&at, share), 0);

  const int rtiles = units / cache.kv_heads;
  const uint32_t ring = iris::smem_u32(smem) + warp * Sh::kRing;
  float* red = reinterpret_cast<float*>(smem + 4 * Sh::kRing);

  // ---- loads, up to D - 1 stages ahead of the arithmetic
  iris_paged_at_t ld = at;
  int64_t to_load = count;
  auto find_page = [&]() {  // of this lane's key (lanes 16-31 as lanes 0-15)
    const int p = ld.i * IRIS_PAGED_TILE + warp * 16 + (lane & 15);
    return p < ld.len ? iris_paged_page(&cache, ld.s, p) : -1;
  };
  int page = find_page();
  auto issue = [&](int stage) {
    if (to_load > 0) {
      const int p = ld.i * IRIS_PAGED_TILE + warp * 16 + (lane & 15);
      const uint32_t have = __ballot_sync(0xffffffffu, page >= 0) & 0xFFFFu;
      const int64_t off = page >= 0 ? iris_paged_offset(&cache, page, p) + (int64_t)(ld.u / rtiles) * cache.head_stride : 0;
      if (lane == 0) seen[warp][stage] = have;
      const uint32_t kd = ring + stage * 2 * Sh::kStageBytes, vd = kd + Sh::kStageBytes;
      constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;  // rows one instruction of the warp covers
#pragma unroll
      for (int j = 0; j < 16 / RPI; j++) {
        const int r = j * RPI + lane / CH, ch = lane % CH;
        const int64_t o = __shfl_sync(0xffffffffu, off, r) + ch * 8;
        const int bytes = (have >> r) & 1 ? 16 : 0;
        const uint32_t d = r * (HD * 2) + ((ch ^ (r & 7)) << 4);
        cp_async16(kd + d, (const __nv_bfloat16*)cache.k + o, bytes);
        cp_async16(vd + d, (const __nv_bfloat16*)cache.v + o, bytes);
      }
      if (--to_load > 0) {
        iris_paged_next(&ld, units, &cache, a.seq, a.pos);
        page = find_page();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < D - 1; s++) issue(s);

  // ---- arithmetic
  const float c = a.scale * 1.4426950408889634f;
  uint32_t qf[HD / 16][2];
  float o[HD / 8][4], m = -INFINITY, l = 0.f;
  int heads_here = 0, head0 = 0;
  bool fresh = true, begun_here = false;
  int stage = 0;
  for (int64_t k = 0; k < count; k++) {
    if (fresh) {
      fresh = false;
      begun_here = at.i == 0;
      const int kvh = at.u / rtiles, r = at.u - kvh * rtiles;
      head0 = kvh * group + r * IRIS_PAGED_HEADS;
      heads_here = min(IRIS_PAGED_HEADS, group - r * IRIS_PAGED_HEADS);
      const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (int64_t)at.t * a.ldq + (int64_t)(head0 + g) * HD + 2 * i4;
#pragma unroll
      for (int j = 0; j < HD / 16; j++) {
        qf[j][0] = g < heads_here ? *reinterpret_cast<const uint32_t*>(q + j * 16) : 0u;
        qf[j][1] = g < heads_here ? *reinterpret_cast<const uint32_t*>(q + j * 16 + 8) : 0u;
      }
#pragma unroll
      for (int j = 0; j < HD / 8; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
      m = -INFINITY;
      l = 0.f;
    }
    issue(stage == 0 ? D - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    __syncwarp();
    const uint32_t kd = ring + stage * 2 * Sh::kStageBytes, vd = kd + Sh::kStageBytes;
    const uint32_t have = seen[warp][stage];
    if (have) {
      // scores of 8 heads x 16 keys: s0 keys 2 i4, 2 i4 + 1, s1 the same + 8
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
      // matrices (keys 0-7, columns 0-7), (keys 0-7, 8-15), (keys 8-15, 0-7), (keys 8-15, 8-15) of each 16 columns
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
      for (int j = 0; j < HD / 16; j++) {
        uint32_t b[4];
        ldsm4(b, kd + kr * (HD * 2) + (((2 * j + kc) ^ (kr & 7)) << 4));
        mma_bf16(s0, qf[j][0], 0u, qf[j][1], 0u, b[0], b[1]);
        mma_bf16(s1, qf[j][0], 0u, qf[j][1], 0u, b[2], b[3]);
      }
      float x0 = s0[0] * c, x1 = s0[1] * c, x2 = s1[0] * c, x3 = s1[1] * c;
      if (have != 0xFFFFu) {
        const uint32_t hv = have >> (2 * i4);
        if (!(hv & 1)) x0 = -INFINITY;
        if (!(hv & 2)) x1 = -INFINITY;
        if (!(hv & 0x100)) x2 = -INFINITY;
        if (!(hv & 0x200)) x3 = -INFINITY;
      }
      float mn = fmaxf(fmaxf(x0, x1), fmaxf(x2, x3));
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
      mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
      mn = fmaxf(mn, m);
      const float base = mn == -INFINITY ? 0.f : mn;  // scores of -inf weigh nothing
      if (__any_sync(0xffffffffu, mn != m)) {
        const float f = exp2_approx(m - base);
        l *= f;
#pragma unroll
        for (int j = 0; j < HD / 8; j++) o[j][0] *= f, o[j][1] *= f, o[j][2] *= f, o[j][3] *= f;
        m = mn;
      }
      const float p0 = exp2_approx(x0 - base), p1 = exp2_approx(x1 - base), p2 = exp2_approx(x2 - base),
                  p3 = exp2_approx(x3 - base);
      l += (p0 + p1) + (p2 + p3);
      const uint32_t h0 = pack2(p0, p1), h1 = pack2(p2, p3);
      const float2 u0 = unpack2(h0), u1 = unpack2(h1);
      const uint32_t e0 = pack2(p0 - u0.x, p1 - u0.y), e1 = pack2(p2 - u1.x, p3 - u1.y);
      // transposed: (keys 0-7, columns 0-7), (keys 8-15, 0-7), (keys 0-7, 8-15), (keys 8-15, 8-15)
      const int vr = lane & 15, vc = lane >> 4;
#pragma unroll
      for (int j = 0; j < HD / 16; j++) {
        uint32_t b[4];
        ldsm4t(b, vd + vr * (HD * 2) + (((2 * j + vc) ^ (vr & 7)) << 4));
        mma_bf16(o[2 * j], h0, e0, h1, e1, b[0], b[1]);
        mma_bf16(o[2 * j + 1], h0, e0, h1, e1, b[2], b[3]);
      }
    }
    __syncwarp();  // this stage is filled again by the next iteration's issue
    stage = stage == D - 1 ? 0 : stage + 1;
    const bool ends = at.i == at.n - 1;
    if (ends || k == count - 1) {
      // join the four warps' sums of this unit (or piece)
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      float* mine_f = red + warp * Sh::kSlot;
      if (i4 == 0) mine_f[2 * g] = m, mine_f[2 * g + 1] = l;
#pragma unroll
      for (int j = 0; j < HD / 8; j++)
        *reinterpret_cast<float2*>(mine_f + 2 * IRIS_PAGED_HEADS + g * HD + j * 8 + 2 * i4) =
            make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
      __syncthreads();
      const bool whole = ends && begun_here;
      float* slot = a.ws + paged_slots_at(gridDim.x) + (size_t)(2 * blockIdx.x + (begun_here ? 1 : 0)) * Sh::kSlot;
      for (int e = tid; e < heads_here * (HD / 4); e += 128) {
        const int h = e / (HD / 4), col = (e % (HD / 4)) * 4;
        float mm = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) mm = fmaxf(mm, red[w * Sh::kSlot + 2 * h]);
        const float base = mm == -INFINITY ? 0.f : mm;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; w++) {
          const float f = exp2_approx(red[w * Sh::kSlot + 2 * h] - base);
          sum += f * red[w * Sh::kSlot + 2 * h + 1];
          const float4 v = *reinterpret_cast<const float4*>(red + w * Sh::kSlot + 2 * IRIS_PAGED_HEADS + h * HD + col);
          y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
        }
        if (whole) {
          const float r = sum == 0.f ? 0.f : 1.0f / sum;
          *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + (int64_t)at.t * a.ldo + (int64_t)(head0 + h) * HD + col) =
              make_uint2(pack2(y.x * r, y.y * r), pack2(y.z * r, y.w * r));
        } else {
          if (col == 0) slot[2 * h] = mm, slot[2 * h + 1] = sum;
          *reinterpret_cast<float4*>(slot + 2 * IRIS_PAGED_HEADS + h * HD + col) = y;
        }
      }
      __syncthreads();
      fresh = true;
    }
    if (k < count - 1) iris_paged_next(&at, units, &cache, a.seq, a.pos);
  }
}

// One block per (share border, query head of a unit): where the border is the
// first inside its unit, the unit's pieces are added up, in order.
template <int HD>
__global__ void __launch_bounds__(256) paged_join_kernel(const __grid_constant__ IrisPagedAttention a, int ctas) {
  using Sh = PagedShape<HD>;
  constexpr int COLS = HD / 4, PARTS = 256 / COLS;
  __shared__ float4 acc[PARTS][COLS];
  __shared__ float wsum[PARTS], wmax[8];
  const int c = blockIdx.x + 1, h = blockIdx.y, tid = threadIdx.x;
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const int4 join = reinterpret_cast<const int4*>(a.ws)[c];
  if (join.z == 0) return;
  const int units = iris_paged_units(&a.cache, a.heads), group = a.heads / a.cache.kv_heads;
  const int rtiles = units / a.cache.kv_heads, kvh = join.y / rtiles, r = join.y - kvh * rtiles;
  if (h >= group - r * IRIS_PAGED_HEADS) return;
  const float* slots = a.ws + paged_slots_at(ctas);
  auto piece = [&](int p) { return slots + (size_t)(p == 0 ? 2 * c - 1 : 2 * (c + p - 1)) * Sh::kSlot; };
  const int n = join.z + 1;
  float mm = -INFINITY;
  for (int p = tid; p < n; p += 256) mm = fmaxf(mm, piece(p)[2 * h]);
#pragma unroll
  for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  if (tid % 32 == 0) wmax[tid / 32] = mm;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; w++) mm = fmaxf(mm, wmax[w]);
  const float base = mm == -INFINITY ? 0.f : mm;
  const int part = tid / COLS, col = tid % COLS;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  float sum = 0.f;
#pragma unroll 4
  for (int p = part; p < n; p += PARTS) {
    const float* s = piece(p);
    const float f = exp2_approx(s[2 * h] - base);
    const float4 v = *reinterpret_cast<const float4*>(s + 2 * IRIS_PAGED_HEADS + h * HD + col * 4);
    sum += f * s[2 * h + 1];
    y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
  }
  acc[part][col] = y;
  if (col == 0) wsum[part] = sum;
  __syncthreads();
  if (part) return;
  for (int p = 1; p < PARTS; p++) {
    const float4 v = acc[p][col];
    sum += wsum[p];
    y.x += v.x, y.y += v.y, y.z += v.z, y.w += v.w;
  }
  const float f = sum == 0.f ? 0.f : 1.0f / sum;
  const int head = kvh * group + r * IRIS_PAGED_HEADS + h;
  *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + (int64_t)join.x * a.ldo + (int64_t)head * HD + col * 4) =
      make_uint2(pack2(y.x * f, y.y * f), pack2(y.z * f, y.w * f));
}

// ------------------------------------------------------------------ log probabilities
__device__ __forceinline__ float value(const float* p, int64_t i) { return p[i]; }
__device__ __forceinline__ float value(const __nv_bfloat16* p, int64_t i) { return __bfloat162float(p[i]); }

// Order of the alternatives: larger values first, equal ones by id, NaN before
// all; as one whole number a value, larger first.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  if (x != x) return 0xFF800001u;  // one above +inf
  const uint32_t u = __float_as_uint(x + 0.0f);  // -0 counts as 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

template <typename T, typename F>
__device__ T block_reduce(T v, T* red, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  T t = red[0];
  for (int w = 1; w < (int)blockDim.x / 32; w++) t = f(t, red[w]);
  return t;
}

// One block per row: the maximum, the sums, then top_k rounds of the best
// (value, id) below the one before.
template <typename In>
__global__ void __launch_bounds__(256) logprobs_kernel(const __grid_constant__ IrisLogprobs a) {
  __shared__ float redf[8];
  __shared__ unsigned long long redu[8];
  const int r = blockIdx.x;
  const In* x = (const In*)a.logits + (int64_t)r * a.ld;
  auto fmx = [](float u, float v) { return fmaxf(u, v); };
  auto add = [](float u, float v) { return u + v; };
  auto umx = [](unsigned long long u, unsigned long long v) { return u > v ? u : v; };
  float m = -INFINITY;
  for (int i = threadIdx.x; i < a.vocab; i += 256) m = fmaxf(m, value(x, i));
  m = block_reduce(m, redf, fmx);
  float s1 = 0.f, s2 = 0.f;
  const bool none = m == -INFINITY;  // or nothing but NaN, which the sums then show
  for (int i = threadIdx.x; i < a.vocab; i += 256) {
    const float d = none ? value(x, i) : value(x, i) - m, e = expf(d);
    s1 += e;
    s2 += fmaxf(d, -1000.f) * e;  // a logit of -inf adds 0
  }
  s1 = block_reduce(s1, redf, add);
  s2 = block_reduce(s2, redf, add);
  const float lse = s1 == 0.f ? 0.f : m + logf(s1);
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const int t = a.targets[r];
      a.logprob[r] = t >= 0 && t < a.vocab ? value(x, t) - lse : 0.f;
    }
    if (a.entropy) a.entropy[r] = s1 == 0.f ? 0.f : logf(s1) - s2 / s1;
  }
  unsigned long long below = ~0ull;
  for (int k = 0; k < a.top_k; k++) {
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += 256) {
      const unsigned long long c = (unsigned long long)rank_bits(value(x, i)) << 32 | (uint32_t)~i;
      if (c < below) best = umx(best, c);
    }
    best = block_reduce(best, redu, umx);
    below = best;
    if (threadIdx.x == 0) {
      const int id = (int)~(uint32_t)best;
      if (a.top_ids) a.top_ids[(int64_t)r * a.top_k + k] = id;
      if (a.top_logprobs) a.top_logprobs[(int64_t)r * a.top_k + k] = value(x, id) - lse;
    }
  }
}

}  // namespace

// ------------------------------------------------------------------ launches
extern "C" cudaError_t iris_launch_rope_append(const IrisRopeAppend* a, int f32, int num_sms, cudaStream_t stream) {
  const int groups = 256 / (a->cache.head_dim / 8);
  const int slices = (a->heads + 2 * a->cache.kv_heads + groups - 1) / groups;
  // few tokens: a block per slice of heads, so that they run side by side
  const dim3 grid(a->tokens, a->tokens * slices <= 4 * num_sms ? slices : 1);
  auto go = [&](auto kernel) {
    kernel<<<grid, 256, 0, stream>>>(*a);
    return cudaGetLastError();
  };
  if (f32) {
    if (a->cache.head_dim == 64) return go(rope_append_kernel<float, 64>);
    if (a->cache.head_dim == 128) return go(rope_append_kernel<float, 128>);
    return go(rope_append_kernel<float, 256>);
  }
  if (a->cache.head_dim == 64) return go(rope_append_kernel<__nv_bfloat16, 64>);
  if (a->cache.head_dim == 128) return go(rope_append_kernel<__nv_bfloat16, 128>);
  return go(rope_append_kernel<__nv_bfloat16, 256>);
}

// CTAs of an attention launch: as many as the device holds at once, no more than the tables have room for tiles
template <int HD>
static int paged_ctas(const iris_gpu_kv_cache_t* c, int heads, int64_t rows, int num_sms) {
  const int64_t all = (int64_t)num_sms * PagedShape<HD>::kCtas;
  const int64_t room = iris_paged_tiles(iris_paged_len(c, 0x7FFFFFFF));
  const int64_t most = rows * iris_paged_units(c, heads);
  return (int)(most >= all || most * room >= all ? all : most * room);
}

template <int HD>
static cudaError_t launch_paged(const IrisPagedAttention* a, int num_sms, cudaStream_t stream, int* launches) {
  const int ctas = paged_ctas<HD>(&a->cache, a->heads, a->rows, num_sms);
  cudaError_t e = iris::launch_overlapped(paged_attention_kernel<HD>, dim3(ctas), dim3(128), PagedShape<HD>::kSmem,
                                          stream, *a);
  *launches = 1;
  if (e != cudaSuccess || ctas == 1) return e;
  const int group = a->heads / a->cache.kv_heads;
  *launches = 2;
  return iris::launch_overlapped(paged_join_kernel<HD>, dim3(ctas - 1, group < IRIS_PAGED_HEADS ? group : IRIS_PAGED_HEADS),
                                 dim3(256), 0, stream, *a, ctas);
}

template <int HD>
static size_t paged_ws(int num_sms) {
  const int ctas = num_sms * PagedShape<HD>::kCtas;
  return (paged_slots_at(ctas) + (size_t)2 * ctas * PagedShape<HD>::kSlot) * sizeof(float);
}

extern "C" size_t iris_paged_attention_ws_bytes(const iris_gpu_kv_cache_t* cache, int heads, int num_sms) {
  (void)heads;
  return cache->head_dim == 64 ? paged_ws<64>(num_sms) : cache->head_dim == 128 ? paged_ws<128>(num_sms) : paged_ws<256>(num_sms);
}

extern "C" cudaError_t iris_launch_paged_attention(const IrisPagedAttention* a, int num_sms, cudaStream_t stream,
                                                   int* launches) {
  if (a->cache.head_dim == 64) return launch_paged<64>(a, num_sms, stream, launches);
  if (a->cache.head_dim == 128) return launch_paged<128>(a, num_sms, stream, launches);
  return launch_paged<256>(a, num_sms, stream, launches);
}

// dynamic shared memory limits, once per device, so that launches may be captured
extern "C" cudaError_t iris_lm_init(void) {
  cudaError_t e = cudaFuncSetAttribute(paged_attention_kernel<64>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       PagedShape<64>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(paged_attention_kernel<128>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             PagedShape<128>::kSmem);
  if (e == cudaSuccess)
    e = cudaFuncSetAttribute(paged_attention_kernel<256>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             PagedShape<256>::kSmem);
  return e;
}

extern "C" size_t iris_logprobs_ws_bytes(int rows, int vocab) {
  (void)rows, (void)vocab;
  return 16;
}

extern "C" cudaError_t iris_launch_logprobs(const IrisLogprobs* a, int f32, int num_sms, cudaStream_t stream,
                                            int* launches) {
  (void)num_sms;
  *launches = 1;
  if (f32)
    logprobs_kernel<float><<<a->rows, 256, 0, stream>>>(*a);
  else
    logprobs_kernel<__nv_bfloat16><<<a->rows, 256, 0, stream>>>(*a);
  return cudaGetLastError();
}
