// Language-model operators: rotary positions written into a paged key-value
// cache, attention over the cache, and token log probabilities with entropy
// and the best alternatives.  Sums, softmax statistics and rotations are f32;
// bf16 appears where the tensors have it, rounded once on the way out.
#include "iris_kernels.h"

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

// Element offset in the pools of key `p` of sequence `s` (head 0), or -1 where
// the table or the pool has no such key.
__device__ __forceinline__ int64_t key_offset(const iris_gpu_kv_cache_t& c, int s, int p) {
  const int b = p / c.page_size;
  if (b >= c.max_blocks) return -1;
  const int page = c.table[(int64_t)s * c.table_stride + b];
  if (page < 0 || page >= c.num_pages) return -1;
  return (int64_t)page * c.page_stride + (int64_t)(p - b * c.page_size) * c.token_stride;
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
  const int64_t slot = key_offset(a.cache, seq, pos);
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
// One block per (row, query head); warp w takes the keys w, w + 4, ..., a
// lane HD / 32 columns, with a running maximum and sum per warp, joined at the end.
template <int HD>
__global__ void __launch_bounds__(128) paged_attention_kernel(const __grid_constant__ IrisPagedAttention a) {
  constexpr int C = HD / 32;
  __shared__ float sm_m[4], sm_l[4], sm_o[4][HD];
  const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int seq = a.seq ? a.seq[t] : t;
  if (seq < 0 || seq >= a.cache.num_seqs) return;
  const int64_t cap = (int64_t)a.cache.max_blocks * a.cache.page_size;
  const int64_t last = min((int64_t)a.pos[t], cap - 1);
  const int kvh = h / (a.heads / a.cache.kv_heads);
  const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (int64_t)t * a.ldq + h * HD;
  float qv[C], o[C], m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < C; i++) qv[i] = __bfloat162float(q[lane * C + i]), o[i] = 0.f;
  for (int64_t j = warp; j <= last; j += 4) {
    const int64_t at = key_offset(a.cache, seq, (int)j);
    if (at < 0) continue;
    const __nv_bfloat16* k = (const __nv_bfloat16*)a.cache.k + at + (int64_t)kvh * a.cache.head_stride + lane * C;
    const __nv_bfloat16* v = (const __nv_bfloat16*)a.cache.v + at + (int64_t)kvh * a.cache.head_stride + lane * C;
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < C; i++) x += qv[i] * __bfloat162float(k[i]);
#pragma unroll
    for (int s = 16; s; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
    x *= a.scale;
    const float mn = fmaxf(m, x), f = expf(m - mn), p = expf(x - mn);
    l = l * f + p;
#pragma unroll
    for (int i = 0; i < C; i++) o[i] = o[i] * f + p * __bfloat162float(v[i]);
    m = mn;
  }
  if (lane == 0) sm_m[warp] = m, sm_l[warp] = l;
#pragma unroll
  for (int i = 0; i < C; i++) sm_o[warp][lane * C + i] = o[i];
  __syncthreads();
  const float mm = fmaxf(fmaxf(sm_m[0], sm_m[1]), fmaxf(sm_m[2], sm_m[3]));
  float f[4], sum = 0.f;
#pragma unroll
  for (int w = 0; w < 4; w++) f[w] = sm_l[w] == 0.f ? 0.f : expf(sm_m[w] - mm), sum += f[w] * sm_l[w];
  __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)t * a.ldo + h * HD;
  for (int c = threadIdx.x; c < HD; c += 128) {
    float y = 0.f;
#pragma unroll
    for (int w = 0; w < 4; w++) y += f[w] * sm_o[w][c];
    out[c] = __float2bfloat16_rn(sum == 0.f ? 0.f : y / sum);
  }
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

extern "C" size_t iris_paged_attention_ws_bytes(const iris_gpu_kv_cache_t* cache, int heads, int num_sms) {
  (void)cache, (void)heads, (void)num_sms;
  return 16;
}

extern "C" cudaError_t iris_launch_paged_attention(const IrisPagedAttention* a, int num_sms, cudaStream_t stream,
                                                   int* launches) {
  (void)num_sms;
  *launches = 1;
  const dim3 grid(a->rows, a->heads);
  if (a->cache.head_dim == 64)
    paged_attention_kernel<64><<<grid, 128, 0, stream>>>(*a);
  else if (a->cache.head_dim == 128)
    paged_attention_kernel<128><<<grid, 128, 0, stream>>>(*a);
  else
    paged_attention_kernel<256><<<grid, 128, 0, stream>>>(*a);
  return cudaGetLastError();
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
