// Language-model operators: rotary positions written into a paged key-value
// cache, attention over the cache, and token log probabilities with entropy
// and the best alternatives.  Sums, softmax statistics and rotations are f32;
// bf16 appears where the tensors have it, rounded once on the way out.
#include <type_traits>

#include "iris_kernels.h"
#include "lm_device.cuh"
#include "paged.h"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <math.h>
#include <stdint.h>

namespace {

// ------------------------------------------------------------------ rotary positions into the cache
// Bound by the bytes of Q, K and V, in once and out once.  One block per token
// and slice of its heads; HD / 8 lanes take a head, two runs of 4 columns each:
// the two sides of the same 4 pairs in the half layout, neighbouring runs in the
// interleaved one and behind rot_dim, so that a lane turns its pairs alone and
// has the same angles for every head.  The angles are evaluated once for the
// block: pair i turns by pos * turns[i] (64-bit, wrapping at a whole turn), whose
// top 32 bits as a signed fraction of a half turn go to sincospi.  A lane reads
// all of its heads (ROPE_HEADS at most, by the grid) before anything else, so
// that the chain position -> page -> slot and the angles come at no time of
// their own.
// Measured on 8191 tokens of 32 + 8 + 8 heads of 128, f32 (302 MB, 46.5 us at
// the measured copy rate): 51 us.  Blocks of 64 threads: with 128 it took 1.07
// of that, with 256 1.16 (the instructions per block and per head are half of
// the time's issue slots).
constexpr int ROPE_HEADS = 4, ROPE_THREADS = 64;

__device__ __forceinline__ float4 values4(uint4 u) {
  return make_float4(__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w));
}
__device__ __forceinline__ float4 values4(uint2 u) {
  const float2 a = unpack2(u.x), b = unpack2(u.y);
  return make_float4(a.x, a.y, b.x, b.y);
}
template <typename In> struct Raw4 { using T = uint4; };
template <> struct Raw4<__nv_bfloat16> { using T = uint2; };

// (a, b) of four pairs turned: the pairs' first and second values
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  const float u = a * c - b * s;
  b = a * s + b * c;
  a = u;
}

// A lane's 8 columns of a head (ca .. ca + 3 and cb .. cb + 3) through the norm with weights w (NULL: none) and the rotation
// by c4, s4: of pairs across x and y where `halves`, else, where `turned`, of neighbours.  The head's lanes are together in a
// warp and take the same way.
template <int HD>
__device__ __forceinline__ void norm_turn(float4& x, float4& y, const float* w, float eps, int ca, int cb, bool halves,
                                          bool turned, float4 c4, float4 s4) {
  constexpr int LPH = HD / 8;
  if (w) {
    float ss = ((x.x * x.x + x.y * x.y) + (x.z * x.z + x.w * x.w)) + ((y.x * y.x + y.y * y.y) + (y.z * y.z + y.w * y.w));
    const uint32_t lanes = LPH == 32 ? 0xffffffffu : ((1u << (LPH & 31)) - 1) << (threadIdx.x % 32 / LPH * LPH);
#pragma unroll
    for (int o = LPH / 2; o; o >>= 1) ss += __shfl_xor_sync(lanes, ss, o);
    const float r = rsqrtf(ss * (1.0f / HD) + eps);
    const float4 wa = *reinterpret_cast<const float4*>(w + ca), wb = *reinterpret_cast<const float4*>(w + cb);
    x.x *= r * wa.x, x.y *= r * wa.y, x.z *= r * wa.z, x.w *= r * wa.w;
    y.x *= r * wb.x, y.y *= r * wb.y, y.z *= r * wb.z, y.w *= r * wb.w;
  }
  if (halves) {
    turn(x.x, y.x, c4.x, s4.x), turn(x.y, y.y, c4.y, s4.y), turn(x.z, y.z, c4.z, s4.z), turn(x.w, y.w, c4.w, s4.w);
  } else if (turned) {
    turn(x.x, x.y, c4.x, s4.x), turn(x.z, x.w, c4.y, s4.y), turn(y.x, y.y, c4.z, s4.z), turn(y.z, y.w, c4.w, s4.w);
  }
}

// cos and sin of a pair at a position
__device__ __forceinline__ void angle(uint64_t turns, float amplitude, int pos, float& c, float& s) {
  const uint64_t turn = (uint64_t)pos * turns;
  sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &s, &c);
  c *= amplitude;
  s *= amplitude;
}

template <typename In, int HD>
__global__ void __launch_bounds__(ROPE_THREADS) rope_append_kernel(const __grid_constant__ IrisRopeAppend a) {
  constexpr int LPH = HD / 8, GROUPS = ROPE_THREADS / LPH;
  using Raw = typename Raw4<In>::T;
  __shared__ __align__(16) float cs[128], sn[128];
  const int t = blockIdx.x;
  const int nh = a.heads, nkv = a.cache.kv_heads, total = nh + 2 * nkv;
  const int rd = a.rope.rot_dim, lane = threadIdx.x % LPH;
  const bool turned = lane < rd / 8, halves = a.rope.layout == IRIS_ROPE_HALF && turned;
  const int ca = halves ? lane * 4 : lane * 8, cb = halves ? rd / 2 + lane * 4 : lane * 8 + 4;
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const In* q = (const In*)a.q + (int64_t)t * a.ldq;
  const In* k = (const In*)a.k + (int64_t)t * a.ldk - nh * HD;
  const In* v = (const In*)a.v + (int64_t)t * a.ldv - (nh + nkv) * HD;
  auto row = [&](int h) { return (h < nh ? q : h < nh + nkv ? k : v) + h * HD; };
  const int first = blockIdx.y * GROUPS + threadIdx.x / LPH, step = gridDim.y * GROUPS;
  const int seq = a.seq[t], pos = a.pos[t];
  Raw ra[ROPE_HEADS], rb[ROPE_HEADS];
#pragma unroll
  for (int i = 0; i < ROPE_HEADS; i++) {
    ra[i] = rb[i] = Raw();
    if (first + i * step < total) {
      const In* x = row(first + i * step);
      ra[i] = *reinterpret_cast<const Raw*>(x + ca);
      rb[i] = *reinterpret_cast<const Raw*>(x + cb);
    }
  }
  if (seq < 0 || seq >= a.cache.num_seqs || pos < 0) return;
  const int block = iris_paged_block(a.div, pos), page = iris_paged_page(&a.cache, seq, block);
  for (int i = threadIdx.x; i < rd / 2; i += ROPE_THREADS) angle(a.rope.turns[i], a.rope.amplitude, pos, cs[i], sn[i]);
  const int64_t slot = page < 0 ? -1 : iris_paged_offset(&a.cache, page, pos - block * a.cache.page_size);
  __nv_bfloat16* qo = (__nv_bfloat16*)a.q_out + (int64_t)t * a.ldq_out;
  __nv_bfloat16* ko = (__nv_bfloat16*)a.cache.k + slot;
  __nv_bfloat16* vo = (__nv_bfloat16*)a.cache.v + slot;
  __syncthreads();
  float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
  if (turned) c4 = *reinterpret_cast<const float4*>(cs + lane * 4), s4 = *reinterpret_cast<const float4*>(sn + lane * 4);
  auto one = [&](int h, float4 x, float4 y) {
    const bool is_q = h < nh, is_v = h >= nh + nkv;
    if (!is_v) norm_turn<HD>(x, y, is_q ? a.q_norm : a.k_norm, a.eps, ca, cb, halves, turned, c4, s4);
    if (!is_q && slot < 0) return;
    __nv_bfloat16* to = is_q ? qo + h * HD : is_v ? vo + (int64_t)(h - nh - nkv) * a.cache.head_stride
                                                  : ko + (int64_t)(h - nh) * a.cache.head_stride;
    *reinterpret_cast<uint2*>(to + ca) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
    *reinterpret_cast<uint2*>(to + cb) = make_uint2(pack2(y.x, y.y), pack2(y.z, y.w));
  };
#pragma unroll
  for (int i = 0; i < ROPE_HEADS; i++)
    if (first + i * step < total) one(first + i * step, values4(ra[i]), values4(rb[i]));
}

// ------------------------------------------------------------------ keys and values into an 8-bit cache
// A scale is shared by a block of tokens, so the tokens of a call that belong to one
// block of the cache (its mates) are taken together, by the thread block that meets
// the first of them: it looks for the others among all tokens of the call, in
// whatever order they stand (a token whose mate is the row before is left out at
// once, so that a prompt's rows are searched once a block of the cache).  Lanes hold
// columns as above; a warp has a (head, K or V) and BATCH of its mates in
// registers, and goes over the mates twice, for the largest magnitude and, behind the
// scale, for the values, from the registers where all fit.  Other blocks of the same
// launch do the queries, 64 threads a token as above.
// The search goes with the product of the call's tokens and the cache's blocks that
// they fill.  bf16, 32 + 8 + 8 heads of 128, blocks of 16, beside rope_append: a prompt
// of 8192 63 us (36), of 32768 320 (138), of 131072 2500 (542); single tokens of 1024
// sequences 37 (7.5), of 8192 240 (37).
constexpr int APPEND8_THREADS = 256, APPEND8_WARPS = APPEND8_THREADS / 32;
constexpr int APPEND8_TOKENS = 8;  // that a block goes through where there are many

// four values at a scale as e4m3, what is not finite as NaN
__device__ __forceinline__ uint32_t to_e4m3(float4 x, float f) {
  auto value = [&](float v) { return fabsf(v) <= 3.4028235e38f ? v * f : __uint_as_float(0x7FC00000u); };
  uint32_t r;
  asm("{\n\t.reg .b16 a, b;\n\tcvt.rn.satfinite.e4m3x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e4m3x2.f32 b, %4, %3;\n\t"
      "mov.b32 %0, {a, b};\n\t}"
      : "=r"(r)
      : "f"(value(x.x)), "f"(value(x.y)), "f"(value(x.z)), "f"(value(x.w)));
  return r;
}
__device__ __forceinline__ uint32_t scaled_e4m3(uint32_t w, float f) {
  uint32_t lo, hi;
  e4m3_to_f16(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&lo)), b = __half22float2(*reinterpret_cast<const __half2*>(&hi));
  return to_e4m3(make_float4(a.x, a.y, b.x, b.y), f);
}

// the larger of the magnitudes' bits, of finite ones
__device__ __forceinline__ uint32_t most_bits(uint32_t top, float4 x) {
  const float v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const uint32_t b = __float_as_uint(v[i]) & 0x7FFFFFFFu;
    top = b < 0x7F800000u && b > top ? b : top;
  }
  return top;
}

// exponent of the least scale that brings a magnitude within 448 = 1.75 * 2^8
__device__ __forceinline__ int exponent8(uint32_t bits) {
  const int e = (int)(bits >> 23) - 8 + ((bits & 0x7FFFFFu) > 0x600000u);
  return min(max(e, IRIS_EXP8_MIN), IRIS_EXP8_MAX);
}

// grid: kv_blocks of them for keys and values, items (head, K or V) in turn, `per` tokens each; then the queries, `slices` of the
// heads in turn
struct Append8Plan {
  int kv_blocks, items, per, slices;
};

// MANY: tokens.  Half as many mates in registers and twice the blocks on an SM: 8191 tokens of 32 + 8 + 8 heads of 128, f32, 94 us
// -> 75; 64 tokens 6.4 -> 8.3.  At 128 columns a block of 16 tokens is more than the 8 held then, so that its rows are read, and
// their angles worked out, twice; and f32 at 64 registers spills (some 310 bytes of stores and 450 of loads a thread).
template <typename In, int HD, bool MANY>
__global__ void __launch_bounds__(APPEND8_THREADS, MANY ? 4 : 2) rope_append8_kernel(const __grid_constant__ IrisRopeAppend a,
                                                                          const __grid_constant__ Append8Plan plan) {
  constexpr int LPH = HD / 8, UNITS = 32 / LPH;               // lanes of a (token, head), of which a warp takes UNITS
  constexpr int MOST = MANY ? 4 : 8, ROUNDS = 16 / UNITS < MOST ? 16 / UNITS : MOST, BATCH = ROUNDS * UNITS;  // slots held at a time
  using Raw = typename Raw4<In>::T;
  __shared__ __align__(16) float cs[16][HD / 2], sn[16][HD / 2];
  __shared__ uint64_t turns[HD / 2];  // (from the arguments each lane's own costs a turn of its own)
  __shared__ int rows[128];  // of the call, by the block's slots
  __shared__ int first;
  const int tid = threadIdx.x, lane = tid % LPH, unit = tid % 32 / LPH;
  const int nkv = a.cache.kv_heads, rd = a.rope.rot_dim, size = a.exp.block;
  const bool turned = lane < rd / 8, halves = a.rope.layout == IRIS_ROPE_HALF && turned;
  const int ca = halves ? lane * 4 : lane * 8, cb = halves ? rd / 2 + lane * 4 : lane * 8 + 4;
  for (int i = tid; i < rd / 2; i += APPEND8_THREADS) turns[i] = a.rope.turns[i];
  __syncthreads();
  iris::grid_dep_wait();
  iris::grid_dep_launch();

  if ((int)blockIdx.x >= plan.kv_blocks) {  // queries
    constexpr int GROUPS = ROPE_THREADS / LPH, SUBS = APPEND8_THREADS / ROPE_THREADS;
    const int b = (int)blockIdx.x - plan.kv_blocks, sub = tid / ROPE_THREADS, in = tid % ROPE_THREADS;
    const int t = b / plan.slices * SUBS + sub, nh = a.heads;
    if (t >= a.tokens) return;
    const int head0 = b % plan.slices * GROUPS + in / LPH, step = plan.slices * GROUPS;
    const In* q = (const In*)a.q + (int64_t)t * a.ldq;
    const int seq = a.seq[t], pos = a.pos[t];
    Raw ra[ROPE_HEADS], rb[ROPE_HEADS];
#pragma unroll
    for (int i = 0; i < ROPE_HEADS; i++) {
      ra[i] = rb[i] = Raw();
      if (head0 + i * step < nh) {
        ra[i] = *reinterpret_cast<const Raw*>(q + (head0 + i * step) * HD + ca);
        rb[i] = *reinterpret_cast<const Raw*>(q + (head0 + i * step) * HD + cb);
      }
    }
    if (seq < 0 || seq >= a.cache.num_seqs || pos < 0) return;  // (all threads of the token)
    float *c = &cs[0][0] + sub * 128, *s = &sn[0][0] + sub * 128;
    for (int i = in; i < rd / 2; i += ROPE_THREADS) angle(turns[i], a.rope.amplitude, pos, c[i], s[i]);
    asm volatile("bar.sync %0, %1;" ::"r"(sub + 1), "n"(ROPE_THREADS) : "memory");
    float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
    if (turned) c4 = *reinterpret_cast<const float4*>(c + lane * 4), s4 = *reinterpret_cast<const float4*>(s + lane * 4);
    __nv_bfloat16* out = (__nv_bfloat16*)a.q_out + (int64_t)t * a.ldq_out;
#pragma unroll
    for (int i = 0; i < ROPE_HEADS; i++) {
      if (head0 + i * step >= nh) continue;
      float4 x = values4(ra[i]), y = values4(rb[i]);
      norm_turn<HD>(x, y, a.q_norm, a.eps, ca, cb, halves, turned, c4, s4);
      __nv_bfloat16* to = out + (head0 + i * step) * HD;
      *reinterpret_cast<uint2*>(to + ca) = make_uint2(pack2(x.x, x.y), pack2(x.z, x.w));
      *reinterpret_cast<uint2*>(to + cb) = make_uint2(pack2(y.x, y.y), pack2(y.z, y.w));
    }
    return;
  }

  const int item = (int)blockIdx.x % plan.items * APPEND8_WARPS + tid / 32, head = item < nkv ? item : item - nkv;
  const bool works = item < 2 * nkv, is_v = item >= nkv;
  const int t0 = (int)blockIdx.x / plan.items * plan.per, t1 = min(a.tokens, t0 + plan.per);
  for (int t = t0; t < t1; t++) {
    const int seq = a.seq[t], pos = a.pos[t];
    const int seq_before = t ? a.seq[t - 1] : -1, pos_before = t ? a.pos[t - 1] : -1;
    if (seq < 0 || seq >= a.cache.num_seqs || pos < 0) continue;
    const int part = iris_paged_block(a.exp.div, pos), begin = part * size;  // the block of the sequence, its first position
    if (seq_before == seq && pos_before >= 0 && iris_paged_block(a.exp.div, pos_before) == part) continue;
    const int block = iris_paged_block(a.div, pos), page = iris_paged_page(&a.cache, seq, block);
    if (page < 0) continue;
    __syncthreads();  // the last token's mates are done with
    for (int i = tid; i < size; i += APPEND8_THREADS) rows[i] = -1;
    if (tid == 0) first = t;
    __syncthreads();
    auto mate = [&](int u, int its_seq) {
      if (its_seq != seq) return;
      const int p = a.pos[u], at = p - begin;
      if (p < 0 || at < 0 || at >= size) return;
      atomicMax(&rows[at], u);
      atomicMin(&first, u);
    };
    if (size == 1) {  // none but itself
      if (tid == 0) rows[0] = t;
    } else if ((reinterpret_cast<uintptr_t>(a.seq) & 15) == 0) {
      constexpr int FLY = 8;  // 8192 tokens in one round
      const int4* four = reinterpret_cast<const int4*>(a.seq);
      for (int i0 = tid; i0 < a.tokens / 4; i0 += FLY * APPEND8_THREADS) {
        int4 s[FLY];
#pragma unroll
        for (int j = 0; j < FLY; j++)
          s[j] = i0 + j * APPEND8_THREADS < a.tokens / 4 ? __ldg(four + i0 + j * APPEND8_THREADS) : make_int4(-1, -1, -1, -1);
#pragma unroll
        for (int j = 0; j < FLY; j++) {
          const int u = 4 * (i0 + j * APPEND8_THREADS);
          if (s[j].x != seq && s[j].y != seq && s[j].z != seq && s[j].w != seq) continue;
          mate(u, s[j].x), mate(u + 1, s[j].y), mate(u + 2, s[j].z), mate(u + 3, s[j].w);
        }
      }
      if (tid < a.tokens % 4) mate(a.tokens / 4 * 4 + tid, a.seq[a.tokens / 4 * 4 + tid]);
    } else {
      for (int u = tid; u < a.tokens; u += APPEND8_THREADS) mate(u, a.seq[u]);
    }
    __syncthreads();
    if (first != t) continue;

    const int first_slot = begin - block * a.cache.page_size;  // of the page
    const bool fresh = rows[0] >= 0, whole = size <= BATCH;
    const In* from = (const In*)(is_v ? a.v : a.k) + (works ? head : 0) * HD;
    const int64_t ld = is_v ? a.ldv : a.ldk;
    uint8_t* to = (uint8_t*)(is_v ? a.cache.v : a.cache.k) + iris_paged_offset(&a.cache, page, first_slot) +
                  (works ? head : 0) * a.cache.head_stride;
    uint8_t* at_exp = (is_v ? a.exp.v : a.exp.k) + page * a.exp.page_stride +
                      iris_paged_block(a.exp.div, first_slot) * a.exp.block_stride + (works ? head : 0) * a.exp.head_stride;
    const int old = works ? exp8(*at_exp) : 0;
    Raw ra[ROUNDS], rb[ROUNDS];
    int row[ROUNDS];
    // the values of a batch's mates, and their angles
    auto load = [&](int slot0) {
#pragma unroll
      for (int j = 0; j < ROUNDS; j++) {
        const int s = slot0 + j * UNITS + unit;
        row[j] = works && s < size ? rows[s] : -1;
        if (row[j] >= 0) {
          const In* r = from + row[j] * ld;
          ra[j] = *reinterpret_cast<const Raw*>(r + ca);
          rb[j] = *reinterpret_cast<const Raw*>(r + cb);
        }
      }
      if ((int)blockIdx.x % plan.items * APPEND8_WARPS >= nkv) return;  // V alone in this block
      __syncthreads();
      for (int i = tid; i < BATCH * (rd / 2); i += APPEND8_THREADS) {
        const int s = i / (rd / 2), p = i - s * (rd / 2);
        if (slot0 + s < size && rows[slot0 + s] >= 0) angle(turns[p], a.rope.amplitude, begin + slot0 + s, cs[s][p], sn[s][p]);
      }
      __syncthreads();
    };
    auto value = [&](int j, float4& x, float4& y) {
      x = values4(ra[j]), y = values4(rb[j]);
      if (is_v) return;
      float4 c4 = make_float4(1.f, 1.f, 1.f, 1.f), s4 = make_float4(0.f, 0.f, 0.f, 0.f);
      if (turned) {
        c4 = *reinterpret_cast<const float4*>(&cs[j * UNITS + unit][lane * 4]);
        s4 = *reinterpret_cast<const float4*>(&sn[j * UNITS + unit][lane * 4]);
      }
      norm_turn<HD>(x, y, a.k_norm, a.eps, ca, cb, halves, turned, c4, s4);
    };
    uint32_t top = 0;
    for (int slot0 = 0; slot0 < size; slot0 += BATCH) {
      load(slot0);
#pragma unroll
      for (int j = 0; j < ROUNDS; j++) {
        if (row[j] < 0) continue;
        float4 x, y;
        value(j, x, y);
        top = most_bits(most_bits(top, x), y);
      }
    }
    int exp = exponent8(__reduce_max_sync(0xffffffffu, top));
    if (!fresh) exp = max(exp, old);
    if (works && tid % 32 == 0) *at_exp = (uint8_t)exp;
    const float f = scale8(254 - exp), down = scale8(127 + min(0, old - exp));
    for (int slot0 = 0; slot0 < size; slot0 += BATCH) {
      if (!whole) load(slot0);
#pragma unroll
      for (int j = 0; j < ROUNDS; j++) {
        const int s = slot0 + j * UNITS + unit;
        uint8_t* at = to + s * a.cache.token_stride;
        if (row[j] >= 0) {
          float4 x, y;
          value(j, x, y);
          *reinterpret_cast<uint32_t*>(at + ca) = to_e4m3(x, f);
          *reinterpret_cast<uint32_t*>(at + cb) = to_e4m3(y, f);
        } else if (works && s < size && !fresh && exp > old) {  // what was there, to the larger scale
          uint2* w = reinterpret_cast<uint2*>(at + lane * 8);
          *w = make_uint2(scaled_e4m3(w->x, down), scaled_e4m3(w->y, down));
        }
      }
    }
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
// p counts with 16 bits in the product, its first 8 and bf16(the rest) (with 8 the
// result would be off by sqrt(2) of its own rounding; with 16 one value in 500 is
// rounded the other way than the 64-bit result, with f32 weights one in 2000), and
// with all of f32 in l.  Up to 8 heads fill half of the product's
// rows and the second parts the other half, at no extra instruction; the halves
// of o are added at the end.  For 9 to 16 heads on a key-value head the second
// part is a second product.  At head_dim 256 two warps share 16 keys and hold
// half of o's columns each (all of them did not fit a warp's registers).
// At a unit's end the four warps' sums are joined in shared memory and written,
// or, where a share's border cuts the unit, left for the join kernel.

// of two bf16, all bits of each one that is an infinity or NaN
__device__ __forceinline__ uint32_t not_finite2(uint32_t x) {
  return ((x & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) | ((x & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u);
}

// Two weights as a first part of 8 bits, cut off, and a second one of the next 8, rounded.  The last bit of a weight is
// set, so that neither part of one of 2^-100 or more is 0 or less: times an infinite value, both are the infinity.  (The
// second part of a lighter one may round to 0, and 0 times it is NaN.)
__device__ __forceinline__ void split2(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  const uint32_t b0 = __float_as_uint(p0) | 1u, b1 = __float_as_uint(p1) | 1u;
  hi = __byte_perm(b0, b1, 0x7632);
  lo = pack2(__uint_as_float(b0) - __uint_as_float(b0 & 0xFFFF0000u), __uint_as_float(b1) - __uint_as_float(b1 & 0xFFFF0000u));
}

// A cache's elements: bf16, or e4m3 with exponents (an 8-bit cache).
//
// Over 8 bits the products are of f16, which holds every e4m3 value; the queries of
// a head are scaled by a power of two to fill f16's range (steps of 2^-38 of the
// largest, where these are wider than a column's own bits).  A key's scale multiplies its score.  The value's scale 2^ve
// joins the weight instead: with t = s c + ve the running maximum is that of t, p =
// 2^(t - m + 15), in the upper part of f16's range, and l adds up p 2^-ve in f32.  p
// comes in two parts of f16, the second what the first one's rounding left: 22
// bits, or steps of 2^-39 of the largest where that is more.  (One part, 11 bits and
// steps of 2^-24, took 200 us instead of 207 for a prompt of 2047, 104 and 104 for 64
// rows of up to 8192 keys, 32.5 and 34.9 for 64 with 32 heads on 2 of 64.)
typedef __nv_fp8_storage_t e4m3;
template <typename E> constexpr bool kEight = sizeof(E) == 1;
constexpr float UP8 = 15.f;  // (added to t - m, not taken from m: of a large m it would be rounded away)

__device__ __forceinline__ void split8(float p0, float p1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(p0, p1);
  const float2 first = __half22float2(h);
  hi = *reinterpret_cast<const uint32_t*>(&h);
  lo = pack2h(p0 - first.x, p1 - first.y);
}

// bytes of a row of K or V lie in 16-byte chunks; chunk ch of row r is at place swz(ch, r), so that ldmatrix meets no bank
// conflict
template <int BYTES>
__device__ __forceinline__ int swz(int ch, int r) { return BYTES == 64 ? ch ^ (r >> 1 & 3) : ch ^ (r & 7); }

// The scales of 16 (a block's: 64) keys of a stage.
template <int N>
struct Scales8 {
  float k[N];       // 2^(ke - 127)
  float v[N];       // ve - 127
  float v_inv[N];   // 2^(127 - ve)
};
template <int N>
__device__ __forceinline__ void put_scales(Scales8<N>& to, int i, int ke, int ve) {
  to.k[i] = scale8(ke), to.v[i] = (float)(ve - 127), to.v_inv[i] = scale8(254 - ve);
}
// Exponents of a key's place (nothing is done with them here, which would wait for them).
__device__ __forceinline__ void read_exps(const iris_kv_exp_t& x, int page, int slot, int64_t head, int& ke, int& ve) {
  const int64_t at = page * x.page_stride + iris_paged_block(x.div, slot) * x.block_stride + head;
  ke = __ldg(x.k + at);
  ve = __ldg(x.v + at);
}

// Page of block b of sequence s as the table has it, to be held to the pool when it is used, a round later: a comparison
// here would wait for it.
__device__ __forceinline__ int table_page(const iris_gpu_kv_cache_t& c, int s, int b) {
  return b < c.max_blocks ? __ldg(c.table + (int64_t)s * c.table_stride + b) : -1;
}

// A head's queries as f16 for the products over 8 bits: columns 16 j + 4 i4 .. + 3 of each 16 into words `lo` and `hi` of
// qf[j], scaled by a power of two that brings the largest finite one to 2^14 or more.  Returns what undoes it.  (All lanes
// take part; the four of a head have it together.)
template <int HD, int N>
__device__ __forceinline__ float queries8(const __nv_bfloat16* q, bool live, int i4, uint32_t (&qf)[HD / 16][N], int lo, int hi) {
  uint2 u[HD / 16];
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < HD / 16; j++) {
    u[j] = live ? *reinterpret_cast<const uint2*>(q + 16 * j + 4 * i4) : make_uint2(0u, 0u);
    const uint32_t w[4] = {u[j].x << 16, u[j].x, u[j].y << 16, u[j].y};
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t b = w[i] & 0x7FFF0000u;
      top = b < 0x7F800000u && b > top ? b : top;
    }
  }
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
  top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
  const int up = min(268 - (int)(top >> 23), 253);
  const float f = scale8(up);
#pragma unroll
  for (int j = 0; j < HD / 16; j++) {
    const float2 a = unpack2(u[j].x), b = unpack2(u[j].y);
    qf[j][lo] = pack2h(a.x * f, a.y * f);
    qf[j][hi] = pack2h(b.x * f, b.y * f);
  }
  return scale8(254 - up);
}

// of four e4m3, all bits of each one that is NaN
__device__ __forceinline__ uint32_t nan4(uint32_t x) { return __vcmpeq4(x & 0x7F7F7F7Fu, 0x7F7F7F7Fu); }

// HD: head_dim.  MH: query heads of a unit (8 or 16).
template <typename E, int HD, int MH>
struct PagedShape {
  // Keys of a tile that a warp takes.  Over 8 bits 32 have half the steps' shuffles, page numbers and scales (64 rows of 1 to
  // 8192 keys, 32 heads on 8 of 128: 100.3 us instead of 102.6; of few rows, one of 512 keys 6.5 us either way, 8 of 512 9.2
  // and 10.1, one of 2048 10.5 and 10.3; 319 instructions for 16 keys and 4 heads).
  static constexpr int kKeys = kEight<E> ? 32 : 16;
  static constexpr int kGroups = IRIS_PAGED_TILE / kKeys;        // of them
  static constexpr int kPair = HD / 128 ? HD / 128 : 1;          // warps on the same keys, 128 columns of o each
  static constexpr int kThreads = 32 * kGroups * kPair;
  // CTAs on an SM and stages of a ring.  At head_dim 64 (256 rows of 0 to 2048 keys, 14 heads on 2) 4 x 2 took 0.84 and
  // 3 x 4 0.88 of the time of 2 x 6, 5 x 2 1.03 and 6 x 2 1.4 of that of 4 x 2: the arithmetic of 16 short keys is
  // latency and wants warps, until registers spill.  At 128 and 256 a ring of three stages fills shared memory, with MH =
  // 16 two.
  static constexpr int kRow = HD * (int)sizeof(E);               // bytes of a row
  // Over 8 bits (64 rows of 1 to 8192 keys, 32 heads on 8 of 128) 4 CTAs of two warps with 3 stages 100.3 us, 5 x 2 103.7, 6 x 2
  // 109, 3 x 4 168: loads in flight as much as warps.
  static constexpr int kCtas = kEight<E> ? (HD == 64 ? (MH == 16 ? 6 : 8) : HD == 128 ? 4 : 2)
                                         : HD == 64 ? 4 : HD == 128 ? 2 : 1;
  static constexpr int kStages = kEight<E> ? 3 : HD == 64 || MH == 16 ? 2 : 3;
  static constexpr int kStageBytes = kKeys * kRow;               // a warp's rows of K or of V
  static constexpr int kRing = kStages * 2 * kStageBytes;        // of its keys of a tile
  static constexpr int kSlot = MH * (HD + 2);                    // floats of a piece: m, l, then o
  // the sums of a unit's end lie behind the rings; over 8 bits in the place of the tile used last, which is as large
  static constexpr int kSmem = kGroups * (kRing + (kEight<E> ? 0 : kSlot * 4));
  static_assert(!kEight<E> || 2 * kStageBytes >= MH * HD * 4, "a warp's sums fit");
  // column of o of head h in the sums of 16 keys in shared memory, which are laid out as a piece: the heads of a store's
  // half warp, eight or every other one of them, fall into different banks
  __device__ static int col(int h, int c) { return c ^ ((kEight<E> ? h >> 1 : h) & 3) << 3; }
};

// Offset of the first slot in the workspace (floats), after the joins
// of every share
__host__ __device__ __forceinline__ size_t paged_slots_at(int ctas) { return (size_t)ctas * 4; }

// A CTA's first place of the line, and its entry of the joins {row, unit, later pieces, rows of the run}; rows that see
// nothing get their zeros.  `places`: of one unit of a row.  False where there is no tile in its share.
template <int T, typename Places>
__device__ __forceinline__ bool paged_begin(const IrisPagedAttention& a, int units, iris_paged_at_t* at, Places places) {
  constexpr int W = T / 32;
  __shared__ int64_t scan[W];
  __shared__ int64_t found_prefix;
  __shared__ int found_row;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  // this share's first place: prefix sums over the rows, a run of rows per thread (up to 32 rows: in each warp by itself)
  const bool few = a.rows <= 32;
  const int run = (a.rows + T - 1) / T, r0 = min(a.rows, (few ? lane : tid) * run), r1 = min(a.rows, r0 + run);
  int64_t mine = 0;
  for (int t = r0; t < r1; t++) mine += places(t);
  int64_t incl = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += v;
  }
  int64_t before = incl - mine, total = 0;
  if (few) {
    total = __shfl_sync(0xffffffffu, incl, 31);
  } else {
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    for (int w = 0; w < W; w++) {
      if (w < warp) before += scan[w];
      total += scan[w];
    }
  }
  total *= units;
  // (divisions in 32 bits where they do: 64-bit ones take a tenth of a microsecond each)
  const int64_t share =
      total <= 0x7FFFFFFF ? iris_paged_share32((uint32_t)total, gridDim.x) : iris_paged_share(total, gridDim.x);
  const int64_t start = blockIdx.x * share;
  int4* joins = reinterpret_cast<int4*>(a.ws);
  // rows that see nothing give zeros
  for (int t = blockIdx.x; t < a.rows; t += gridDim.x)
    if (iris_paged_seq(&a.cache, a.seq, t) >= 0 && a.pos[t] < 0) {
      uint4* o = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (int64_t)t * a.ldo);
      for (int c = tid; c < a.heads * (a.cache.head_dim / 8); c += T) o[c] = make_uint4(0u, 0u, 0u, 0u);
    }
  if (start >= total) {
    if (tid == 0) joins[blockIdx.x] = make_int4(0, 0, 0, 0);
    return false;
  }
  int64_t prefix;
  {
    // the row whose before * units <= start < (before + mine) * units
    const int64_t x = total <= 0x7FFFFFFF ? (uint32_t)start / (uint32_t)units : start / units;
    const bool here = before <= x && x < before + mine;
    if (few) {
      const int from = __ffs(__ballot_sync(0xffffffffu, here)) - 1;  // run is 1: lane t holds row t
      at->t = from;
      prefix = __shfl_sync(0xffffffffu, before, from);
    } else {
      if (here) {
        int t = r0;
        int64_t p = before;
        for (;; t++) {
          const int n = places(t);
          if (x < p + n) break;
          p += n;
        }
        found_row = t;
        found_prefix = p;
      }
      __syncthreads();
      at->t = found_row;
      prefix = found_prefix;
    }
  }
  const bool any = iris_paged_start(at, start - prefix * units, min(share, total - start), units, &a.cache, a.seq, a.pos);
  if (tid == 0) joins[blockIdx.x] = make_int4(at->t, at->u, any ? iris_paged_join(at, share) : 0, at->count);
  return any;
}

// CLUSTER: few rows and short tables.  A cluster of blocks, or one, takes one unit, an
// equal part of its tiles each, and joins the parts in distributed shared
// memory: one launch, and no round through the workspace.
template <typename E, int HD, int MH, bool CLUSTER>
__global__ void __launch_bounds__(PagedShape<E, HD, MH>::kThreads, PagedShape<E, HD, MH>::kCtas)
paged_attention_kernel(const __grid_constant__ IrisPagedAttention a) {
  using Sh = PagedShape<E, HD, MH>;
  constexpr bool EIGHT = kEight<E>;
  constexpr int D = Sh::kStages, CH = Sh::kRow / 16;  // CH: 16-byte chunks of a row
  constexpr int PAIR = Sh::kPair, T = Sh::kThreads, OC = HD / PAIR;  // OC: columns of o a warp holds
  constexpr bool WIDE = MH == 16;
  extern __shared__ __align__(128) uint8_t smem[];
  constexpr int KEYS = Sh::kKeys, GROUPS = Sh::kGroups;
  __shared__ uint32_t seen[GROUPS][D];  // of a warp's keys of a tile and stage: which exist
  __shared__ __align__(16) Scales8<EIGHT ? KEYS : 1> scales[EIGHT ? GROUPS : 1][EIGHT ? D : 1];
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, i4 = lane % 4;
  const int kg = warp / PAIR, half = warp % PAIR;  // which keys of a tile, which columns of o
  auto sync_keys = [&]() {  // the warps on the same keys
    if constexpr (PAIR == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(kg + 1), "n"(32 * PAIR) : "memory");
  };
  const iris_gpu_kv_cache_t& cache = a.cache;
  const int units = iris_paged_units(&cache, a.heads), group = a.heads / cache.kv_heads;
  iris::grid_dep_wait();
  iris::grid_dep_launch();

  iris_paged_at_t at;
  at.rows = at.span = at.count = 0;
  const uint32_t parts = CLUSTER ? iris::cluster_nctarank() : 1, part = CLUSTER ? iris::cluster_ctarank() : 0;
  bool any = true;
  if constexpr (CLUSTER) {
    const int unit = blockIdx.x / parts;
    at.t = unit / units;
    at.u = unit - at.t * units;
    iris_paged_row(&at, &cache, a.seq, a.pos);
    if (at.n == 0) {  // nothing to see, for the whole cluster
      if (at.s >= 0 && part == 0) {
        const int r = at.u % (units / cache.kv_heads), h0 = at.u / (units / cache.kv_heads) * group + r * MH;
        uint4* o = reinterpret_cast<uint4*>((__nv_bfloat16*)a.out + (int64_t)at.t * a.ldo + (int64_t)h0 * HD);
        for (int c = tid; c < min(MH, group - r * MH) * (HD / 8); c += T) o[c] = make_uint4(0u, 0u, 0u, 0u);
      }
      return;
    }
    at.i = (int)((int64_t)at.n * part / parts);
    at.left = (int)((int64_t)at.n * (part + 1) / parts) - at.i;
    any = at.left > 0;
  } else {
    any = paged_begin<T>(a, units, &at, [&](int t) { return iris_paged_row_places(&cache, a.seq, a.pos, t); });
    if (!any) return;
  }

  const int rtiles = units / cache.kv_heads;
  const uint32_t ring = iris::smem_u32(smem) + kg * Sh::kRing;
  // m and l, and o, of the sums of key group w at a unit's end, behind the use of stage `used`
  __shared__ float2 sums8[EIGHT ? GROUPS : 1][EIGHT ? MH : 1];
  int used = 0;
  auto ml_of = [&](int w) {
    return EIGHT ? sums8[w] : reinterpret_cast<float2*>(smem + GROUPS * Sh::kRing + w * Sh::kSlot * 4);
  };
  auto o_of = [&](int w) {
    return reinterpret_cast<float*>(EIGHT ? smem + w * Sh::kRing + used * 2 * Sh::kStageBytes
                                          : smem + GROUPS * Sh::kRing + (w * Sh::kSlot + 2 * MH) * 4);
  };
  // a cluster's part stays in shared memory, where the first stage's tiles lay (over 8 bits in the sums' order of columns,
  // since the first group's may lie just there: a thread writes what it alone read)
  __shared__ float2 part8[EIGHT ? MH : 1];
  auto part_o = [&](float* slot, int h, int col) { return EIGHT ? slot + h * HD + Sh::col(h, col) : slot + 2 * MH + h * HD + col; };

  // ---- loads, up to D - 1 stages ahead of the arithmetic
  iris_paged_at_t ld = at;
  bool loads = any;
  int page, slot;                  // of this lane's key (with 16, lanes 16-31 as lanes 0-15) of the next tile to load
  int64_t head = 0;                // its head's offset
  int64_t exp_head = 0;            // the same among the exponents
  int ke = 127, ve = 127;          // exponents of this lane's key of the tile loaded last, on their way to shared memory
  int exps_to = -1;                // their stage
  auto find = [&]() {
    const int p = ld.i * IRIS_PAGED_TILE + kg * KEYS + lane % KEYS, b = iris_paged_block(a.div, p);
    slot = p - b * cache.page_size;
    page = p < ld.len ? table_page(cache, ld.s, b) : -1;
    if (ld.i == 0) {
      head = (int64_t)(ld.u / rtiles) * cache.head_stride;
      if constexpr (EIGHT) exp_head = (int64_t)(ld.u / rtiles) * a.exp.head_stride;
    }
  };
  head = (int64_t)(ld.u / rtiles) * cache.head_stride;
  if constexpr (EIGHT) exp_head = (int64_t)(ld.u / rtiles) * a.exp.head_stride;
  if (loads) find();
  auto issue = [&](int stage) {
    if constexpr (EIGHT) {
      // the exponents of the stage before: read a round ago, needed in the next one at the earliest
      if (exps_to >= 0 && half == 0) put_scales(scales[kg][exps_to], lane, exp8(ke), exp8(ve));
      exps_to = loads ? stage : -1;
    }
    if (loads) {
      page = (uint32_t)page < (uint32_t)cache.num_pages ? page : -1;
      const uint32_t have = __ballot_sync(0xffffffffu, page >= 0) & (0xffffffffu >> (32 - KEYS));
      const int64_t off = page >= 0 ? iris_paged_offset(&cache, page, slot) + head : 0;
      if (half == 0 && lane == 0) seen[kg][stage] = have;
      if constexpr (EIGHT) {
        ke = ve = 127;
        if (page >= 0) read_exps(a.exp, page, slot, exp_head, ke, ve);
      }
      const uint32_t kd = ring + stage * 2 * Sh::kStageBytes, vd = kd + Sh::kStageBytes;
      constexpr int RPI = 32 / CH > 0 ? 32 / CH : 1;  // rows one instruction of the warp covers
      if constexpr (EIGHT) {
        // places in 32 bits, counted in 16 bytes: half the instructions of 64-bit ones
        const uint32_t place = (uint32_t)(off >> 4);
        auto copy = [&](auto all) {
#pragma unroll
          for (int j = 0; j < KEYS / RPI / PAIR; j++) {
            const int r = (j * PAIR + half) * RPI + lane / CH, ch = lane % CH;
            const size_t o = (size_t)(__shfl_sync(0xffffffffu, place, r) + ch) * 16;
            const int bytes = decltype(all)::value || (have >> r) & 1 ? 16 : 0;
            const uint32_t d = r * Sh::kRow + (swz<Sh::kRow>(ch, r) << 4);
            cp_async16(kd + d, (const E*)cache.k + o, bytes);
            cp_async16(vd + d, (const E*)cache.v + o, bytes);
          }
        };
        if (have == 0xffffffffu >> (32 - KEYS)) copy(std::true_type());
        else copy(std::false_type());
      }
#pragma unroll
      for (int j = 0; !EIGHT && j < KEYS / RPI / PAIR; j++) {
        const int r = (j * PAIR + half) * RPI + lane / CH, ch = lane % CH;
        const int64_t o = __shfl_sync(0xffffffffu, off, r) + ch * (16 / (int)sizeof(E));
        const int bytes = (have >> r) & 1 ? 16 : 0;
        const uint32_t d = r * Sh::kRow + (swz<Sh::kRow>(ch, r) << 4);
        cp_async16(kd + d, (const E*)cache.k + o, bytes);
        cp_async16(vd + d, (const E*)cache.v + o, bytes);
      }
      loads = iris_paged_more(&ld);
      if (loads) {
        iris_paged_next(&ld, units, &cache, a.seq, a.pos);
        find();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < D - 1; s++) issue(s);

  // ---- arithmetic.  Rows of the products: head g, and head g + 8 where MH is 16.
  constexpr int R = WIDE ? 2 : 1;
  const float c = a.scale * 1.4426950408889634f;
  constexpr int S = EIGHT ? 2 * R : R;  // heads whose sums a lane has part of: g and g + 8; over 8 bits 2 i4, 2 i4 + 1 and 8 more
  uint32_t qf[HD / 16][2 * R];
  float o[EIGHT ? R * OC / 16 : OC / 8][4], m[S], l[S];
  [[maybe_unused]] float cq[S];  // c times what the queries were divided by
  int heads_here = 0, head0 = 0;
  auto begin_unit = [&]() {
    const int kvh = at.u / rtiles, r = at.u - kvh * rtiles;
    head0 = kvh * group + r * MH;
    heads_here = min(MH, group - r * MH);
    const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (int64_t)at.t * a.ldq + (int64_t)(head0 + g) * HD;
#pragma unroll
    for (int h = 0; h < R; h++) {
      const bool live = g + 8 * h < heads_here;
      if constexpr (EIGHT) {
        const float f = c * queries8<HD, 2 * R>(q + h * 8 * HD, live, i4, qf, 2 * h, 2 * h + 1);
        cq[2 * h] = __shfl_sync(0xffffffffu, f, 8 * i4);
        cq[2 * h + 1] = __shfl_sync(0xffffffffu, f, 8 * i4 + 4);
      } else {
#pragma unroll
        for (int j = 0; j < HD / 16; j++) {
          qf[j][h] = live ? *reinterpret_cast<const uint32_t*>(q + 2 * i4 + h * 8 * HD + j * 16) : 0u;
          qf[j][R + h] = live ? *reinterpret_cast<const uint32_t*>(q + 2 * i4 + h * 8 * HD + j * 16 + 8) : 0u;
        }
      }
    }
#pragma unroll
    for (int h = 0; h < S; h++) m[h] = -INFINITY, l[h] = 0.f;
  };
  auto clear = [&]() {
#pragma unroll
    for (auto& x : o) x[0] = x[1] = x[2] = x[3] = 0.f;
  };
  begin_unit();
  clear();
  bool begun_here = at.i == 0;
  int stage = 0;
  for (bool more = any; more;) {
    more = iris_paged_more(&at);
    issue(stage == 0 ? D - 1 : stage - 1);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 1) : "memory");
    sync_keys();
    const uint32_t kd = ring + stage * 2 * Sh::kStageBytes, vd = kd + Sh::kStageBytes;
    const uint32_t have = seen[kg][stage];
    if (!EIGHT && have) {
      // scores of a row and 16 keys: s0 keys 2 i4, 2 i4 + 1 (of head g, then of head g + 8), s1 the same + 8
      float s0[4] = {0.f, 0.f, 0.f, 0.f}, s1[4] = {0.f, 0.f, 0.f, 0.f};
      // matrices (keys 0-7, columns 0-7), (keys 0-7, 8-15), (keys 8-15, 0-7), (keys 8-15, 8-15) of each 16 columns
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
      for (int j = 0; j < HD / 16; j++) {
        uint32_t b[4];
        ldsm4(b, kd + kr * (HD * 2) + (((2 * j + kc) ^ (kr & 7)) << 4));
        const uint32_t a1 = WIDE ? qf[j][1] : 0u, a3 = WIDE ? qf[j][2 * R - 1] : 0u;
        mma_bf16(s0, qf[j][0], a1, qf[j][R], a3, b[0], b[1]);
        mma_bf16(s1, qf[j][0], a1, qf[j][R], a3, b[2], b[3]);
      }
      uint32_t hi[R][2], lo[R][2];
      bool moved = false;
      float f[R];
#pragma unroll
      for (int h = 0; h < R; h++) {
        float x0 = s0[2 * h] * c, x1 = s0[2 * h + 1] * c, x2 = s1[2 * h] * c, x3 = s1[2 * h + 1] * c;
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
        mn = fmaxf(mn, m[h]);
        const float base = mn == -INFINITY ? 0.f : mn;  // scores of -inf weigh nothing
        f[h] = exp2_approx(m[h] - base);
        moved |= mn != m[h];
        m[h] = mn;
        const float p0 = exp2_approx(x0 - base), p1 = exp2_approx(x1 - base), p2 = exp2_approx(x2 - base),
                    p3 = exp2_approx(x3 - base);
        l[h] = l[h] * f[h] + ((p0 + p1) + (p2 + p3));
        split2(p0, p1, hi[h][0], lo[h][0]);
        split2(p2, p3, hi[h][1], lo[h][1]);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < OC / 8; j++) {
          o[j][0] *= f[0], o[j][1] *= f[0];
          o[j][2] *= f[R - 1], o[j][3] *= f[R - 1];
        }
      }
      // transposed: (keys 0-7, columns 0-7), (keys 8-15, 0-7), (keys 0-7, 8-15), (keys 8-15, 8-15)
      const int vr = lane & 15, vc = (lane >> 4) + half * (OC / 8);
#pragma unroll
      for (int j = 0; j < OC / 16; j++) {
        uint32_t b[4];
        ldsm4t(b, vd + vr * (HD * 2) + (((2 * j + vc) ^ (vr & 7)) << 4));
#pragma unroll
        for (int n = 0; n < 2; n++) {
          if constexpr (WIDE) {
            mma_bf16(o[2 * j + n], hi[0][0], hi[1][0], hi[0][1], hi[1][1], b[2 * n], b[2 * n + 1]);
            mma_bf16(o[2 * j + n], lo[0][0], lo[1][0], lo[0][1], lo[1][1], b[2 * n], b[2 * n + 1]);
          } else {
            mma_bf16(o[2 * j + n], hi[0][0], lo[0][0], hi[0][1], lo[0][1], b[2 * n], b[2 * n + 1]);
          }
        }
      }
    }
    if constexpr (EIGHT) {
      if (have) {
        // The products the other way round, keys (then columns) as the 16 rows and heads as the 8 columns: no row is idle, and o
        // of 8 heads takes half the registers.  Of each 16 keys k: scores of g (0, 1) and g + 8 (2, 3), heads 2 i4 and 2 i4 +
        // 1, and 8 more.
        constexpr int KS = KEYS / 16;
        float x[KS][R][4];
        // (keys 0-7, columns 0-15), (keys 0-7, 16-31), (keys 8-15, 0-15), (keys 8-15, 16-31) of each 32 columns, four of
        // them, 4 i4 .. 4 i4 + 3, in a lane's word
        const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int r = 0; r < R; r++) x[k][r][0] = x[k][r][1] = x[k][r][2] = x[k][r][3] = 0.f;
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
          for (int k = 0; k < KS; k++) {  // (a product waits for the one before it on the same 16 keys)
            uint32_t b[4];
            ldsm4(b, kd + (k * 16 + kr) * Sh::kRow + (swz<Sh::kRow>(2 * j + kc, kr) << 4));
#pragma unroll
            for (int n = 0; n < 2; n++) {
              uint32_t a0, a1, a2, a3;
              e4m3_to_f16(b[n], a0, a2);
              e4m3_to_f16(b[2 + n], a1, a3);
#pragma unroll
              for (int r = 0; r < R; r++) mma_f16(x[k][r], a0, a1, a2, a3, qf[2 * j + n][2 * r], qf[2 * j + n][2 * r + 1]);
            }
          }
        const auto& sc = scales[kg][stage];
        float kx[2 * KS], vx[2 * KS], vi[2 * KS];  // of keys 8 i + g
#pragma unroll
        for (int i = 0; i < 2 * KS; i++) kx[i] = sc.k[8 * i + g], vx[i] = sc.v[8 * i + g], vi[i] = sc.v_inv[8 * i + g];
        uint32_t pt[KS][R][2], rest[KS][R][2];
        float f[S];
        bool moved = false;
#pragma unroll
        for (int r = 0; r < R; r++) {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            const int e = 2 * r + h;
            float mn = m[e];
#pragma unroll
            for (int i = 0; i < 2 * KS; i++) {
              float& y = x[i / 2][r][i % 2 * 2 + h];
              y = (y * kx[i]) * cq[e] + vx[i];  // (cq kx may be past f32, where y is not)
              if (have != (0xffffffffu >> (32 - KEYS)) && !(have >> g & 1u << 8 * i)) y = -INFINITY;
              mn = fmaxf(mn, y);
            }
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 4));
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 8));
            mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 16));
            const float base = mn == -INFINITY ? 0.f : mn;  // scores of -inf weigh nothing
            f[e] = exp2_approx(m[e] - base);
            moved |= mn != m[e];
            m[e] = mn;
            float sum = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * KS; i++) {
              float& y = x[i / 2][r][i % 2 * 2 + h];
              y = exp2_approx((y - base) + UP8);
              sum += y * vi[i];
            }
            l[e] = l[e] * f[e] + sum;
          }
#pragma unroll
          for (int k = 0; k < KS; k++) {
#pragma unroll
            for (int i = 0; i < 2; i++) {
              uint32_t hi, lo;
              split8(x[k][r][2 * i], x[k][r][2 * i + 1], hi, lo);
              pt[k][r][i] = transposed(hi), rest[k][r][i] = transposed(lo);
            }
          }
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int j = 0; j < OC / 16; j++)
#pragma unroll
            for (int r = 0; r < R; r++) {
              float* y = o[j * R + r];
              y[0] *= f[2 * r], y[1] *= f[2 * r + 1], y[2] *= f[2 * r], y[3] *= f[2 * r + 1];
            }
        }
        // a lane's word: columns 2 g and 2 g + 1 of keys 2 i4 and 2 i4 + 1 (transposed, as over 16 bits); the rows of the product
        // are the even columns of a chunk and then the odd ones
        const int vr = lane & 15, vc = (lane >> 4) + half * (OC / 16);
#pragma unroll
        for (int k = 0; k < KS; k++)
#pragma unroll
          for (int j = 0; j < OC / 32; j++) {
            uint32_t b[4];
            ldsm4t(b, vd + (k * 16 + vr) * Sh::kRow + (swz<Sh::kRow>(2 * j + vc, vr) << 4));
#pragma unroll
            for (int n = 0; n < 2; n++) {
              uint32_t a0, a1, a2, a3;
              e4m3_to_f16(__byte_perm(b[2 * n], 0u, 0x3120), a0, a1);
              e4m3_to_f16(__byte_perm(b[2 * n + 1], 0u, 0x3120), a2, a3);
#pragma unroll
              for (int r = 0; r < R; r++) {
                mma_f16(o[(2 * j + n) * R + r], a0, a1, a2, a3, pt[k][r][0], pt[k][r][1]);
                mma_f16(o[(2 * j + n) * R + r], a0, a1, a2, a3, rest[k][r][0], rest[k][r][1]);
              }
            }
          }
      }
    }
    sync_keys();  // this stage is filled again by the next iteration's issue
    used = stage;
    stage = stage == D - 1 ? 0 : stage + 1;
    const bool ends = at.i == at.n - 1;
    if (ends || !more) {
      // the sums of the tile's key groups joined: this unit, or the piece of it that is here
#pragma unroll
      for (int h = 0; h < S; h++) {
        constexpr int step = EIGHT ? 4 : 1;  // between the lanes that have a head's parts
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], step);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2 * step);
        if constexpr (EIGHT) l[h] += __shfl_xor_sync(0xffffffffu, l[h], 16);
        const int head = EIGHT ? h / 2 * 8 + 2 * i4 + h % 2 : g + 8 * h;
        if (half == 0 && (EIGHT ? g : i4) == 0) ml_of(kg)[head] = make_float2(m[h], l[h]);
      }
      float* mine_o = o_of(kg) + g * HD;
      if constexpr (EIGHT) {
#pragma unroll
        for (int h = 0; h < S; h++) {
          const int head = h / 2 * 8 + 2 * i4 + h % 2;
#pragma unroll
          for (int j = 0; j < OC / 16; j++) {
            const float* y = o[j * R + h / 2] + h % 2;
            *reinterpret_cast<float2*>(o_of(kg) + head * HD + Sh::col(head, half * OC + j * 16 + 2 * g)) = make_float2(y[0], y[2]);
          }
        }
      }
#pragma unroll
      for (int j = 0; !EIGHT && j < OC / 8; j++) {
        float* to = mine_o + Sh::col(g, half * OC + j * 8 + 2 * i4);
        if constexpr (WIDE) {
          *reinterpret_cast<float2*>(to) = make_float2(o[j][0], o[j][1]);
          *reinterpret_cast<float2*>(to + 8 * HD) = make_float2(o[j][2], o[j][3]);
        } else {
          *reinterpret_cast<float2*>(to) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
        }
      }
      const bool whole = !CLUSTER && ends && begun_here;
      float* slot = CLUSTER ? reinterpret_cast<float*>(smem)
                            : a.ws + paged_slots_at(gridDim.x) + (size_t)(2 * blockIdx.x + (begun_here ? 1 : 0)) * Sh::kSlot;
      __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)at.t * a.ldo + (int64_t)head0 * HD;
      const int heads = heads_here;
      if (more) {  // the next unit's queries come while this one is joined
        iris_paged_next(&at, units, &cache, a.seq, a.pos);
        begin_unit();
        begun_here = true;
      }
      __syncthreads();
      for (int e = tid; e < heads * (HD / 4); e += T) {
        const int h = e / (HD / 4), col = (e % (HD / 4)) * 4;
        float mm = -INFINITY, sum = 0.f;
#pragma unroll
        for (int w = 0; w < GROUPS; w++) mm = fmaxf(mm, ml_of(w)[h].x);
        const float base = mm == -INFINITY ? 0.f : mm;
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < GROUPS; w++) {
          const float2 ml = ml_of(w)[h];
          const float s = exp2_approx(ml.x - base);
          sum += s * ml.y;
          const float4 v = *reinterpret_cast<const float4*>(o_of(w) + h * HD + Sh::col(h, col));
          y.x += s * v.x, y.y += s * v.y, y.z += s * v.z, y.w += s * v.w;
        }
        if (whole) {
          const float r = sum == 0.f ? 0.f : 1.0f / sum;
          *reinterpret_cast<uint2*>(out + h * HD + col) = make_uint2(pack2(y.x * r, y.y * r), pack2(y.z * r, y.w * r));
        } else {
          float2* ml = CLUSTER && EIGHT ? part8 : reinterpret_cast<float2*>(slot);
          if (col == 0) ml[h] = make_float2(mm, sum);
          *reinterpret_cast<float4*>(CLUSTER ? part_o(slot, h, col) : slot + 2 * MH + h * HD + col) = y;
        }
      }
      clear();
      __syncthreads();
    } else {
      at.i++;
      at.left--;
    }
  }
  if constexpr (CLUSTER) {
    float* slot = reinterpret_cast<float*>(smem);
    float2* part_ml = EIGHT ? part8 : reinterpret_cast<float2*>(slot);
    if (!any)
      for (int h = tid; h < heads_here; h += T) part_ml[h] = make_float2(-INFINITY, -1.f);  // no key; a sum is never under 0
    __syncwarp();
    iris::cluster_sync();
    __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)at.t * a.ldo + (int64_t)head0 * HD;
    for (int e = tid + part * T; e < heads_here * (HD / 4); e += T * parts) {
      const int h = e / (HD / 4), col = (e % (HD / 4)) * 4;
      float mm = -INFINITY, sum = 0.f;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      for (uint32_t p = 0; p < parts; p++) {
        const float2 ml = iris::cluster_map(part_ml, p)[h];
        if (ml.y < 0.f) continue;  // no key: its columns were not written
        const float4 v = *reinterpret_cast<const float4*>(part_o(iris::cluster_map(slot, p), h, col));
        const float mn = fmaxf(mm, ml.x), base = mn == -INFINITY ? 0.f : mn;
        const float f = exp2_approx(mm - base), s = exp2_approx(ml.x - base);
        mm = mn;
        sum = f * sum + s * ml.y;
        y.x = f * y.x + s * v.x, y.y = f * y.y + s * v.y, y.z = f * y.z + s * v.z, y.w = f * y.w + s * v.w;
      }
      const float r = sum == 0.f ? 0.f : 1.0f / sum;
      *reinterpret_cast<uint2*>(out + h * HD + col) = make_uint2(pack2(y.x * r, y.y * r), pack2(y.z * r, y.w * r));
    }
    __syncwarp();
    iris::cluster_sync();  // the others have read this block's part
  }
}

// Several rows of a sequence, as the tokens of a prompt: a unit is a run of up
// to 64 / heads (head_dim 256: 128 / heads) consecutive rows of one sequence
// (paged.h), one key-value head and up to 16 of the query heads on it, so that
// the cache is read once for all of them.  Each warp holds 16 (row, head) pairs and
// goes over all keys of a tile, which the block loads together, two tiles ahead;
// what none of its pairs sees it leaves out.  A unit of up to 16 pairs would leave
// all warps but one idle: there four warps take 16 keys of a tile each for all
// pairs, and their sums are joined in shared memory.  Bound by the products, 6 flops
// a score and column, two of them for the second part of p, and by a warp's softmax
// between them: registers allow two warps a scheduler, the tensor pipe of mma.sync
// is active 55 % of the time (a prompt of 8192, 32 heads on 8 of 128: 2636 us, 209
// TFLOP/s counting 4 flops, an eighth of the measured peak).
template <typename E, int HD>
struct RunShape {
  static constexpr int kPairs = HD == 256 ? 128 : 64;             // (row, head) pairs of a unit
  static constexpr int kWarps = kPairs / 16, kThreads = 32 * kWarps;
  // CTAs on an SM: what registers allow (a warp holds queries, scores and o of 16 pairs).  At 128 none spills; at 64 three
  // CTAs spill 34 bytes a thread, at 256 one of eight warps 454
  static constexpr int kCtas = HD == 64 ? 3 : HD == 128 ? 2 : 1;
  static constexpr int kStages = 3;  // (two took 1.07 of the time with a prompt of 2048, 32 heads on 8 of 128)
  // keys whose scores a warp holds at a time; a prompt of 2048, 8 heads on 2 of 256, with four warps: 16 330 us, 32 248,
  // with eight warps 162
  static constexpr int kKeys = HD == 256 ? 32 : 64;
  static constexpr int kRow = HD * (int)sizeof(E);                // bytes of a row
  static constexpr int kPart = IRIS_PAGED_TILE * kRow;            // bytes of K or of V of a tile
  static constexpr int kSlot = kPairs * (HD + 2);                 // floats of a piece, as in PagedShape
  // the sums of a narrow unit take the place of the tile used last, which over 8 bits is too small
  static constexpr int kSmem = kStages * 2 * kPart + (kEight<E> ? 64 * HD * 4 : 0);
};

// query heads of a unit of runs
__device__ __forceinline__ int run_heads(int group) { return group < 16 ? group : 16; }

template <typename E, int HD>
__global__ void __launch_bounds__(RunShape<E, HD>::kThreads, RunShape<E, HD>::kCtas)
paged_runs_kernel(const __grid_constant__ IrisPagedAttention a) {
  using Sh = RunShape<E, HD>;
  constexpr bool EIGHT = kEight<E>;
  constexpr int D = Sh::kStages, CH = Sh::kRow / 16, T = Sh::kThreads, NB = HD / 8;
  constexpr int MINE = IRIS_PAGED_TILE / Sh::kWarps;  // keys of a tile that a warp loads, 16 or 8
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) uint16_t seen[D][4];  // of each 16 keys of a stage's tile: which exist
  __shared__ float2 red_ml[64];
  __shared__ __align__(16) Scales8<EIGHT ? IRIS_PAGED_TILE : 1> scales[EIGHT ? D : 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, g = lane / 4, i4 = lane % 4;
  const iris_gpu_kv_cache_t& cache = a.cache;
  const int units = iris_paged_units(&cache, a.heads), group = a.heads / cache.kv_heads, rtiles = units / cache.kv_heads;
  const int hu = run_heads(group), span = Sh::kPairs / hu;
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  iris_paged_at_t at;
  at.rows = a.rows, at.span = span, at.count = 0;
  if (!paged_begin<T>(a, units, &at, [&](int t) {
        return iris_paged_run_places(&cache, a.seq, a.pos, a.rows, span, t);
      }))
    return;

  // ---- loads, up to D - 1 stages ahead of the arithmetic: each warp its keys of a tile
  iris_paged_at_t ld = at;
  bool loads = true;
  int page, slot;  // of this lane's key (the lanes past a warp's keys as its first) of the next tile to load
  int64_t head;    // its head's offset
  int64_t exp_head = 0;            // the same among the exponents
  int ke = 127, ve = 127;          // exponents of this lane's key of the tile loaded last, on their way to shared memory
  int exps_to = -1;                // their stage
  auto find = [&]() {
    const int p = ld.i * IRIS_PAGED_TILE + warp * MINE + lane % MINE, b = iris_paged_block(a.div, p);
    slot = p - b * cache.page_size;
    page = p < ld.len ? table_page(cache, ld.s, b) : -1;
    head = (int64_t)(ld.u / rtiles) * cache.head_stride;
    if constexpr (EIGHT) exp_head = (int64_t)(ld.u / rtiles) * a.exp.head_stride;
  };
  find();
  const uint32_t ring = iris::smem_u32(smem);
  auto issue = [&](int stage) {
    if constexpr (EIGHT) {
      // the exponents of the stage before: read a round ago, needed behind the next barrier at the earliest
      if (exps_to >= 0 && lane < MINE) put_scales(scales[exps_to], warp * MINE + lane, exp8(ke), exp8(ve));
      exps_to = loads ? stage : -1;
    }
    if (loads) {
      page = (uint32_t)page < (uint32_t)cache.num_pages ? page : -1;
      if constexpr (EIGHT) {
        ke = ve = 127;
        if (page >= 0) read_exps(a.exp, page, slot, exp_head, ke, ve);
      }
      const uint32_t have = __ballot_sync(0xffffffffu, page >= 0) & ((1u << MINE) - 1);
      const int64_t off = page >= 0 ? iris_paged_offset(&cache, page, slot) + head : 0;
      if (lane == 0) {
        if constexpr (MINE == 16) seen[stage][warp] = (uint16_t)have;
        else reinterpret_cast<uint8_t*>(seen[stage])[warp] = (uint8_t)have;
      }
      const uint32_t kd = ring + stage * 2 * Sh::kPart + warp * MINE * Sh::kRow, vd = kd + Sh::kPart;
      constexpr int RPI = 32 / CH;  // rows one instruction of the warp covers
#pragma unroll
      for (int j = 0; j < MINE / RPI; j++) {
        const int r = j * RPI + lane / CH, ch = lane % CH;
        const int64_t o = __shfl_sync(0xffffffffu, off, r) + ch * (16 / (int)sizeof(E));
        const int bytes = (have >> r) & 1 ? 16 : 0;
        const uint32_t d = r * Sh::kRow + (swz<Sh::kRow>(ch, r) << 4);
        cp_async16(kd + d, (const E*)cache.k + o, bytes);
        cp_async16(vd + d, (const E*)cache.v + o, bytes);
      }
      loads = iris_paged_more(&ld);
      if (loads) {
        iris_paged_next(&ld, units, &cache, a.seq, a.pos);
        find();
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  for (int s = 0; s < D - 1; s++) issue(s);

  // ---- arithmetic.  This lane's pairs: e = warp 16 + g and e + 8; pair e is row e / hu, head e % hu of the unit.
  // (`narrow`: a unit of up to 16 pairs, e = g and e + 8 in each of four warps)
  const float c = a.scale * 1.4426950408889634f;
  uint32_t qf[HD / 16][4];
  float o[NB][4], m[2], l[2];
  float cq[2];                  // c times what the queries were divided by
  int row[2], col0[2], len[2];  // the pair's row of the call, its head's first column, its keys (0: no such pair)
  int most = 0, least = 0;      // of the warp's pairs
  bool narrow = false;
  auto begin_unit = [&]() {
    narrow = at.count * hu <= 16;
    const int kvh = at.u / rtiles, r = at.u - kvh * rtiles;
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int e = (narrow && warp < 4 ? 0 : warp * 16) + g + 8 * h, in = e / hu, hh = e - in * hu;
      const bool live = in < at.count && hh < group - r * 16;
      row[h] = at.t + in;
      col0[h] = (kvh * group + r * 16 + hh) * HD;
      len[h] = live ? iris_paged_len(&cache, a.pos[at.t + in]) : 0;
      const __nv_bfloat16* q = (const __nv_bfloat16*)a.q + (int64_t)row[h] * a.ldq + col0[h];
      if constexpr (EIGHT) {
        cq[h] = c * queries8<HD, 4>(q, live, i4, qf, h, 2 + h);
      } else {
#pragma unroll
        for (int j = 0; j < HD / 16; j++) {
          qf[j][h] = live ? *reinterpret_cast<const uint32_t*>(q + 2 * i4 + j * 16) : 0u;
          qf[j][2 + h] = live ? *reinterpret_cast<const uint32_t*>(q + 2 * i4 + j * 16 + 8) : 0u;
        }
      }
      if (!live) row[h] = -1;
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
    // (a pair that does not exist gives nothing, whatever its sums)
    most = (int)__reduce_max_sync(0xffffffffu, (unsigned)max(len[0], len[1]));
    least = (int)__reduce_min_sync(0xffffffffu, (unsigned)min(row[0] < 0 ? 0x7FFFFFFF : len[0], row[1] < 0 ? 0x7FFFFFFF : len[1]));
#pragma unroll
    for (int j = 0; j < NB; j++) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
  };
  begin_unit();
  bool begun_here = at.i == 0;
  int stage = 0;
  for (bool more = true; more;) {
    more = iris_paged_more(&at);
    asm volatile("cp.async.wait_group %0;" ::"n"(D - 2) : "memory");
    __syncthreads();  // this tile has come, and the one before it is done with
    issue(stage == 0 ? D - 1 : stage - 1);
    const uint32_t kd = ring + stage * 2 * Sh::kPart, vd = kd + Sh::kPart;
    const int first = at.i * IRIS_PAGED_TILE;
    // this warp's pairs and keys k0 .. of the tile; `plain`: all pairs see them all
    auto step = [&](auto keys, auto plain, int k0) {
      constexpr int KEYS = decltype(keys)::value;
      constexpr bool PLAIN = decltype(plain)::value;
      const int live = most - first - k0, clear = least - first - k0;  // keys from k0 on that a pair sees, that all see
      // scores of a row and 8 keys: keys 2 i4, 2 i4 + 1 of row g, then of row g + 8
      float s[KEYS / 8][4];
#pragma unroll
      for (int n = 0; n < KEYS / 8; n++) s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
      // matrices (keys 0-7, columns 0-7), (keys 0-7, 8-15), (keys 8-15, 0-7), (keys 8-15, 8-15) of each 16 columns
      const int kr = (lane & 7) + ((lane >> 4) << 3), kc = (lane >> 3) & 1;
      if constexpr (EIGHT) {
#pragma unroll
        for (int j = 0; j < HD / 32; j++)
#pragma unroll
          for (int n = 0; n < KEYS / 16; n++) {
            if (!PLAIN && n * 16 >= live) continue;
            uint32_t b[4];
            ldsm4(b, kd + (k0 + n * 16 + kr) * Sh::kRow + (swz<Sh::kRow>(2 * j + kc, kr) << 4));
#pragma unroll
            for (int i = 0; i < 2; i++) {
              const uint32_t* qj = qf[2 * j + i];
              uint32_t b0, b1;
              e4m3_to_f16(b[i], b0, b1);
              mma_f16(s[2 * n], qj[0], qj[1], qj[2], qj[3], b0, b1);
              e4m3_to_f16(b[2 + i], b0, b1);
              mma_f16(s[2 * n + 1], qj[0], qj[1], qj[2], qj[3], b0, b1);
            }
          }
      }
#pragma unroll
      for (int j = 0; !EIGHT && j < HD / 16; j++)
#pragma unroll
        for (int n = 0; n < KEYS / 16; n++) {
          if (!PLAIN && n * 16 >= live) continue;
          uint32_t b[4];
          ldsm4(b, kd + (k0 + n * 16 + kr) * (HD * 2) + (((2 * j + kc) ^ (kr & 7)) << 4));
          mma_bf16(s[2 * n], qf[j][0], qf[j][1], qf[j][2], qf[j][3], b[0], b[1]);
          mma_bf16(s[2 * n + 1], qf[j][0], qf[j][1], qf[j][2], qf[j][3], b[2], b[3]);
        }
      float mx[2] = {-INFINITY, -INFINITY};
#pragma unroll
      for (int n = 0; n < KEYS / 16; n++) {
        const uint32_t have = seen[stage][k0 / 16 + n];
        const bool all = PLAIN || ((n + 1) * 16 <= clear && have == 0xFFFFu);
        [[maybe_unused]] float2 kx[2], vx[2];  // scales of keys 2 i4, 2 i4 + 1, and 8 more
        if constexpr (EIGHT) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            kx[i] = *reinterpret_cast<const float2*>(scales[stage].k + k0 + n * 16 + 8 * i + 2 * i4);
            vx[i] = *reinterpret_cast<const float2*>(scales[stage].v + k0 + n * 16 + 8 * i + 2 * i4);
          }
        }
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int h = e / 2 % 2, key = e / 4 * 8 + 2 * i4 + e % 2;
          float& x = s[2 * n + e / 4][e % 4];
          if constexpr (EIGHT) x = (x * (e % 2 ? kx[e / 4].y : kx[e / 4].x)) * cq[h] + (e % 2 ? vx[e / 4].y : vx[e / 4].x);
          else x *= c;
          if (!all && (n * 16 + key >= len[h] - first - k0 || !(have >> key & 1))) x = -INFINITY;
          mx[h] = fmaxf(mx[h], x);
        }
      }
      float f[2], base[2];
      bool moved = false;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        float mn = mx[h];
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 1));
        mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, 2));
        mn = fmaxf(mn, m[h]);
        base[h] = mn == -INFINITY ? 0.f : mn;  // scores of -inf weigh nothing
        f[h] = exp2_approx(m[h] - base[h]);
        moved |= mn != m[h];
        m[h] = mn;
        l[h] *= f[h];
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int j = 0; j < NB; j++) o[j][0] *= f[0], o[j][1] *= f[0], o[j][2] *= f[1], o[j][3] *= f[1];
      }
      // transposed: (keys 0-7, columns 0-7), (keys 8-15, 0-7), (keys 0-7, 8-15), (keys 8-15, 8-15)
      const int vr = lane & 15, vc = lane >> 4;
      auto add_values = [&](auto finite) {
#pragma unroll
        for (int n = 0; n < KEYS / 16; n++) {
          if (!PLAIN && n * 16 >= live) continue;
          uint32_t hi[4], lo[4];
          [[maybe_unused]] float2 vi[2];
          if constexpr (EIGHT) {
#pragma unroll
            for (int i = 0; i < 2; i++)
              vi[i] = *reinterpret_cast<const float2*>(scales[stage].v_inv + k0 + n * 16 + 8 * i + 2 * i4);
          }
#pragma unroll
          for (int k = 0; k < 4; k++) {  // rows g, g + 8, g, g + 8; keys 0-7, 0-7, 8-15, 8-15
            const int h = k & 1, b = 2 * n + k / 2;
            float t0 = s[b][2 * h] - base[h], t1 = s[b][2 * h + 1] - base[h];
            if constexpr (EIGHT) t0 += UP8, t1 += UP8;
            const float p0 = exp2_approx(t0), p1 = exp2_approx(t1);
            if constexpr (EIGHT) {
              l[h] += p0 * vi[k / 2].x + p1 * vi[k / 2].y;
              split8(p0, p1, hi[k], lo[k]);
            } else {
              l[h] += p0 + p1;
              split2(p0, p1, hi[k], lo[k]);
            }
          }
          if constexpr (EIGHT) {
#pragma unroll
            for (int j = 0; j < HD / 32; j++) {
              uint32_t b[4];
              ldsm4t(b, vd + (k0 + n * 16 + vr) * Sh::kRow + (swz<Sh::kRow>(2 * j + vc, vr) << 4));
#pragma unroll
              for (int i = 0; i < 2; i++) {
                if constexpr (!decltype(finite)::value) b[2 * i] &= ~nan4(b[2 * i]), b[2 * i + 1] &= ~nan4(b[2 * i + 1]);
                uint32_t e0, e1, d0, d1;  // even and odd columns
                e4m3_to_f16(__byte_perm(b[2 * i], 0u, 0x3120), e0, d0);
                e4m3_to_f16(__byte_perm(b[2 * i + 1], 0u, 0x3120), e1, d1);
                mma_f16(o[4 * j + 2 * i], hi[0], hi[1], hi[2], hi[3], e0, e1);
                mma_f16(o[4 * j + 2 * i + 1], hi[0], hi[1], hi[2], hi[3], d0, d1);
                mma_f16(o[4 * j + 2 * i], lo[0], lo[1], lo[2], lo[3], e0, e1);
                mma_f16(o[4 * j + 2 * i + 1], lo[0], lo[1], lo[2], lo[3], d0, d1);
              }
            }
          }
#pragma unroll
          for (int j = 0; !EIGHT && j < HD / 16; j++) {
            uint32_t b[4];
            ldsm4t(b, vd + (k0 + n * 16 + vr) * (HD * 2) + (((2 * j + vc) ^ (vr & 7)) << 4));
            if constexpr (!decltype(finite)::value) {
#pragma unroll
              for (int k = 0; k < 4; k++) b[k] &= ~not_finite2(b[k]);
            }
            mma_bf16(o[2 * j], hi[0], hi[1], hi[2], hi[3], b[0], b[1]);
            mma_bf16(o[2 * j + 1], hi[0], hi[1], hi[2], hi[3], b[2], b[3]);
            mma_bf16(o[2 * j], lo[0], lo[1], lo[2], lo[3], b[0], b[1]);
            mma_bf16(o[2 * j + 1], lo[0], lo[1], lo[2], lo[3], b[2], b[3]);
          }
        }
      };
      // A value that one of the rows must not see may be an infinity or NaN, which a weight of zero does not take out of
      // the product: where there are any, they go in by themselves, to the rows that see them.
      bool odd = false;
      if (!PLAIN && clear < KEYS) {
        for (int e = max(0, clear) * CH + lane; e < min(KEYS, (live + 15) & ~15) * CH; e += 32) {
          const uint4 v = *reinterpret_cast<const uint4*>(smem + (vd - ring) + (k0 * CH + e) * 16);
          if constexpr (EIGHT) odd |= (nan4(v.x) | nan4(v.y) | nan4(v.z) | nan4(v.w)) != 0;
          else odd |= (not_finite2(v.x) | not_finite2(v.y) | not_finite2(v.z) | not_finite2(v.w)) != 0;
        }
        odd = __any_sync(0xffffffffu, odd);
      }
      if (!odd) {
        add_values(std::true_type());
      } else {
        add_values(std::false_type());
        if constexpr (EIGHT) {
          for (int key = k0; key < k0 + min(KEYS, live); key++)
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
              const uint32_t bad = nan4(*reinterpret_cast<const uint32_t*>(smem + (vd - ring) + key * Sh::kRow +
                                                                           (swz<Sh::kRow>(j, key) << 4) + i4 * 4));
#pragma unroll
              for (int i = 0; i < 4; i++) {
                if (!(bad >> 8 * i & 1)) continue;
                float* to = o[2 * j + i % 2];
                if (key < len[0] - first) to[i / 2] = NAN;
                if (key < len[1] - first) to[2 + i / 2] = NAN;
              }
            }
        }
        for (int key = k0; !EIGHT && key < k0 + min(KEYS, live); key++)
#pragma unroll
          for (int j = 0; j < NB; j++) {
            const uint32_t v = *reinterpret_cast<const uint32_t*>(smem + (vd - ring) + key * (HD * 2) +
                                                                  ((j ^ (key & 7)) << 4) + i4 * 4);
            const uint32_t bad = not_finite2(v);
            if (!bad) continue;
            const float2 x = unpack2(v & bad);  // the finite one as 0
            if (key < len[0] - first) o[j][0] += x.x, o[j][1] += x.y;
            if (key < len[1] - first) o[j][2] += x.x, o[j][3] += x.y;
          }
      }
    };
    if (first < most) {
      const uint2 all = *reinterpret_cast<const uint2*>(seen[stage]);
      const bool plain = first <= least - IRIS_PAGED_TILE && (all.x & all.y) == 0xFFFFFFFFu;
      constexpr std::integral_constant<int, 16> few{};
      constexpr std::integral_constant<int, Sh::kKeys> many{};
      if (narrow) {
        if (plain) step(few, std::true_type(), warp * 16);
        else step(few, std::false_type(), warp * 16);
      } else if (plain) {
#pragma unroll
        for (int k0 = 0; k0 < IRIS_PAGED_TILE; k0 += Sh::kKeys) step(many, std::true_type(), k0);
      } else {
#pragma unroll
        for (int k0 = 0; k0 < IRIS_PAGED_TILE; k0 += Sh::kKeys)
          if (first + k0 < most) step(many, std::false_type(), k0);
      }
    }
    float* red = reinterpret_cast<float*>(smem + (EIGHT ? D : stage) * 2 * Sh::kPart);
    stage = stage == D - 1 ? 0 : stage + 1;
    const bool ends = at.i == at.n - 1;
    if (ends || !more) {  // this unit, or the piece of it that is here
      float* slot = a.ws + paged_slots_at(gridDim.x) + (size_t)(2 * blockIdx.x + (begun_here ? 1 : 0)) * Sh::kSlot;
      if (narrow) __syncthreads();  // all are done with the tile, whose place the sums take
      const bool whole = ends && begun_here;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (row[h] < 0) continue;
        const int e = warp * 16 + g + 8 * h;
        if (whole && !narrow) {
          const float r = l[h] == 0.f ? 0.f : 1.0f / l[h];
          __nv_bfloat16* out = (__nv_bfloat16*)a.out + (int64_t)row[h] * a.ldo + col0[h];
          if constexpr (EIGHT) {
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
              const float *x = o[2 * j] + 2 * h, *y = o[2 * j + 1] + 2 * h;
              *reinterpret_cast<uint2*>(out + j * 16 + 4 * i4) = make_uint2(pack2(x[0] * r, y[0] * r), pack2(x[1] * r, y[1] * r));
            }
          } else {
#pragma unroll
            for (int j = 0; j < NB; j++)
              *reinterpret_cast<uint32_t*>(out + 2 * i4 + j * 8) = pack2(o[j][2 * h] * r, o[j][2 * h + 1] * r);
          }
        } else {
          float* to = (narrow ? red : slot + 2 * Sh::kPairs) + e * HD;
          const int turn = narrow ? (g & 3) << 3 : 0;  // the eight pairs of a store's half warp fall into different banks
          if (i4 == 0) (narrow ? red_ml : reinterpret_cast<float2*>(slot))[e] = make_float2(m[h], l[h]);
          if constexpr (EIGHT) {
#pragma unroll
            for (int j = 0; j < HD / 16; j++) {
              const float *x = o[2 * j] + 2 * h, *y = o[2 * j + 1] + 2 * h;
              *reinterpret_cast<float4*>(to + ((j * 16 + 4 * i4) ^ turn)) = make_float4(x[0], y[0], x[1], y[1]);
            }
          } else {
#pragma unroll
            for (int j = 0; j < NB; j++)
              *reinterpret_cast<float2*>(to + ((j * 8 + 2 * i4) ^ turn)) = make_float2(o[j][2 * h], o[j][2 * h + 1]);
          }
        }
      }
      if (narrow) {
        const int kvh = at.u / rtiles, r = at.u - kvh * rtiles, hs = min(hu, group - r * 16);
        __syncthreads();
        for (int x = threadIdx.x; x < at.count * hu * (HD / 4); x += T) {
          const int e = x / (HD / 4), col = (x % (HD / 4)) * 4, in = e / hu, hh = e - in * hu;
          if (hh >= hs) continue;
          float mm = -INFINITY, sum = 0.f;
#pragma unroll
          for (int w = 0; w < 4; w++) mm = fmaxf(mm, red_ml[w * 16 + e].x);
          const float to_base = mm == -INFINITY ? 0.f : mm;
          float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const float f = exp2_approx(red_ml[w * 16 + e].x - to_base);
            sum += f * red_ml[w * 16 + e].y;
            const float4 v = *reinterpret_cast<const float4*>(red + (w * 16 + e) * HD + (col ^ (e & 3) << 3));
            y.x += f * v.x, y.y += f * v.y, y.z += f * v.z, y.w += f * v.w;
          }
          if (whole) {
            const float f = sum == 0.f ? 0.f : 1.0f / sum;
            *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + (int64_t)(at.t + in) * a.ldo +
                                      (int64_t)(kvh * group + r * 16 + hh) * HD + col) =
                make_uint2(pack2(y.x * f, y.y * f), pack2(y.z * f, y.w * f));
          } else {
            if (col == 0) slot[2 * e] = mm, slot[2 * e + 1] = sum;
            *reinterpret_cast<float4*>(slot + 2 * Sh::kPairs + e * HD + col) = y;
          }
        }
      }
      if (more) {
        iris_paged_next(&at, units, &cache, a.seq, a.pos);
        begin_unit();
        begun_here = true;
      }
    } else {
      at.i++;
      at.left--;
    }
  }
}

// Adds up the pieces of cut units.  A thread takes four columns of a head; where
// those are fewer than the threads, the block has parts that take every
// parts-th piece each and are added at the end.  Two ways to find the pieces:
// many units, most of them in two pieces: a block per share border, which works
// where its border is the first inside a unit, for all heads that fit, and
// reads the first pieces before it knows how many there are; few units in many
// pieces (FEW): a block per unit and head, which works out the unit's borders from
// the rows' lengths while the attention kernel runs (one row, 16 heads on one of
// 128 and 131072 keys, 295 pieces: 24 us, in the first way some 40 more).
constexpr int JOIN_THREADS = 512;

template <int HD, int MH, bool FEW>
__global__ void __launch_bounds__(JOIN_THREADS)
paged_join_kernel(const __grid_constant__ IrisPagedAttention a, int ctas, int per_block) {
  using Sh = PagedShape<__nv_bfloat16, HD, MH>;  // pieces are f32, alike for both
  constexpr int COLS = HD / 4;
  __shared__ float4 acc[JOIN_THREADS];
  __shared__ float2 ml[JOIN_THREADS / COLS];
  const int units = iris_paged_units(&a.cache, a.heads), group = a.heads / a.cache.kv_heads;
  const int width = per_block * COLS;  // threads of a part
  const int parts = JOIN_THREADS / width, part = threadIdx.x / width, i = threadIdx.x - part * width;
  const int h = blockIdx.y * per_block + i / COLS, col = i % COLS;
  const bool works = part < parts && h < min(group, MH);
  const int4* joins = reinterpret_cast<const int4*>(a.ws);
  int c = blockIdx.x + 1, row = 0, unit = 0, n = 0;
  if constexpr (FEW) {
    // the rows are the attention kernel's inputs: nothing that still runs writes them
    row = blockIdx.x / units, unit = blockIdx.x - row * units;
    int64_t begin = 0, total = 0;
    int places = 0;
    for (int t = 0; t < a.rows; t++) {
      const int n_t = iris_paged_row_places(&a.cache, a.seq, a.pos, t);
      if (t < row) begin += n_t;
      if (t == row) places = n_t;
      total += n_t;
    }
    begin = begin * units + (int64_t)unit * places;
    if (places) n = iris_paged_cut(begin, places - IRIS_PAGED_EXTRA, iris_paged_share(total * units, ctas), &c);
    iris::grid_dep_wait();
    iris::grid_dep_launch();
    if (!n) return;
    n++;
  } else {
    iris::grid_dep_wait();
    iris::grid_dep_launch();
  }
  const float* slots = a.ws + paged_slots_at(ctas);
  auto place = [&](int p) { return slots + (size_t)(p == 0 ? 2 * c - 1 : min(2 * (c + p - 1), 2 * ctas - 1)) * Sh::kSlot; };
  auto ml_of = [&](int p) { return *reinterpret_cast<const float2*>(place(p) + 2 * h); };
  auto o_of = [&](int p) { return *reinterpret_cast<const float4*>(place(p) + 2 * MH + h * HD + col * 4); };
  float m = -INFINITY, l = 0.f;
  float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
  auto add = [&](float2 s, float4 v) {
    const float mn = fmaxf(m, s.x), base = mn == -INFINITY ? 0.f : mn;
    const float f = exp2_approx(m - base), e = exp2_approx(s.x - base);
    m = mn;
    l = f * l + e * s.y;
    y.x = f * y.x + e * v.x, y.y = f * y.y + e * v.y, y.z = f * y.z + e * v.z, y.w = f * y.w + e * v.w;
  };
  float2 s0 = make_float2(0.f, 0.f);
  float4 v0 = y;
  if (works) s0 = ml_of(part), v0 = o_of(part);
  if constexpr (!FEW) {
    const int4 j = joins[c];
    if (j.z == 0) return;
    row = j.x, unit = j.y, n = j.z + 1;
  }
  const int rtiles = units / a.cache.kv_heads, kvh = unit / rtiles, r = unit - kvh * rtiles;
  const bool live = works && h < group - r * MH;
  if (live && part < n) add(s0, v0);
  if (live)
    for (int p = part + parts; p < n; p += 4 * parts) {
      float2 s[4];
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] = ml_of(min(p + j * parts, n - 1)), v[j] = o_of(min(p + j * parts, n - 1));
#pragma unroll
      for (int j = 0; j < 4; j++)
        if (p + j * parts < n) add(s[j], v[j]);
    }
  if (parts > 1) {
    acc[threadIdx.x] = y;
    if (col == 0) ml[threadIdx.x / COLS] = make_float2(m, l);
    __syncthreads();
    for (int p = 1; part == 0 && p < parts && p < n; p++) add(ml[(p * width + i) / COLS], acc[p * width + i]);
  }
  if (part || !live) return;
  const float f = l == 0.f ? 0.f : 1.0f / l;
  const int head = kvh * group + r * MH + h;
  *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + (int64_t)row * a.ldo + (int64_t)head * HD + col * 4) =
      make_uint2(pack2(y.x * f, y.y * f), pack2(y.z * f, y.w * f));
}

// The same for pieces of runs: two blocks per share border.
constexpr int RUN_JOIN_THREADS = 256;

template <int HD>
__global__ void __launch_bounds__(RUN_JOIN_THREADS)
paged_runs_join_kernel(const __grid_constant__ IrisPagedAttention a, int ctas) {
  using Sh = RunShape<__nv_bfloat16, HD>;
  constexpr int COLS = HD / 4, SLOT = Sh::kSlot;
  const int units = iris_paged_units(&a.cache, a.heads), group = a.heads / a.cache.kv_heads, rtiles = units / a.cache.kv_heads;
  const int c = blockIdx.x + 1, hu = run_heads(group);
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const int4 j = reinterpret_cast<const int4*>(a.ws)[c];
  if (j.z == 0) return;
  const int n = j.z + 1, kvh = j.y / rtiles, r = j.y - kvh * rtiles;
  const float* slots = a.ws + paged_slots_at(ctas);
  for (int x = blockIdx.y * RUN_JOIN_THREADS + threadIdx.x; x < j.w * hu * COLS; x += gridDim.y * RUN_JOIN_THREADS) {
    const int e = x / COLS, col = x % COLS * 4, in = e / hu, hh = e - in * hu;
    if (hh >= group - r * 16) continue;
    float m = -INFINITY, l = 0.f;
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < n; p += 4) {
      float2 s[4];
      float4 v[4];
#pragma unroll
      for (int k = 0; k < 4; k++) {
        const int q = min(p + k, n - 1);
        const float* slot = slots + (size_t)(q == 0 ? 2 * c - 1 : 2 * (c + q - 1)) * SLOT;
        s[k] = *reinterpret_cast<const float2*>(slot + 2 * e);
        v[k] = *reinterpret_cast<const float4*>(slot + 2 * Sh::kPairs + e * HD + col);
      }
#pragma unroll
      for (int k = 0; k < 4; k++) {
        if (p + k >= n) continue;
        const float mn = fmaxf(m, s[k].x), base = mn == -INFINITY ? 0.f : mn;
        const float f = exp2_approx(m - base), g = exp2_approx(s[k].x - base);
        m = mn;
        l = f * l + g * s[k].y;
        y.x = f * y.x + g * v[k].x, y.y = f * y.y + g * v[k].y, y.z = f * y.z + g * v[k].z, y.w = f * y.w + g * v[k].w;
      }
    }
    const float f = l == 0.f ? 0.f : 1.0f / l;
    *reinterpret_cast<uint2*>((__nv_bfloat16*)a.out + (int64_t)(j.x + in) * a.ldo + (int64_t)(kvh * group + r * 16 + hh) * HD + col) =
        make_uint2(pack2(y.x * f, y.y * f), pack2(y.z * f, y.w * f));
  }
}

// ------------------------------------------------------------------ log probabilities
// Bound by the logits' bytes, and close behind by the exponentials (16 a clock
// and SM) and the instructions around them.  One pass, against the running
// maximum m:
//   s1 = sum e^(x - m),   s2 = sum (x - m) e^(x - m)
// from which log softmax x = (x - m) - log s1 and the entropy log s1 - s2 / s1.
// A new maximum m' turns the sums into f s1 and f (s2 + (m - m') s1), f =
// e^(m - m').  For the alternatives the pass leaves the largest value of every
// block: the k largest values of a row lie in the k blocks with the largest
// maxima (each of k blocks ahead of another one holds a value ahead of all of
// the other's), so what follows reads those k blocks again and nothing else.

// LP_BLOCK values a block: vocab / LP_BLOCK maxima and k LP_BLOCK values are read again, alike at
// LP_BLOCK = sqrt(vocab / k), 87 for 151936 and k = 20; 256 is one load of the warp
constexpr int LP_BLOCK = 256;
constexpr int LP_LOADS = 8;    // 16-byte loads of a lane in flight
constexpr int LP_CLUSTER = 8, LP_CLUSTER_BLOCKS = 8192;  // blocks on a row where there are few, most blocks of values then

template <typename In>
struct LpShape {
  static constexpr int kVec = 16 / sizeof(In);                  // values of a load
  static constexpr int kPer = LP_BLOCK / (32 * kVec);           // loads of a block
  static constexpr int kBlocks = LP_LOADS / kPer;               // blocks in flight
};

// Two f32 in one register pair, for the packed instructions.
__device__ __forceinline__ uint64_t pair(float a, float b) {
  uint64_t v;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
  return v;
}
__device__ __forceinline__ float2 halves(uint64_t v) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
  return f;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Sums against m, moved to mn >= m.
__device__ __forceinline__ void raise(float& m, float& s1, float& s2, float mn) {
  if (m != mn) {
    if (m != -INFINITY) {
      const float d = m - mn, f = exp2_approx(d * kLog2e);
      s2 = f == 0.f ? 0.f : f * (s2 + d * s1);  // d s1 may be infinite where f is 0
      s1 = f * s1;
    }
    m = mn;
  }
}

// over the warp, NaN if one is
__device__ __forceinline__ float warp_max_nan(float v) {
  float y;
  asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(v));
  return y;
}
// The same in pairs, -inf (and what is below it in f32's terms) as -1e37.
template <typename In>
__device__ __forceinline__ void vec_pairs(uint4 u, uint64_t x[8 / sizeof(In)]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  if constexpr (sizeof(In) == 4) {
#pragma unroll
    for (int i = 0; i < 2; i++)
      x[i] = pair(max_nan(__uint_as_float(w[2 * i]), -1e37f), max_nan(__uint_as_float(w[2 * i + 1]), -1e37f));
  } else {
    const __nv_bfloat162 low = __floats2bfloat162_rn(-1e37f, -1e37f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w[i]), low);
      const float2 f = unpack2(*reinterpret_cast<const uint32_t*>(&h));
      x[i] = pair(f.x, f.y);
    }
  }
}

// One of them.
template <typename In>
__device__ __forceinline__ float vec_value(uint4 u, int q) {
  constexpr int PER = 4 / sizeof(In);  // of a word
  const uint32_t a = q & PER ? u.y : u.x, b = q & PER ? u.w : u.z, w = q & 2 * PER ? b : a;
  if constexpr (sizeof(In) == 4) return __uint_as_float(w);
  else return __uint_as_float(q & 1 ? w & 0xFFFF0000u : w << 16);
}

struct LpPlan {
  int nblk;    // blocks of a row
  int rounds;  // of kBlocks blocks each, per warp
  int warps;   // of a row
  float4* sums;     // [rows][warps] m, s1, s2
  uint32_t* maxima; // [rows][nblk] rank of each block's largest value, 0 for a block outside the row
};

// Part w of a row, by one warp; its sums and its blocks' maxima go where out says.
template <typename In, typename Out>
__device__ __forceinline__ void logprobs_part(const IrisLogprobs& a, const LpPlan& plan, int row, int w, Out out) {
  using Sh = LpShape<In>;
  const int lane = threadIdx.x % 32;
  const In* x = (const In*)a.logits + (int64_t)row * a.ld;
  const int off = row_offset(x);
  float m = -INFINITY;                        // the warp's
  uint64_t s1[2] = {0, 0}, s2[2] = {0, 0};    // the lane's, two in each register pair
  constexpr int STEP = LP_LOADS * 32 * Sh::kVec;  // values of a round
  int b = w * plan.rounds * Sh::kBlocks + lane;   // the block whose maximum this lane writes
  int e0 = w * plan.rounds * STEP - off;
  const bool keeps = a.top_k && lane < Sh::kBlocks;
  for (int r = 0; r < plan.rounds; r++, b += Sh::kBlocks, e0 += STEP) {
    if (e0 >= a.vocab) {  // blocks are counted for the row that begins furthest from a 16-byte boundary
      if (keeps && b < plan.nblk) out.maximum(row, b, 0u);
      continue;
    }
    uint4 u[LP_LOADS];
    if (e0 >= 0 && e0 + STEP <= a.vocab) {
      const uint4* p = reinterpret_cast<const uint4*>(x + e0) + lane;
#pragma unroll
      for (int j = 0; j < LP_LOADS; j++) u[j] = __ldg(p + j * 32);
    } else {
#pragma unroll
      for (int j = 0; j < LP_LOADS; j++) u[j] = row_vec(x, e0 + (j * 32 + lane) * Sh::kVec, a.vocab);
    }
    float best = 0.f, now = m;
#pragma unroll
    for (int i = 0; i < Sh::kBlocks; i++) {
      float cm = vec_max<In>(u[i * Sh::kPer]);
#pragma unroll
      for (int j = 1; j < Sh::kPer; j++) cm = max_nan(cm, vec_max<In>(u[i * Sh::kPer + j]));
      cm = warp_max_nan(cm);
      if (lane == i) best = cm;
      now = fmaxf(now, cm);
    }
    if (keeps && b < plan.nblk) out.maximum(row, b, e0 + lane * LP_BLOCK < a.vocab ? rank_bits(best) : 0u);
    if (now > m) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
        float2 u1 = halves(s1[i]), u2 = halves(s2[i]);
        float from = m;
        raise(from, u1.x, u2.x, now);
        from = m;
        raise(from, u1.y, u2.y, now);
        s1[i] = pair(u1.x, u1.y), s2[i] = pair(u2.x, u2.y);
      }
      m = now;
    }
    if (m > -1e36f) {
      // 3 instructions a value and its exponential.  Values are held at -1e37 (under any such maximum e^(x - m) is 0
      // there and below), so that one of -inf adds 0 and not 0 inf.
      const uint64_t c = pair(kLog2e, kLog2e), nm = pair(-m, -m);
#pragma unroll
      for (int j = 0; j < LP_LOADS; j++) {
        uint64_t x[Sh::kVec / 2];
        vec_pairs<In>(u[j], x);
#pragma unroll
        for (int i = 0; i < Sh::kVec / 2; i++) {
          const uint64_t d = add2(x[i], nm);
          const float2 y = halves(mul2(d, c));
          const uint64_t e = pair(exp2_approx(y.x), exp2_approx(y.y));
          s1[i & 1] = add2(s1[i & 1], e);
          s2[i & 1] = fma2(d, e, s2[i & 1]);
        }
      }
    } else {  // nothing but -inf and NaN so far, or next to the least value
      const float base = m == -INFINITY ? 0.f : m;
      for (int j = 0; j < LP_LOADS; j++) {
        float v[Sh::kVec];
        vec_values<In>(u[j], v);
        for (int i = 0; i < Sh::kVec; i++) {
          const float d = v[i] - base, e = exp2_approx(d * kLog2e);
          s1[0] = add2(s1[0], pair(e, 0.f));
          s2[0] = add2(s2[0], pair(fmaxf(d, -1000.f) * e, 0.f));
        }
      }
    }
  }
  const float2 u1 = halves(add2(s1[0], s1[1])), u2 = halves(add2(s2[0], s2[1]));
  const float t1 = warp_add(u1.x + u1.y), t2 = warp_add(u2.x + u2.y);
  if (lane == 0) out.sum(make_float4(m, t1, t2, 0.f));
}

struct ToWorkspace {
  const LpPlan& plan;
  // parts of all rows in one line: a warp's own number is its place
  __device__ void sum(float4 v) const { plan.sums[blockIdx.x * 8 + threadIdx.x / 32] = v; }
  __device__ void maximum(int64_t row, int b, uint32_t r) const { plan.maxima[row * plan.nblk + b] = r; }
};

template <typename In>
__global__ void __launch_bounds__(256, 4) logprobs_stream_kernel(const __grid_constant__ IrisLogprobs a,
                                                                 const __grid_constant__ LpPlan plan) {
  const uint32_t wid = blockIdx.x * 8 + threadIdx.x / 32;
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const uint32_t row = wid / (uint32_t)plan.warps;
  if (row >= (uint32_t)a.rows) return;
  const int w = (int)(wid - row * plan.warps);
  logprobs_part<In>(a, plan, (int)row, w, ToWorkspace{plan});
}

// The k largest of the places that items(least, f) hands to f (each thread its
// own share of them, the same on every call; all different, none 0; it may leave
// out values under least()), largest first, into best; returns how many there are.  `from`: where it is known that k
// places reach it, else 0.  Without one, or where many reach it (the
// least maximum of a few blocks is not far up), every thread's largest place is
// ranked against 32 of them, and the least of the 32 that k of them reach is such a
// value.  The few places that reach it are put in order by counting.  Only where
// more than LP_LIST do even then, many of the largest in one thread's share, is a
// closer value searched by halving.
constexpr int LP_LIST = 512;
template <int THREADS>
struct TopK {
  uint64_t own[THREADS], list[LP_LIST], best[32], pick[THREADS / 32];
  int reach[THREADS / 32];
  int n;
  unsigned sum;
};

template <int THREADS, typename Items>
__device__ int select_top(TopK<THREADS>& s, int k, uint64_t from, Items items) {
  constexpr int W = THREADS / 32;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  for (int step = from ? 0 : 1;; step++) {  // 0: what is known, 1: with the ranking, then: closer
    if (step == 1) {
      uint64_t own = 0;
      items([&]() { return own ? rank_value((uint32_t)(own >> 32)) : -INFINITY; }, [&](uint64_t p) { own = p > own ? p : own; });
      s.own[tid] = own;
      __syncthreads();
      uint64_t o[W], pick = 1;  // 1: fewer than k threads have a place
      int reach = THREADS + 1;
#pragma unroll
      for (int i = 0; i < W; i++) o[i] = s.own[i * 32 + lane];
#pragma unroll
      for (int j = 0; j < 32 / W; j++) {
        const uint64_t c = s.own[(warp * (32 / W) + j) * W];
        int n = 0;
#pragma unroll
        for (int i = 0; i < W; i++) n += o[i] >= c;
        n = __reduce_add_sync(0xffffffffu, n);
        if (c && n >= k && n < reach) pick = c, reach = n;
      }
      if (lane == 0) s.pick[warp] = pick, s.reach[warp] = reach;
      __syncthreads();
      uint64_t ranked = s.pick[0];
      reach = s.reach[0];
#pragma unroll
      for (int i = 1; i < W; i++)
        if (s.reach[i] < reach) ranked = s.pick[i], reach = s.reach[i];
      from = ranked > from ? ranked : from;
    }
    if (tid == 0) s.n = 0;
    __syncthreads();
    const float least = from > 1 ? rank_value((uint32_t)(from >> 32)) : -INFINITY;
    items([&]() { return least; }, [&](uint64_t p) {
      if (p >= from) {
        const int at = atomicAdd(&s.n, 1);
        if (at < LP_LIST) s.list[at] = p;
      }
    });
    __syncthreads();
    if (s.n <= (step == 0 ? LP_LIST / 2 : LP_LIST)) break;  // (putting n in order takes n^2 steps)
    if (step == 0) continue;
    uint64_t hi = 0xFF800002ull << 32;  // over all places
    while (true) {
      const uint64_t mid = from + (hi - from) / 2;
      if (tid == 0) s.sum = 0;
      __syncthreads();
      unsigned c = 0;
      items([&]() { return least; }, [&](uint64_t p) { c += p >= mid; });
      c = __reduce_add_sync(0xffffffffu, c);
      if (tid % 32 == 0) atomicAdd(&s.sum, c);
      __syncthreads();
      c = s.sum;
      __syncthreads();
      if (c < (unsigned)k) {
        hi = mid;
      } else {
        from = mid;
        if (c <= LP_LIST) break;
      }
    }
  }
  const int n = s.n;
  for (int c = tid; c < n; c += THREADS) {
    const uint64_t p = s.list[c];
    int ahead = 0;
#pragma unroll 8
    for (int j = 0; j < n; j++) ahead += s.list[j] > p;
    if (ahead < k) s.best[ahead] = p;
  }
  __syncthreads();
  return min(n, k);
}

// The parts' sums of a row joined, the outputs, the alternatives, by THREADS
// threads of a block (the others have left it).  Bound by latency: a chain of
// three reads and some twenty barriers.
template <typename In, int THREADS>
__device__ __forceinline__ void logprobs_row(const IrisLogprobs& a, const LpPlan& plan, int64_t row, const float4* sums,
                                             const uint32_t* maxima) {
  using Sh = LpShape<In>;
  constexpr int WARPS = THREADS / 32, HELD = 5;
  __shared__ TopK<THREADS> top;
  __shared__ uint64_t blocks[32];
  __shared__ float red[3][WARPS];
  const int tid = threadIdx.x;
  const In* x = (const In*)a.logits + row * a.ld;
  float given = 0.f;
  bool has = false;
  if (tid == 0 && a.logprob) {
    const int t = a.targets[row];
    has = t >= 0 && t < a.vocab;
    if (has) {
      if constexpr (sizeof(In) == 4) given = x[t];
      else given = __bfloat162float(x[t]);
    }
  }
  uint32_t held[HELD];  // the first maxima, read with the sums
#pragma unroll
  for (int i = 0; i < HELD; i++) held[i] = a.top_k && tid + i * THREADS < plan.nblk ? maxima[tid + i * THREADS] : 0u;
  float m = -INFINITY, s1 = 0.f, s2 = 0.f;
  for (int w = tid; w < plan.warps; w += THREADS) {
    float4 v = sums[w];
    const float mn = fmaxf(m, v.x);
    raise(m, s1, s2, mn);
    raise(v.x, v.y, v.z, mn);
    s1 += v.y;
    s2 += v.z;
  }
  float mm = warp_max(m);
  if (tid % 32 == 0) red[0][tid / 32] = mm;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < WARPS; w++) mm = fmaxf(mm, red[0][w]);
  raise(m, s1, s2, mm);
  s1 = warp_add(s1), s2 = warp_add(s2);
  if (tid % 32 == 0) red[1][tid / 32] = s1, red[2][tid / 32] = s2;
  __syncthreads();
  s1 = s2 = 0.f;
#pragma unroll
  for (int w = 0; w < WARPS; w++) s1 += red[1][w], s2 += red[2][w];
  const float log_s1 = logf(s1);
  auto log_softmax = [&](float x) { return s1 == 0.f ? -INFINITY : (x - m) - log_s1; };  // no sum: -inf alone
  if (tid == 0) {
    if (a.logprob) a.logprob[row] = has ? log_softmax(given) : 0.f;
    if (a.entropy) a.entropy[row] = s1 == 0.f ? 0.f : log_s1 - s2 / s1;
  }
  if (!a.top_k) return;
  const int nb = select_top(top, a.top_k, 0, [&](auto, auto f) {
#pragma unroll
    for (int i = 0; i < HELD; i++)
      if (held[i]) f(place(held[i], tid + i * THREADS));
    for (int b = tid + HELD * THREADS; b < plan.nblk; b += THREADS) {
      const uint32_t r = maxima[b];
      if (r) f(place(r, b));
    }
  });
  if (tid < nb) blocks[tid] = top.best[tid];
  __syncthreads();
  // k blocks: each holds a value no less than the k-th maximum
  const uint64_t from = nb == a.top_k ? blocks[nb - 1] >> 32 << 32 : 0;
  const int off = row_offset(x);
  select_top(top, a.top_k, from, [&](auto least, auto f) {
    constexpr int VPB = LP_BLOCK / Sh::kVec, FLY = 5;
    for (int j0 = tid; j0 < nb * VPB; j0 += FLY * THREADS) {
      uint4 u[FLY];
      int e[FLY];
#pragma unroll
      for (int i = 0; i < FLY; i++) {
        const int j = j0 + i * THREADS;
        e[i] = j < nb * VPB ? (int)~(uint32_t)blocks[j / VPB] * LP_BLOCK - off + j % VPB * Sh::kVec : a.vocab;
        u[i] = row_vec(x, e[i], a.vocab);
      }
#pragma unroll
      for (int i = 0; i < FLY; i++) {
        // which values are not under least (a NaN is under nothing): few, so that they are taken one by one
        const float lo = least();
        float v[Sh::kVec];
        vec_values<In>(u[i], v);
        uint32_t reach = 0;
#pragma unroll
        for (int q = 0; q < Sh::kVec; q++) reach |= v[q] < lo ? 0u : 1u << q;
        for (; reach; reach &= reach - 1) {
          const int q = __ffs(reach) - 1, id = e[i] + q;
          if ((uint32_t)id < (uint32_t)a.vocab) f(place(rank_bits(vec_value<In>(u[i], q)), (uint32_t)id));
        }
      }
    }
  });
  if (tid < a.top_k) {
    const uint64_t p = top.best[tid];
    if (a.top_ids) a.top_ids[row * a.top_k + tid] = (int)~(uint32_t)p;
    if (a.top_logprobs) a.top_logprobs[row * a.top_k + tid] = log_softmax(rank_value((uint32_t)(p >> 32)));
  }
}

template <typename In, int THREADS>
__global__ void __launch_bounds__(THREADS) logprobs_finish_kernel(const __grid_constant__ IrisLogprobs a,
                                                                  const __grid_constant__ LpPlan plan) {
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  const int64_t row = blockIdx.x;
  logprobs_row<In, THREADS>(a, plan, row, plan.sums + row * plan.warps, plan.maxima + row * plan.nblk);
}

// Few rows: both in one launch, a cluster per row, whose barrier stands between;
// the parts leave their sums and maxima in the first block's shared memory.
struct ToFirstBlock {
  float4* sums;
  uint32_t* maxima;
  int w;
  __device__ void sum(float4 v) const { *iris::cluster_map(sums + w, 0) = v; }
  __device__ void maximum(int64_t, int b, uint32_t r) const { *iris::cluster_map(maxima + b, 0) = r; }
};

template <typename In>
__global__ void __launch_bounds__(512, 2) logprobs_cluster_kernel(const __grid_constant__ IrisLogprobs a,
                                                                  const __grid_constant__ LpPlan plan) {
  extern __shared__ __align__(128) uint8_t smem[];
  const int row = blockIdx.x / LP_CLUSTER, rank = blockIdx.x % LP_CLUSTER;
  const int w = rank * (blockDim.x / 32) + threadIdx.x / 32;
  float4* sums = reinterpret_cast<float4*>(smem);
  uint32_t* maxima = reinterpret_cast<uint32_t*>(sums + plan.warps);
  iris::cluster_sync();  // the first block is there
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  if (w < plan.warps) logprobs_part<In>(a, plan, row, w, ToFirstBlock{sums, maxima, w});
  __syncwarp();
  iris::cluster_sync();
  if (rank == 0 && threadIdx.x < 256) logprobs_row<In, 256>(a, plan, row, sums, maxima);
}

}  // namespace

// ------------------------------------------------------------------ launches
extern "C" cudaError_t iris_launch_rope_append(IrisRopeAppend* a, int f32, int num_sms, cudaStream_t stream) {
  a->div = iris_paged_div(a->cache.page_size);
  const int groups = ROPE_THREADS / (a->cache.head_dim / 8);
  const int slices = (a->heads + 2 * a->cache.kv_heads + groups - 1) / groups;  // with a head per group of lanes
  // few tokens: a block per slice, so that they run side by side; else ROPE_HEADS slices a block, the most the kernel takes
  const bool few = (int64_t)a->tokens * slices * ROPE_THREADS <= 1024 * num_sms;
  const dim3 grid(a->tokens, few ? slices : (slices + ROPE_HEADS - 1) / ROPE_HEADS);
  auto go = [&](auto kernel) { return iris::launch_overlapped(kernel, grid, dim3(ROPE_THREADS), 0, stream, *a); };
  if (f32) {
    if (a->cache.head_dim == 64) return go(rope_append_kernel<float, 64>);
    if (a->cache.head_dim == 128) return go(rope_append_kernel<float, 128>);
    return go(rope_append_kernel<float, 256>);
  }
  if (a->cache.head_dim == 64) return go(rope_append_kernel<__nv_bfloat16, 64>);
  if (a->cache.head_dim == 128) return go(rope_append_kernel<__nv_bfloat16, 128>);
  return go(rope_append_kernel<__nv_bfloat16, 256>);
}

extern "C" cudaError_t iris_launch_rope_append8(IrisRopeAppend* a, int f32, int num_sms, cudaStream_t stream) {
  a->div = iris_paged_div(a->cache.page_size);
  a->exp.div = iris_paged_div(a->exp.block);
  Append8Plan plan;
  plan.items = (2 * a->cache.kv_heads + APPEND8_WARPS - 1) / APPEND8_WARPS;
  const bool many = a->tokens > 8 * num_sms;
  plan.per = many && a->exp.block >= APPEND8_TOKENS ? APPEND8_TOKENS : 1;
  const int64_t kv = ((int64_t)a->tokens + plan.per - 1) / plan.per * plan.items;
  const int groups = ROPE_THREADS / (a->cache.head_dim / 8), all = (a->heads + groups - 1) / groups;
  // as for iris_launch_rope_append
  const bool few = (int64_t)a->tokens * all * ROPE_THREADS <= 1024 * num_sms;
  plan.slices = few ? all : (all + ROPE_HEADS - 1) / ROPE_HEADS;
  constexpr int subs = APPEND8_THREADS / ROPE_THREADS;
  const int64_t blocks = kv + ((int64_t)a->tokens + subs - 1) / subs * plan.slices;
  if (blocks > 0x7FFFFFFF) return cudaErrorInvalidValue;
  plan.kv_blocks = (int)kv;
  auto go = [&](auto kernel) {
    return iris::launch_overlapped(kernel, dim3((unsigned)blocks), dim3(APPEND8_THREADS), 0, stream, *a, plan);
  };
  auto of = [&](auto in, auto is_many) {
    using In = decltype(in);
    constexpr bool M = decltype(is_many)::value;
    if (a->cache.head_dim == 64) return go(rope_append8_kernel<In, 64, M>);
    if (a->cache.head_dim == 128) return go(rope_append8_kernel<In, 128, M>);
    return go(rope_append8_kernel<In, 256, M>);
  };
  if (f32) return many ? of(0.f, std::true_type()) : of(0.f, std::false_type());
  return many ? of(__nv_bfloat16(), std::true_type()) : of(__nv_bfloat16(), std::false_type());
}

// CTAs of an attention launch: as many as the device holds at once, no more than the tables have room for tiles
static int paged_ctas(const iris_gpu_kv_cache_t* c, int heads, int64_t rows, int all) {
  const int64_t room = iris_paged_tiles(iris_paged_len(c, 0x7FFFFFFF)) + IRIS_PAGED_EXTRA;
  const int64_t most = rows * iris_paged_units(c, heads);
  return most >= all || most * room >= all ? all : (int)(most * room);
}

constexpr int CLUSTER_TILES = 4;

template <typename E, int HD, int MH>
struct PagedLaunch {
  using Sh = PagedShape<E, HD, MH>;
  using Runs = RunShape<E, HD>;
  static size_t ws_bytes(int num_sms) {
    const int ctas = num_sms * Sh::kCtas, runs = num_sms * Runs::kCtas;
    const size_t one = paged_slots_at(ctas) + (size_t)2 * ctas * Sh::kSlot;
    const size_t several = paged_slots_at(runs) + (size_t)2 * runs * Runs::kSlot;
    return (one > several ? one : several) * sizeof(float);
  }
  static cudaError_t init() {
    cudaError_t e = cudaFuncSetAttribute(paged_runs_kernel<E, HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, Runs::kSmem);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(paged_attention_kernel<E, HD, MH, false>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                               Sh::kSmem);
    if (e != cudaSuccess) return e;
    return cudaFuncSetAttribute(paged_attention_kernel<E, HD, MH, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kSmem);
  }
  static cudaError_t launch(const IrisPagedAttention* a, int num_sms, cudaStream_t stream, int* launches) {
    // few rows: a block, or a cluster of up to 8, on each unit, all on the device at once (clusters of 4 and 8 do not fill
    // every SM: 72 of 4, 288 blocks of 296, took 11.7 us with 512 keys, 72 of 2 7.5), where the tables have room for no
    // more than CLUSTER_TILES tiles a block, or where the blocks are more than half of what the device holds, up to twice
    // that: equal shares of all tiles gain the less the fewer CTAs would be idle without.  On the device, two kernels ->
    // one, 32 heads on 8 of 128: a row of 512 keys 5.9 us both, 8 rows of 512 9.2 -> 7.2, a row of 2048 (4 tiles a block)
    // 8.0 -> 8.4, of 4096 (8 tiles) 9.4 -> 11.6, 37 rows of 200 10.3 -> 8.3, of 512 (8 tiles, every slot taken) 15.6 ->
    // 12.9, of 1 to 512 13.0 -> 12.0, 6 rows of 1200 (5 tiles) 11.2 -> 10.0; the caller is spared a launch, 3 us
    const int64_t units = (int64_t)a->rows * iris_paged_units(&a->cache, a->heads);
    const int room = iris_paged_tiles(iris_paged_len(&a->cache, 0x7FFFFFFF));
    unsigned parts = 8;
    const int64_t slots = (int64_t)num_sms * Sh::kCtas;
    while (parts > 1 && units * parts > (parts > 2 ? slots * 7 / 8 : slots)) parts /= 2;
    const int64_t tiles = 2 * CLUSTER_TILES * units * parts / slots + 1;  // 2 CLUSTER_TILES with every slot taken
    if (units * parts <= slots && room <= (tiles < CLUSTER_TILES ? CLUSTER_TILES : tiles) * parts) {
      *launches = 1;
      return iris::launch_cluster_overlapped(paged_attention_kernel<E, HD, MH, true>, dim3((unsigned)units * parts),
                                             dim3(Sh::kThreads), Sh::kSmem, parts, stream, *a);
    }
    // four times as many rows as sequences: runs of rows.  On the device, 32 heads on 8 of 128, rows by themselves -> runs:
    // a prompt of 128 15.3 -> 15.8 us, 512 83 -> 31, 2048 934 -> 196, 8192 13.7 -> 2.6 ms; 64 tokens behind 32704 855 ->
    // 188; 4 behind 4092 in 8 sequences 77 -> 38, 4 behind 1020 in 64 164 -> 65.  Below, 2 behind 4094 in 8 45 -> 36, 2
    // behind 1022 in 64 94 -> 62, but 8 heads on 2 of 256 51 -> 56 and 64 single tokens at 1023 beside a prompt of 128 56 ->
    // 93.  The host sees counts only, so that the rule also loses: 64 single tokens beside a prompt of 256 67 -> 98, of 384
    // 89 -> 103 (of 448 101 -> 103, of 512 116 -> 113, of 1024 295 -> 156); 2048 rows of 4 sequences in random order, no
    // runs in them, 303 -> 553.
    if (a->seq && a->rows >= 4 * (int64_t)a->cache.num_seqs) {
      const int ctas = paged_ctas(&a->cache, a->heads, a->rows, num_sms * Runs::kCtas);
      const cudaError_t e = iris::launch_overlapped(paged_runs_kernel<E, HD>, dim3(ctas), dim3(Runs::kThreads), Runs::kSmem, stream, *a);
      *launches = 1;
      if (e != cudaSuccess || ctas == 1) return e;
      *launches = 2;
      return iris::launch_overlapped(paged_runs_join_kernel<HD>, dim3(ctas - 1, 2), dim3(RUN_JOIN_THREADS), 0, stream, *a, ctas);
    }
    const int ctas = paged_ctas(&a->cache, a->heads, a->rows, num_sms * Sh::kCtas);
    cudaError_t e = iris::launch_overlapped(paged_attention_kernel<E, HD, MH, false>, dim3(ctas), dim3(Sh::kThreads), Sh::kSmem,
                                            stream, *a);
    *launches = 1;
    if (e != cudaSuccess || ctas == 1) return e;
    const int group = a->heads / a->cache.kv_heads;
    *launches = 2;
    const int h = group < MH ? group : MH, fit = JOIN_THREADS / (HD / 4);
    if (units * 8 <= ctas)
      return iris::launch_overlapped(paged_join_kernel<HD, MH, true>, dim3((unsigned)units, h), dim3(JOIN_THREADS), 0, stream, *a,
                                     ctas, 1);
    const int per_block = h < fit ? h : fit;
    return iris::launch_overlapped(paged_join_kernel<HD, MH, false>, dim3(ctas - 1, (h + per_block - 1) / per_block),
                                   dim3(JOIN_THREADS), 0, stream, *a, ctas, per_block);
  }
};

// f(PagedLaunch) of the variant for this cache and group of query heads
template <typename E, typename F>
static auto paged_variant(const iris_gpu_kv_cache_t* c, int heads, F f) {
  const bool wide = iris_paged_heads(heads / c->kv_heads) == 16;
  if (c->head_dim == 64) return wide ? f(PagedLaunch<E, 64, 16>()) : f(PagedLaunch<E, 64, 8>());
  if (c->head_dim == 128) return wide ? f(PagedLaunch<E, 128, 16>()) : f(PagedLaunch<E, 128, 8>());
  return wide ? f(PagedLaunch<E, 256, 16>()) : f(PagedLaunch<E, 256, 8>());
}

extern "C" size_t iris_paged_attention_ws_bytes(const iris_gpu_kv_cache_t* cache, int heads, int num_sms) {
  return paged_variant<__nv_bfloat16>(cache, heads, [&](auto v) { return v.ws_bytes(num_sms); });
}

extern "C" cudaError_t iris_launch_paged_attention(IrisPagedAttention* a, int num_sms, cudaStream_t stream, int* launches) {
  a->div = iris_paged_div(a->cache.page_size);
  return paged_variant<__nv_bfloat16>(&a->cache, a->heads, [&](auto v) { return v.launch(a, num_sms, stream, launches); });
}

extern "C" size_t iris_paged_attention8_ws_bytes(const iris_gpu_kv_cache_t* cache, int heads, int num_sms) {
  return paged_variant<e4m3>(cache, heads, [&](auto v) { return v.ws_bytes(num_sms); });
}

extern "C" cudaError_t iris_launch_paged_attention8(IrisPagedAttention* a, int num_sms, cudaStream_t stream, int* launches) {
  a->div = iris_paged_div(a->cache.page_size);
  a->exp.div = iris_paged_div(a->exp.block);
  return paged_variant<e4m3>(&a->cache, a->heads, [&](auto v) { return v.launch(a, num_sms, stream, launches); });
}

// dynamic shared memory limits, once per device, so that launches may be captured
extern "C" cudaError_t iris_lm_init(void) {
  iris_gpu_kv_cache_t c = {};
  c.kv_heads = 1;
  for (int head_dim : {64, 128, 256})
    for (int heads : {8, 16}) {
      c.head_dim = head_dim;
      cudaError_t e = paged_variant<__nv_bfloat16>(&c, heads, [](auto v) { return v.init(); });
      if (e == cudaSuccess) e = paged_variant<e4m3>(&c, heads, [](auto v) { return v.init(); });
      if (e != cudaSuccess) return e;
    }
  return cudaSuccess;
}

static int lp_blocks(int vocab) { return (int)(((int64_t)vocab + 7 + LP_BLOCK - 1) / LP_BLOCK); }  // 7: row_offset at most

static size_t lp_align(size_t n) { return (n + 15) & ~(size_t)15; }

extern "C" size_t iris_logprobs_ws_bytes(int rows, int vocab) {
  const size_t n = (size_t)lp_blocks(vocab);  // warps of a row: at most a block each
  return 16 + (size_t)rows * n * sizeof(float4) + lp_align((size_t)rows * n * sizeof(uint32_t));
}

template <typename In>
static cudaError_t launch_logprobs(const IrisLogprobs* a, int num_sms, cudaStream_t stream, int* launches) {
  LpPlan plan;
  plan.nblk = lp_blocks(a->vocab);
  constexpr int K = LpShape<In>::kBlocks;
  const int all = (plan.nblk + K - 1) / K;  // rounds of loads in a row
  plan.sums = (float4*)a->ws;
  // few rows: a cluster of blocks of 16 warps on each, all of them on the device at once (clusters of 8 do not fill every
  // SM: 32 of 37).  One launch instead of two: 2.5 us less of the caller's time.  On the device, bf16 rows of 151936 with
  // 20 alternatives, one launch and two: 1 row 7.9 and 7.6 us, 16 9.0 and 8.5, 32 10.4 and 9.3, 36 12.3 and 9.4
  const int64_t blocks = (int64_t)a->rows * LP_CLUSTER;
  if (blocks <= 2 * num_sms * 7 / 8 && plan.nblk <= LP_CLUSTER_BLOCKS) {
    plan.rounds = (all + 16 * LP_CLUSTER - 1) / (16 * LP_CLUSTER);
    plan.warps = (all + plan.rounds - 1) / plan.rounds;
    *launches = 1;
    return iris::launch_cluster_overlapped(logprobs_cluster_kernel<In>, dim3((unsigned)blocks), dim3(512),
                                           plan.warps * sizeof(float4) + plan.nblk * sizeof(uint32_t), LP_CLUSTER, stream, *a,
                                           plan);
  }
  // a warp begins and ends with some 100 instructions, as many as 10 values of each lane, and in a second round of loads
  // an SM's warps are out of step: two rounds, as long as every SM is left three times the 32 warps that it holds
  // (512 f32 rows of 151936: 56.2 us with 1, 55.6 with 2, 56.9 with 3, 62.6 with 8; 2047 bf16 rows of 50021: 56.2,
  // 54.1, 53.7, 56.8)
  plan.rounds = all * (int64_t)a->rows >= (int64_t)num_sms * 32 * 3 * 2 ? 2 : 1;
  plan.warps = (all + plan.rounds - 1) / plan.rounds;
  plan.maxima = (uint32_t*)(plan.sums + (size_t)a->rows * plan.warps);
  const int64_t ctas = ((int64_t)a->rows * plan.warps + 7) / 8;
  *launches = 2;
  cudaError_t e = iris::launch_overlapped(logprobs_stream_kernel<In>, dim3((unsigned)ctas), dim3(256), 0, stream, *a, plan);
  if (e != cudaSuccess) return e;
  // Rows that are all on the device at once (4 blocks an SM) take 256 threads each.  128 -> 256: one row of 151936 and 20
  // alternatives (in the cluster) 8.2 -> 7.9 us, 192 f32 rows of 65537 with 8 14.9 -> 13.0, with 32 21.1 -> 15.3, 512 f32
  // rows of 151936 with 5 54.5 -> 53.5; with 512 one row takes 8.6 and 100 f32 rows of 151936 with 8 14.8 for 13.6
  if (a->rows <= 4 * num_sms)
    return iris::launch_overlapped(logprobs_finish_kernel<In, 256>, dim3(a->rows), dim3(256), 0, stream, *a, plan);
  // (9 blocks of 128 an SM) 128 -> 64: 2047 bf16 rows of 50021 with 8 53.3 -> 51.1, with 32 61.3 -> 63.4, 4000 of 32000
  // with 8 70.9 -> 64.2, 1300 of 32000 with 8 26.0 for 27.8
  if (a->rows <= 9 * num_sms)
    return iris::launch_overlapped(logprobs_finish_kernel<In, 128>, dim3(a->rows), dim3(128), 0, stream, *a, plan);
  return iris::launch_overlapped(logprobs_finish_kernel<In, 64>, dim3(a->rows), dim3(64), 0, stream, *a, plan);
}

extern "C" cudaError_t iris_launch_logprobs(const IrisLogprobs* a, int f32, int num_sms, cudaStream_t stream,
                                            int* launches) {
  return f32 ? launch_logprobs<float>(a, num_sms, stream, launches)
             : launch_logprobs<__nv_bfloat16>(a, num_sms, stream, launches);
}
