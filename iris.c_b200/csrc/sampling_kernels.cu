// The next token of each row of logits: temperature, min-p, top-k, top-p, and a
// random number that the caller gives.
#include "iris_kernels.h"
#include "lm_device.cuh"
#include "ptx.cuh"

#include <cuda_bf16.h>
#include <float.h>
#include <math.h>
#include <stdint.h>

namespace {

// A row's tokens stand in line, the largest logit first, equal ones by id.  With m
// the largest and t the temperature a token weighs w = e^((x - m) / t).  Each
// setting keeps a first part of the line (min-p: while w >= min_p; top-k: k tokens;
// top-p: until their sum reaches top_p of what the other two keep), and the random
// number u takes the token at which the sum of weights passes u of what is kept.  So
// all of it is: where in the line does a count, or a sum, cross a number?
//
// The row is read once, by a cluster of blocks that hold it in shared memory.
// With top-k of up to SMP_TOP, in shares of up to SMP_SHARE a block, the tokens above
// a bound (which k of the threads' own largest reach) are few, and so they are where
// min-p leaves few: one block puts them in order and has the answer.  Else a histogram over the distance from m, in parts of
// SMP_SPAN / SMP_BINS of t, says to 2^-14 (large vocabularies: less closely) how the
// sum grows along the line (each value adds its weight relative to its bin's, a whole
// number of 16 bits, so that no order of additions shows); a pass over the row adds up exactly what
// stands ahead of the bins in which the number is crossed and collects their
// tokens, some hundreds, which one block puts in order.  Where they are too many
// (equal logits, high temperatures) the bins are cut further, each time into 16,
// with exact sums, until few are left, or tokens of one value, of which the id decides.
// Weights and sums are 64-bit: a token is taken by where a sum of 100000 weights
// ends, and with 32 bits one row in a hundred would take its neighbour.
// Rows of 151936 f32: one with the usual settings 9.3 us, greedy 4.5, top-p alone 30;
// 512 with the usual settings 167 us, top-p alone 595 (bf16 381), of which 49 for the
// bytes: barriers of the cluster for few rows; for many, latency: 16 warps an SM (registers)
// with 64-bit weights and additions in shared memory, 41 % of the issue slots.
constexpr int SMP_THREADS = 256, SMP_WARPS = SMP_THREADS / 32, SMP_PARTS = 8;
constexpr int SMP_LIST = 1024;  // tokens put in order
constexpr int SMP_TOP = 512;    // largest top-k whose tokens are looked for through a bound, and the largest share of a block in it:
constexpr int SMP_SHARE = 200;  // some 390 tokens reach the 200th of 256 threads' largest, 1570 the last one, more than the lists hold
                                // (512 bf16 rows of 32000, top-k 200 37 us, 256 120 through a bound and then without, 95 without)
constexpr int SMP_BINS = 2048;
constexpr float SMP_SPAN = 24.f;      // (m - x) / t that the bins cover; the last one holds all that is below
constexpr int SMP_CUT = 16, SMP_CUTTERS = 64;  // bins of a closer look, threads that fill bins of their own
constexpr int SMP_SORT = 1024;  // places of the sort by value
constexpr int SMP_OWN = 128;    // vectors of a warp's list
constexpr int SMP_MINE = SMP_BINS / SMP_THREADS, SMP_EACH = SMP_LIST / SMP_THREADS;  // of a thread
static_assert(SMP_MINE % 4 == 0 && SMP_SORT == SMP_LIST, "shares of a thread");

struct SmpSums {  // of the closer bins, from each block of the cluster
  double mass[SMP_PARTS][SMP_CUT];
  uint32_t count[SMP_PARTS][SMP_CUT];
};

struct SmpFound {
  uint64_t place;
  double mass;     // of the line up to and with it
  uint32_t count;
};

struct SmpExact {  // of a block, or a warp of it
  double all, ahead[2];          // sums of all tokens, of those ahead of either window
  uint32_t n_all, n_ahead[2], n[2];  // tokens: all, ahead, in the window
};

struct SmpShared {
  SmpSums next[2];             // in turn, so that one round's may be read while the next one's come
  SmpExact exact[2][SMP_PARTS];
  uint2 two[2][SMP_PARTS];     // two numbers from each block
  SmpExact parts[SMP_WARPS];   // of a block's warps
  double scan[SMP_WARPS];
  float fscan[SMP_WARPS];
  uint32_t iscan[SMP_WARPS];
  double root[64];             // 2^(i / 64)
  SmpFound found;
  uint32_t n[2], lo, hi;
};

// shared memory besides the row: the histogram, in whose place tokens are put in order; lists of the warps, places of the sort or
// sums along a line; and two lists, in whose place the closer bins stand
constexpr int SMP_HIST = SMP_BINS * 4, SMP_ALONG = SMP_BINS * 4;
constexpr int SMP_TAIL = 2 * SMP_LIST * 8;
constexpr int SMP_WORK = SMP_HIST + SMP_ALONG + SMP_TAIL;
static_assert(SMP_TAIL >= SMP_CUT * SMP_CUTTERS * (8 + 4) && SMP_ALONG >= SMP_SORT * 4 &&
                  SMP_ALONG >= SMP_WARPS * SMP_OWN * 4 && SMP_ALONG >= SMP_LIST * 8 && SMP_HIST >= SMP_LIST * 8,
              "the bins and lists fit");

struct SmpWindow {  // part of the line: ranks lo .. hi, `count` tokens, with sums over what stands ahead of it
  uint32_t lo, hi;
  double mass;
  uint32_t ahead, count;
  uint32_t before;  // tokens of the part in the blocks ahead of this one
};

enum SmpKind { SMP_COUNT, SMP_REACH, SMP_PASS };  // count >= n, sum >= number, sum > number

template <typename In, bool HELD>
struct SmpRow {
  static constexpr int VEC = 16 / sizeof(In);
  const IrisSample& a;
  SmpShared& sh;
  uint8_t* smem;
  const In* x;
  int tid, part, parts, off, v0, nv;
  float m, floor_, lowest;   // lowest: what lies under it weighs nothing, e^-600 or less
  double top, inv_t, rate;   // rate: 64 log2(e) / t
  float inv_bin;
  float unit;                // of the histogram's weights, so that a block's tokens in one bin stay within 32 bits
  bool plain;                // no min-p, and a temperature with which -inf weighs nothing by itself
  float near_;               // relative error of the sums along the bins, with room to spare: half a unit of rounding, 2^-17 for
                             // distances and bins' weights in 32 bits, 2^-20 for sums in 32 bits
  uint32_t turn = 0;

  __device__ SmpRow(const IrisSample& a, SmpShared& sh, uint8_t* smem) : a(a), sh(sh), smem(smem) {
    tid = threadIdx.x;
    parts = a.parts;
    part = blockIdx.x % parts;
    x = (const In*)a.logits + (int64_t)(blockIdx.x / parts) * a.ld;
    off = row_offset(x);
    const int all = (int)(((int64_t)a.vocab + off + VEC - 1) / VEC), per = (all + parts - 1) / parts;
    v0 = part * per;
    nv = max(0, min(per, all - v0));
    unit = 65536.f;
    while (unit * ((float)per * VEC) > 4.2e9f) unit *= 0.5f;
    near_ = 1.f / 32768 + 1.f / unit;
  }
  __device__ uint8_t* work() const { return smem + (HELD ? a.held_bytes : 0); }
  __device__ uint32_t* hist() const { return reinterpret_cast<uint32_t*>(work()); }
  __device__ uint32_t* along() const { return reinterpret_cast<uint32_t*>(work() + SMP_HIST); }
  // the tokens that the blocks have found, each in a part of its own of the first one's lists
  __device__ uint64_t* list(int i = 0) const { return reinterpret_cast<uint64_t*>(work() + SMP_HIST + SMP_ALONG) + i * SMP_LIST; }
  __device__ int quota() const { return SMP_LIST / parts; }
  // by the first block, behind the histogram: the tokens in order, and sums along them
  __device__ uint64_t* ordered() const { return reinterpret_cast<uint64_t*>(hist()); }
  __device__ double* line() const { return reinterpret_cast<double*>(along()); }
  __device__ double* cut_mass() const { return reinterpret_cast<double*>(list()); }
  __device__ uint32_t* cut_count() const { return reinterpret_cast<uint32_t*>(cut_mass() + SMP_CUT * SMP_CUTTERS); }

  __device__ void all_sync() const {
    __syncwarp();
    if (parts > 1) iris::cluster_sync();
    else __syncthreads();
  }
  template <typename T>
  __device__ T* at(T* p, int rank) const { return parts > 1 ? iris::cluster_map(p, (uint32_t)rank) : p; }
  // this block's numbers, the same in all threads, to all blocks; those of the blocks after the barrier
  __device__ const uint2* tell(uint32_t v, uint32_t w = 0) {
    uint2* to = sh.two[turn++ & 1];
    if (tid < parts) *at(to + part, tid) = make_uint2(v, w);
    all_sync();
    return to;
  }

  __device__ int first_id(int v) const { return (v0 + v) * VEC - off; }
  __device__ uint4 vec(int v) const {
    if constexpr (HELD) return reinterpret_cast<const uint4*>(smem)[v];
    else return row_vec(x, first_id(v), a.vocab);
  }
  // f(values, id of the first): a vector; values outside the row are -inf
  template <typename F>
  __device__ void vectors(F f, int threads = SMP_THREADS) const {
    for (int v = tid; v < nv; v += threads) {
      float y[VEC];
      vec_values<In>(vec(v), y);
      f(y, first_id(v));
    }
  }
  template <typename F>
  __device__ void each(F f) const {
    vectors([&](const float* y, int id) {
#pragma unroll
      for (int i = 0; i < VEC; i++) f(y[i], id + i);
    });
  }

  // w of y >= floor_, to some 2^-44: 2^(z / 64) with z = 64 log2(e) (y - m) / t as 2^(n >> 6), a root of 2 for n & 63 from
  // a table, and the series of e^r for the rest, |r| <= ln 2 / 128 (Tang, Table-driven implementation of the exponential
  // function, 1989).
  __device__ double weight(float y) const {
    constexpr double c = 0.69314718055994530942 / 64;
    const double z = ((double)fmaxf(y, lowest) - top) * rate;
    const double shifted = z + 0x1.8p52;
    const int n = max(__double2loint(shifted), -64 * 1000);
    const double r = z - (shifted - 0x1.8p52);
    double p = fma(r, c * c * c * c / 24, c * c * c / 6);
    p = fma(r, p, c * c / 2);
    p = fma(r, p, c);
    p = fma(r, p, 1.0) * sh.root[n & 63];
    return __hiloint2double(__double2hiint(p) + (n >> 6) * (1 << 20), __double2loint(p));
  }

  // over the block, the same in all threads
  __device__ uint32_t block_max(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (tid % 32 == 0) sh.iscan[tid / 32] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, sh.iscan[tid % SMP_WARPS]);
    __syncthreads();
    return v;
  }
  __device__ static double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  // sum of what the threads ahead have; *total over the block
  template <typename T>
  __device__ T scan(T v, T* of_warps, T* total) {
    const int lane = tid % 32;
    T incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += y;
    }
    if (lane == 31) of_warps[tid / 32] = incl;
    __syncthreads();
    T w = of_warps[lane % SMP_WARPS];
#pragma unroll
    for (int o = 1; o < SMP_WARPS; o <<= 1) {
      const T y = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += y;
    }
    // (lane i of the first 16: the warps up to and with i)
    const T ahead = __shfl_sync(0xffffffffu, w, (tid / 32 + SMP_WARPS - 1) % SMP_WARPS);
    *total = __shfl_sync(0xffffffffu, w, SMP_WARPS - 1);
    __syncthreads();
    return (tid < 32 ? (T)0 : ahead) + (incl - v);
  }
  __device__ uint32_t scan_count(uint32_t v, uint32_t* total) { return scan(v, sh.iscan, total); }
  __device__ float scan_float(float v, float* total) { return scan(v, sh.fscan, total); }
  // over the blocks' numbers
  __device__ uint32_t most_of(const uint32_t* first_of_pairs) const {
    return __reduce_max_sync(0xffffffffu, tid % 32 < parts ? first_of_pairs[tid % 32 * 2] : 0u);
  }
  __device__ uint32_t least_of(const uint32_t* first_of_pairs) const {
    return __reduce_min_sync(0xffffffffu, tid % 32 < parts ? first_of_pairs[tid % 32 * 2] : 0xffffffffu);
  }

  __device__ bool bounded(int k) const { return k > 0 && k <= min(SMP_TOP, SMP_SHARE * parts); }

  // ---- the row.  From each block its largest value (NaN if there is one), and with top_k = k through a bound a value that its
  // share of k tokens reaches
  __device__ const uint2* load(int k) {
    float best = -INFINITY;
    constexpr int FLY = 20;  // 75 KB of a row in one round
    for (int b = tid; b < nv; b += FLY * SMP_THREADS) {
      uint4 u[FLY];
#pragma unroll
      for (int j = 0; j < FLY; j++) {
        const int v = b + j * SMP_THREADS;
        const uint32_t none = sizeof(In) == 4 ? 0xFF800000u : 0xFF80FF80u;
        u[j] = v < nv ? row_vec(x, first_id(v), a.vocab) : make_uint4(none, none, none, none);
      }
#pragma unroll
      for (int j = 0; j < FLY; j++) {
        const int v = b + j * SMP_THREADS;
        if (HELD && v < nv) reinterpret_cast<uint4*>(smem)[v] = u[j];
        best = max_nan(best, vec_max<In>(u[j]));
      }
    }
    if (tid >= SMP_THREADS - 64) sh.root[tid & 63] = exp2((tid & 63) / 64.0);
    const uint32_t own = rank_bits(best);
    const uint32_t w = __reduce_max_sync(0xffffffffu, own);
    if (tid % 32 == 0) sh.iscan[tid / 32] = w;
    __syncthreads();
    const uint32_t most = __reduce_max_sync(0xffffffffu, sh.iscan[tid % SMP_WARPS]);
    return tell(most, bounded(k) ? reached((k + parts - 1) / parts, own) : 0u);
  }

  // a value that `share` of this block's tokens reach, 0 if it may have fewer; sh.iscan: the warps' largest
  __device__ uint32_t reached(int share, uint32_t own) {
    if (share <= SMP_WARPS / 2) {  // by the warps' largest
      const uint32_t mine = sh.iscan[tid % SMP_WARPS];
      int ahead = 0;
#pragma unroll
      for (int i = 0; i < SMP_WARPS; i++) {
        const uint32_t o = __shfl_sync(0xffffffffu, mine, i);
        ahead += o > mine || (o == mine && i < tid % SMP_WARPS);
      }
      return __reduce_max_sync(0xffffffffu, ahead == share - 1 ? mine : 0u);
    }
    uint32_t reach = 0;  // by the threads', to 20 bits
    for (int bit = 31; bit >= 12; bit--)
      if (__syncthreads_count(own >= (reach | 1u << bit)) >= share) reach |= 1u << bit;
    return reach;
  }

  // ---- the tokens from `from` on into the first block's list; how many each block has
  __device__ const uint2* gather(float from) {
    if (tid == 0) sh.n[0] = 0;
    __syncthreads();
    uint64_t* to = at(list(), 0) + part * quota();
    vectors([&](const float* y, int id) {
      float most = y[0];
#pragma unroll
      for (int i = 1; i < VEC; i++) most = fmaxf(most, y[i]);
      if (most < from || *(volatile uint32_t*)sh.n > quota()) return;  // none, or too many already
#pragma unroll
      for (int i = 0; i < VEC; i++)
        if (y[i] >= from) {
          const uint32_t n = atomicAdd(sh.n, 1);
          if (n < quota()) to[n] = place(rank_bits(y[i]), (uint32_t)(id + i));
        }
    });
    __syncthreads();
    return tell(sh.n[0]);
  }
  // whether the blocks' tokens have all found room
  __device__ bool room(const uint2* n) const {
    return most_of(&n->x) <= quota();
  }

  // ---- by the first block: the blocks' tokens, n in all, in order, largest first, into ordered().  
  __device__ static int tokens_of(const uint2& v, int) { return (int)v.x; }
  __device__ static int tokens_of(const SmpExact& v, int which) { return (int)v.n[which]; }
  template <typename Found>
  __device__ void put_in_order(const Found* from, int n, int which = 0, int blocks = SMP_PARTS) {
    uint64_t* l = ordered();
    // of the tokens of all blocks in a row, this thread's: tid, tid + SMP_THREADS ..
    uint64_t mine[SMP_EACH] = {};
    int begin = 0;
#pragma unroll
    for (int p = 0; p < SMP_PARTS; p++) {
      if (p >= parts || p >= blocks) break;
      const int here = tokens_of(from[p], which);
#pragma unroll
      for (int j = 0; j < SMP_EACH; j++) {
        const int i = tid + j * SMP_THREADS - begin;
        if (i >= 0 && i < here) mine[j] = list(which)[p * quota() + i];
      }
      begin += here;
    }
    if (n <= 128) {
      // how many are ahead of each: n^2 comparisons, 2 to 32 threads a token
      if (tid < n) l[tid] = mine[0];
      __syncthreads();
      int per = 1;
      while (per < 32 && 2 * per * n <= SMP_THREADS) per *= 2;
      const int i = tid / per;
      const uint64_t p = i < n ? l[i] : 0;
      int ahead = 0;
#pragma unroll 4
      for (int j = tid % per; j < n; j += per) ahead += l[j] > p;
      for (int o = per / 2; o; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
      __syncthreads();
      if (i < n && tid % per == 0) l[ahead] = p;
      __syncthreads();
      return;
    }
    // by value into SMP_SORT places, then by comparison within a place
    uint32_t* count = along();
    uint64_t* sorted = list(which);
    uint32_t top_rank = 0, low_rank = 0;
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) {
      count[tid + j * SMP_THREADS] = 0;
      const uint32_t r = (uint32_t)(mine[j] >> 32);
      if (r) top_rank = max(top_rank, r), low_rank = max(low_rank, ~r);
    }
    top_rank = block_max(top_rank);
    low_rank = ~block_max(low_rank);
    const int shift = max(0, 22 - __clz(top_rank - low_rank));
    auto where = [&](uint64_t p) { return (top_rank - (uint32_t)(p >> 32)) >> shift; };
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++)
      if (mine[j]) atomicAdd(count + where(mine[j]), 1u);
    __syncthreads();
    uint32_t own[SMP_EACH], sum = 0, all;
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) own[j] = count[SMP_EACH * tid + j], sum += own[j];
    uint32_t before = scan_count(sum, &all);
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) count[SMP_EACH * tid + j] = before, before += own[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++)
      if (mine[j]) sorted[atomicAdd(count + where(mine[j]), 1u)] = mine[j];  // a place's count becomes its end
    __syncthreads();
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) {
      if (!mine[j]) continue;
      const uint32_t w = where(mine[j]), from_here = w ? count[w - 1] : 0, end = count[w];
      uint32_t ahead = from_here;
      for (uint32_t i = from_here; i < end; i++) ahead += sorted[i] > mine[j];
      l[ahead] = mine[j];
    }
    __syncthreads();
  }
  // number of the n tokens in order for which f(token, weight, sum up to and with it) holds
  template <typename F>
  __device__ uint32_t number(int n, const double w[SMP_EACH], const double c[SMP_EACH], F f) const {
    uint32_t r = 0;
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) {
      if (j * SMP_THREADS >= n) break;
      const int i = tid + j * SMP_THREADS;
      r += __syncthreads_count(i < n && f(i, w[j], c[j]));
    }
    return r;
  }
  // weights of the tokens tid, tid + SMP_THREADS .. of n in order, and the sums up to and with them
  __device__ void sums_of(int n, double w[SMP_EACH], double c[SMP_EACH]) {
    double first = 0.0;
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) {
      w[j] = c[j] = 0.0;
      if (j * SMP_THREADS >= n) continue;
      const int i = tid + j * SMP_THREADS;
      if (i < n) w[j] = weight(rank_value((uint32_t)(ordered()[i] >> 32)));
      double sum;
      c[j] = first + (scan(w[j], sh.scan, &sum) + w[j]);
      first += sum;
    }
  }
  // f(token, sum) by the thread that has token i
  template <typename F>
  __device__ void at_token(uint32_t i, const double c[SMP_EACH], F f) const {
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++)
      if (tid + j * SMP_THREADS == (int)i) f(ordered()[i], c[j]);
  }
  __device__ void answer(int id, double logprob, uint32_t kept) const {
    const int row = blockIdx.x / parts;
    a.ids[row] = id;
    if (a.logprobs) a.logprobs[row] = (float)logprob;
    if (a.kept) a.kept[row] = (int)kept;
  }
  __device__ double logprob(uint64_t p, double mass) const {
    return ((double)rank_value((uint32_t)(p >> 32)) - top) * inv_t - log(mass);
  }

  // ---- all that can be kept is in the list: by the first block
  __device__ void finish(const uint2* from, int n, int k, float p, double u) {
    put_in_order(from, n);
    if (k) n = min(n, k);
    double w[SMP_EACH], c[SMP_EACH];
    sums_of(n, w, c);
    double* sums = line();
#pragma unroll
    for (int j = 0; j < SMP_EACH; j++) sums[tid + j * SMP_THREADS] = c[j];
    __syncthreads();
    const double mass = sums[n - 1];
    uint32_t kept = n;
    if (p < 1.f) {
      const double goal = (double)p * mass;
      kept = max(number(n, w, c, [&](int i, double, double) { return (i ? sums[i - 1] : 0.0) < goal; }), 1u);
    }
    const double m_kept = sums[kept - 1], goal = u * m_kept;
    uint32_t pick = number((int)kept, w, c, [&](int, double, double s) { return s <= goal; });
    if (pick == kept)  // by rounding: the last with a weight (the first one weighs 1)
      pick = number((int)kept, w, c, [&](int, double v, double) { return v > 0.0; }) - 1;
    if (tid == 0) answer((int)~(uint32_t)ordered()[pick], logprob(ordered()[pick], m_kept), kept);
  }

  // ---- how the line grows along the bins: the sum up to and with each bin, to near_ (or the count, a whole number)
  __device__ float distance(float y) const {
    return fminf((plain ? m - y : fminf(m - y, FLT_MAX)) * inv_bin, SMP_BINS - 1);
  }
  __device__ static float nearest(float d) { return (d + 0x1.8p23f) - 0x1.8p23f; }  // whole number, ties to even
  __device__ float bin_of(float y) const { return nearest(distance(y)); }           // the bins are around whole numbers
  // y: the sums up to and with this thread's bins
  template <bool COUNTS>
  __device__ void measure(float y[SMP_MINE], float& last) {
    uint32_t* h = hist();
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) h[i] = 0;
    __syncthreads();
    vectors([&](const float* y, int) {
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const float d = distance(y[i]), b = nearest(d);
        const int at = __float_as_int(d + 0x1.8p23f) & (SMP_BINS - 1);
        if (COUNTS) {
          atomicAdd(h + at, y[i] >= floor_ ? 1u : 0u);
        } else {
          // unit e^-r for the way r behind the bin's middle, |r| <= 12 / 2048 (the series' next term is under 2^-24), as a
          // whole number
          constexpr float step = SMP_SPAN / SMP_BINS;
          const float r = d - b, w = fmaf(r, fmaf(r, 0.5f * step * step * unit, -step * unit), unit + 0x1p23f);
          // (no branches around the additions: they would keep those of a vector apart)
          atomicAdd(h + at, b < SMP_BINS - 1 && (plain || y[i] >= floor_) ? __float_as_uint(w) - 0x4B000000u : 0u);
        }
      }
    });
    all_sync();
    uint32_t n[SMP_MINE] = {}, n_all = 0;
    float s[SMP_MINE] = {}, s_all = 0.f;
#pragma unroll
    for (int p = 0; p < SMP_PARTS; p++) {
      if (p >= parts) break;
      const uint4* from = reinterpret_cast<const uint4*>(at(h, p) + SMP_MINE * tid);
#pragma unroll
      for (int j = 0; j < SMP_MINE; j += 4) {
        const uint4 u = from[j / 4];
        if (COUNTS) n[j] += u.x, n[j + 1] += u.y, n[j + 2] += u.z, n[j + 3] += u.w;
        else s[j] += (float)u.x, s[j + 1] += (float)u.y, s[j + 2] += (float)u.z, s[j + 3] += (float)u.w;
      }
    }
    if (COUNTS) {
#pragma unroll
      for (int j = 0; j < SMP_MINE; j++) n_all += n[j];
      uint32_t all, before = scan_count(n_all, &all);
      last = __uint_as_float(all);
#pragma unroll
      for (int j = 0; j < SMP_MINE; j++) before += n[j], y[j] = __uint_as_float(before);
    } else {
      const float one = exp2_approx(-kLog2e * SMP_SPAN / SMP_BINS * SMP_MINE * tid) / unit;
#pragma unroll
      for (int j = 0; j < SMP_MINE; j++) s[j] *= one * exp2_approx(-kLog2e * SMP_SPAN / SMP_BINS * j), s_all += s[j];
      float before = scan_float(s_all, &last);
#pragma unroll
      for (int j = 0; j < SMP_MINE; j++) before += s[j], y[j] = before;
    }
  }
  // Most that the tokens of the last bin, which was not measured, can weigh.
  __device__ double tail() const { return (double)a.vocab * exp2_approx(-kLog2e * SMP_SPAN * (SMP_BINS - 2) / SMP_BINS); }

  // ---- exact sums of all tokens (if all; for one window their number too) and of those ahead of bin b0[i], and the tokens of bins
  // b0[i] .. b1[i] into the first block's lists, as far as there is room, for one window or two.  From each block
  template <int WINDOWS>
  __device__ const SmpExact* exactly(bool all, const float b0[WINDOWS], const float b1[WINDOWS]) {
    if (tid < 2) sh.n[tid] = 0;
    __syncthreads();
    SmpExact e = {};
    // The vectors that have a token of a window, few, are put into a list of the warp's own and looked at by all its lanes when
    // there are enough.
    uint32_t* own = along() + tid / 32 * SMP_OWN;
    uint32_t found = 0;
    auto look = [&]() {
      __syncwarp();
      for (uint32_t j = tid % 32; j < found; j += 32) {
        const int v = (int)own[j], id = first_id(v);
        float y[VEC];
        vec_values<In>(vec(v), y);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const float b = bin_of(y[i]);
#pragma unroll
          for (int k = 0; k < WINDOWS; k++)
            if (b >= b0[k] && b <= b1[k] && y[i] >= floor_) {
              e.n[k]++;
              const int n = (int)atomicAdd(sh.n + k, 1u);
              if (n < quota()) at(list(k), 0)[part * quota() + n] = place(rank_bits(y[i]), (uint32_t)(id + i));
            }
        }
      }
      __syncwarp();
      found = 0;
    };
    for (int v0 = 0; v0 < nv; v0 += SMP_THREADS) {
      const int v = v0 + tid;
      bool hit = false;
      if (v < nv) {
        float y[VEC], b[VEC], first = SMP_BINS;
        vec_values<In>(vec(v), y);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          b[i] = bin_of(y[i]);
          if (!plain && !(y[i] >= floor_)) b[i] = 2 * SMP_BINS;
          first = fminf(first, b[i]);
#pragma unroll
          for (int k = 0; k < WINDOWS; k++) hit |= b[i] >= b0[k] && b[i] <= b1[k];
        }
        bool ahead = first < b0[0];
        if (WINDOWS == 2) ahead |= first < b0[WINDOWS - 1];
        if (all || ahead) {
          double w[VEC];
#pragma unroll
          for (int i = 0; i < VEC; i++) w[i] = weight(y[i]);
          if (all) {
            if (plain) {
#pragma unroll
              for (int i = 0; i < VEC; i += 2) e.all += w[i] + w[i + 1];
            } else {
#pragma unroll
              for (int i = 0; i < VEC; i++) e.all += b[i] < SMP_BINS ? w[i] : 0.0;
            }
          }
          if (ahead) {
#pragma unroll
            for (int k = 0; k < WINDOWS; k++)
#pragma unroll
              for (int i = 0; i < VEC; i++) {
                e.ahead[k] += b[i] < b0[k] ? w[i] : 0.0;
                e.n_ahead[k] += b[i] < b0[k];
              }
          }
        }
        if (WINDOWS == 1 && all) {  // (with top-p the number of all is not asked for)
#pragma unroll
          for (int i = 0; i < VEC; i++) e.n_all += y[i] >= floor_;
        }
      }
      const uint32_t hits = __ballot_sync(0xffffffffu, hit);
      if (hit) own[found + __popc(hits & ((1u << tid % 32) - 1))] = (uint32_t)v;
      found += __popc(hits);
      if (found > SMP_OWN - 32) look();
    }
    look();
    auto sums = [](SmpExact& v, int lanes) {
      for (int o = lanes / 2; o; o >>= 1) {
        v.all += __shfl_xor_sync(0xffffffffu, v.all, o);
#pragma unroll
        for (int k = 0; k < WINDOWS; k++) v.ahead[k] += __shfl_xor_sync(0xffffffffu, v.ahead[k], o);
      }
      v.n_all = __reduce_add_sync(0xffffffffu, v.n_all);
#pragma unroll
      for (int k = 0; k < WINDOWS; k++) {
        v.n_ahead[k] = __reduce_add_sync(0xffffffffu, v.n_ahead[k]);
        v.n[k] = __reduce_add_sync(0xffffffffu, v.n[k]);
      }
    };
    sums(e, 32);
    if (tid % 32 == 0) sh.parts[tid / 32] = e;
    __syncthreads();
    SmpExact* told = sh.exact[turn++ & 1];
    if (tid < 32) {
      SmpExact v = sh.parts[tid % SMP_WARPS];
      if (tid >= SMP_WARPS) v = {};
      sums(v, 32);
      if (tid < parts) *at(told + part, tid) = v;
    }
    all_sync();
    return told;
  }
  // over the blocks
  __device__ SmpExact sum_of(const SmpExact* told) const {
    SmpExact r = {};
    for (int p = 0; p < parts; p++) {
      const SmpExact v = told[p];
      r.all += v.all, r.n_all += v.n_all;
      for (int k = 0; k < 2; k++) r.ahead[k] += v.ahead[k], r.n_ahead[k] += v.n_ahead[k], r.n[k] += v.n[k];
    }
    return r;
  }
  // whether the tokens of the windows have all found room
  __device__ bool room(const SmpExact* told) const {
    const SmpExact* v = told + (tid % 32 < parts ? tid % 32 : 0);
    return __reduce_max_sync(0xffffffffu, max(v->n[0], v->n[1])) <= quota();
  }

  __device__ static bool crosses(SmpKind kind, double mass, uint32_t count, double goal) {
    return kind == SMP_COUNT ? (double)count >= goal : kind == SMP_REACH ? mass >= goal : mass > goal;
  }

  // ---- the first bin with which a sum of `from` may be reached (a count: is), and the first with which one of `to` surely is
  // passed; y as measure() gives it
  __device__ void bins(bool counts, double from, double to, const float y[SMP_MINE], float& b0, float& b1) {
    if (tid == 0) sh.lo = sh.hi = SMP_BINS - 1;
    __syncthreads();
    // the least of the threads' first bins: a thread's sums and the next one's are rounded apart, so that where they meet neither
    // may see a step
    uint32_t lo = SMP_BINS - 1, hi = SMP_BINS - 1;
#pragma unroll
    for (int j = SMP_MINE - 1; j >= 0; j--) {
      const uint32_t b = SMP_MINE * tid + j;
      if (b >= SMP_BINS - 1) continue;
      const bool may = counts ? (double)__float_as_uint(y[j]) >= from : (double)(y[j] * (1.f + near_)) >= from;
      if (may) lo = b;
      if (counts ? may : (double)(y[j] * (1.f - near_)) > to) hi = b;
    }
    lo = __reduce_min_sync(0xffffffffu, lo), hi = __reduce_min_sync(0xffffffffu, hi);
    if (tid % 32 == 0) {
      if (lo < SMP_BINS - 1) atomicMin(&sh.lo, lo);
      if (hi < SMP_BINS - 1) atomicMin(&sh.hi, hi);
    }
    __syncthreads();
    b0 = (float)sh.lo, b1 = (float)sh.hi;
    __syncthreads();
  }
  // least and most that the sum of all tokens can be, from what was measured
  __device__ double least_sum(float last) const { return (double)last * (1.0 - near_); }
  __device__ double most_sum(float last) const { return (double)last * (1.0 + near_) + tail(); }

  // ---- no top-k: top-p, and the token, in one pass.  How much is kept is known well enough from the bins to say where the
  // token may be.  False where the tokens there find no room; then the sum and number of all are known.
  __device__ bool at_once(float p, double u, const float y[SMP_MINE], float last, double& all, uint32_t& n_all) {
    float b0[2], b1[2];
    double from = least_sum(last), to = most_sum(last);
    if (p < 1.f) {
      from *= (double)p, to *= (double)p;
      bins(false, from, to, y, b0[1], b1[1]);
      // what is kept ends in these bins
#pragma unroll
      for (int j = 0; j < SMP_MINE; j++)
        if (SMP_MINE * tid + j == (int)b1[1]) sh.fscan[0] = y[j];
      __syncthreads();
      to = b1[1] < SMP_BINS - 1 ? (double)sh.fscan[0] * (1.0 + near_) : most_sum(last);
      __syncthreads();
    } else {
      b0[1] = 3 * SMP_BINS, b1[1] = 2.5f * SMP_BINS;  // no window
    }
    bins(false, u * from, u * to, y, b0[0], b1[0]);
    const SmpExact* told = p < 1.f ? exactly<2>(true, b0, b1) : exactly<1>(true, b0, b1);
    if (!room(told)) {
      const SmpExact r = sum_of(told);
      all = r.all, n_all = r.n_all;
      return false;
    }
    if (part) return true;
    const SmpExact r = sum_of(told);
    double mass = r.all, w[SMP_EACH], c[SMP_EACH];
    uint32_t kept = r.n_all;
    uint64_t last_place = 0;
    if (p < 1.f) {
      const uint32_t n = r.n[1];
      put_in_order(told, (int)n, 1);
      sums_of((int)n, w, c);
      const double goal = (double)p * mass;
      const uint32_t ahead = min(number((int)n, w, c, [&](int, double, double s) { return r.ahead[1] + s < goal; }), n - 1);
      at_token(ahead, c, [&](uint64_t place, double s) { sh.found = {place, r.ahead[1] + s, r.n_ahead[1] + ahead + 1}; });
      __syncthreads();
      mass = sh.found.mass, kept = sh.found.count, last_place = sh.found.place;
    }
    const uint32_t n = r.n[0];
    put_in_order(told, (int)n, 0);
    sums_of((int)n, w, c);
    const double goal = u * mass;
    const uint32_t ahead = min(number((int)n, w, c, [&](int, double, double s) { return r.ahead[0] + s <= goal; }), n - 1);
    if (tid == 0) {
      const uint64_t found = r.n_ahead[0] + ahead < kept ? ordered()[ahead] : last_place;  // (else by rounding alone)
      answer((int)~(uint32_t)found, logprob(found, mass), kept);
    }
    return true;
  }

  // ---- the token at which the count or the sum crosses `goal`.  (kind SMP_PASS, the last one: for the first block alone)
  __device__ SmpFound search(SmpKind kind, double goal, const float y[SMP_MINE]) {
    float b0, b1;
    bins(kind == SMP_COUNT, goal, goal, y, b0, b1);
    SmpWindow w;
    const SmpExact* told = exactly<1>(false, &b0, &b1);
    const SmpExact r = sum_of(told);
    w.mass = r.ahead[0], w.ahead = r.n_ahead[0], w.count = r.n[0], w.before = 0;
    for (int q = 0; q < part; q++) w.before += told[q].n[0];
    if (room(told)) return among(kind, goal, w, told, parts);
    // the ranks of these bins, which are monotone in the value
    const uint32_t least = rank_bits(floor_), most = rank_bits(m);
    uint32_t lo = least, hi = most;
    while (lo < hi) {  // smallest rank whose bin is b1 or an earlier one
      const uint32_t mid = lo + (hi - lo) / 2;
      if (bin_of(rank_value(mid)) <= b1) hi = mid;
      else lo = mid + 1;
    }
    w.lo = lo;
    hi = most;
    while (lo < hi) {  // largest whose bin is b0 or a later one
      const uint32_t mid = hi - (hi - lo) / 2;
      if (bin_of(rank_value(mid)) >= b0) lo = mid;
      else hi = mid - 1;
    }
    w.hi = lo;
    return closer(kind, goal, w);
  }

  // ---- the window's tokens are in the first block's list
  template <typename Found>
  __device__ SmpFound among(SmpKind kind, double goal, const SmpWindow& w, const Found* from, int blocks) {
    if (part == 0) {
      const uint32_t n = w.count;
      put_in_order(from, (int)n, 0, blocks);
      double wt[SMP_EACH], c[SMP_EACH];
      sums_of((int)n, wt, c);
      uint32_t ahead = number((int)n, wt, c, [&](int i, double, double s) { return !crosses(kind, w.mass + s, w.ahead + i + 1, goal); });
      ahead = min(ahead, n - 1);
      at_token(ahead, c, [&](uint64_t place, double s) {
        const SmpFound f = {place, w.mass + s, w.ahead + ahead + 1};
        for (int p = 0; p < (kind == SMP_PASS ? 1 : parts); p++) *at(&sh.found, p) = f;
      });
      __syncthreads();
    }
    if (kind != SMP_PASS) all_sync();
    return sh.found;
  }

  // ---- a window of many tokens: exact sums over 16 bins of its ranks, the one with the crossing becomes the window
  __device__ SmpFound closer(SmpKind kind, double goal, SmpWindow w) {
    while (true) {
      all_sync();  // what was found, or listed, before has been read
      if (w.count <= SMP_LIST) {
        if (tid == 0) sh.n[0] = 0;
        __syncthreads();
        // one list, whatever the blocks' shares: the first block's part of it is all
        uint64_t* to = at(list(), 0);
        each([&](float y, int id) {
          const uint32_t r = rank_bits(y);
          if (r - w.lo <= w.hi - w.lo) to[w.before + atomicAdd(sh.n, 1)] = place(r, (uint32_t)id);
        });
        all_sync();
        const uint2 all_in_first = make_uint2(w.count, 0);
        return among(kind, goal, w, &all_in_first, 1);
      }
      if (w.lo == w.hi) return tied(kind, goal, w);
      const uint32_t range = w.hi - w.lo, hi = w.hi, shift = max(0, 28 - __clz(range));
      SmpSums& s = sh.next[turn++ & 1];
      cut(s, w.lo, w.hi, shift);
      const int b = choose(s, kind, goal, w);
      w.hi = hi - ((uint32_t)b << shift);
      const uint64_t below = ((uint64_t)(b + 1) << shift) - 1;
      w.lo = below < hi - w.lo ? hi - (uint32_t)below : w.lo;
    }
  }
  __device__ void cut(SmpSums& to, uint32_t lo, uint32_t hi, uint32_t shift) {
    if (tid < SMP_CUTTERS) {
      double* mass = cut_mass() + tid;
      uint32_t* count = cut_count() + tid;
#pragma unroll
      for (int b = 0; b < SMP_CUT; b++) mass[b * SMP_CUTTERS] = 0.0, count[b * SMP_CUTTERS] = 0;
      vectors([&](const float* y, int) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const uint32_t r = rank_bits(y[i]);
          if (r - lo > hi - lo) continue;
          const int b = (int)((hi - r) >> shift) * SMP_CUTTERS;
          mass[b] += weight(y[i]);
          count[b]++;
        }
      }, SMP_CUTTERS);
    }
    __syncthreads();
    // a warp a bin
    for (int b = tid / 32; b < SMP_CUT; b += SMP_WARPS) {
      const int i = tid % 32;
      const double s = warp_sum(cut_mass()[b * SMP_CUTTERS + i] + cut_mass()[b * SMP_CUTTERS + 32 + i]);
      const uint32_t n = __reduce_add_sync(0xffffffffu, cut_count()[b * SMP_CUTTERS + i] + cut_count()[b * SMP_CUTTERS + 32 + i]);
      if (i < parts) {
        *at(&to.mass[part][b], i) = s;
        *at(&to.count[part][b], i) = n;
      }
    }
    all_sync();
  }
  // the bin of the window in which the number is crossed (rounding: else the last with a token), into w; its number
  __device__ int choose(const SmpSums& s, SmpKind kind, double goal, SmpWindow& w) const {
    int last = 0;
    SmpWindow at = w, hit = w;
    for (int b = 0; b < SMP_CUT; b++) {
      double mass = 0.0;
      uint32_t n = 0, before = 0;
      for (int p = 0; p < parts; p++) {
        mass += s.mass[p][b];
        if (p < part) before += s.count[p][b];
        n += s.count[p][b];
      }
      if (!n) continue;
      last = b;
      hit = at;
      hit.count = n;
      hit.before = before;
      if (crosses(kind, at.mass + mass, at.ahead + n, goal)) break;
      at.mass += mass;
      at.ahead += n;
    }
    w.mass = hit.mass, w.ahead = hit.ahead, w.count = hit.count, w.before = hit.before;
    return last;
  }
  // ---- many tokens of one value: the id decides
  __device__ SmpFound tied(SmpKind kind, double goal, const SmpWindow& w) {
    const float y = rank_value(w.lo);
    const double wt = weight(y);
    double j;
    if (kind == SMP_COUNT) {
      j = goal - w.ahead;
    } else {
      j = wt > 0.0 ? floor((goal - w.mass) / wt) : 0.0;
      j = fmin(fmax(j, 1.0), (double)w.count);
      for (int i = 0; i < 4 && j > 1.0 && crosses(kind, w.mass + (j - 1.0) * wt, 0, goal); i++) j -= 1.0;
      for (int i = 0; i < 4 && j < (double)w.count && !crosses(kind, w.mass + j * wt, 0, goal); i++) j += 1.0;
    }
    const uint32_t nth = (uint32_t)fmin(fmax(j, 1.0), (double)w.count);  // from 1
    uint32_t seen = w.before;
    for (int b = 0; b < nv && seen < nth; b += SMP_THREADS) {
      float v[VEC];
      const bool has = b + tid < nv;
      if (has) vec_values<In>(vec(b + tid), v);
      uint32_t here = 0, total;
#pragma unroll
      for (int i = 0; i < VEC; i++) here += has && v[i] == y;
      uint32_t before = seen + scan_count(here, &total);
      if (has && before < nth && nth <= before + here) {
#pragma unroll
        for (int i = 0; i < VEC; i++)
          if (v[i] == y && ++before == nth) {
            const SmpFound f = {place(w.lo, (uint32_t)(first_id(b + tid) + i)), w.mass + nth * wt, w.ahead + nth};
            for (int p = 0; p < parts; p++) *at(&sh.found, p) = f;
          }
      }
      seen += total;
    }
    all_sync();
    return sh.found;
  }

  __device__ void run() {
    const int row = blockIdx.x / parts;
    float t = a.temperature ? a.temperature[row] : 1.f, p = a.top_p ? a.top_p[row] : 1.f;
    const float min_p = a.min_p ? a.min_p[row] : 0.f;
    int k = a.top_k ? a.top_k[row] : 0;
    double u = a.uniform[row];
    const uint2* told = load(k);
    const uint32_t most = most_of(&told->x);
    if (k < 0 || k >= a.vocab) k = 0;
    u = u > 0.0 ? fmin(u, 0x1.fffffffffffffp-1) : 0.0;
    m = rank_value(most);
    if (!(fabsf(m) <= FLT_MAX) || t != t) {  // nothing to choose from, or no sense in it
      if (part == 0 && tid == 0) answer(-1, -INFINITY, 0);
      return;
    }
    if (t <= 0.f || k == 1 || p <= 0.f) {  // the first in line
      uint32_t first = 0;
      each([&](float y, int id) {
        if (y == m) first = max(first, ~(uint32_t)id);
      });
      told = tell(block_max(first));
      if (part == 0 && tid == 0) {
        for (int q = 0; q < parts; q++) first = max(first, told[q].x);
        answer((int)~first, 0.0, 1);
      }
      return;
    }
    top = m;
    inv_t = 1.0 / (double)t;
    // A temperature under 2^-10 of m's last bit leaves nothing but m, as that one does, and keeps z within 32 bits.
    const float below = rank_value(most - 1), t_weight = fmaxf(t, (m - below) * 0x1p-10f);
    rate = 64 * 1.44269504088896340736 / (double)t_weight;
    lowest = fminf(m - 600.f * t_weight, below);
    floor_ = -FLT_MAX;
    if (min_p >= 1.f) floor_ = m;
    else if (min_p > 0.f) floor_ = fmaxf(floor_, __double2float_ru(top + (double)t * log((double)min_p)));
    if (bounded(k) || (k && k <= SMP_TOP && a.vocab <= SMP_LIST) || min_p > 0.f) {
      float from = floor_;
      if (bounded(k)) {
        const uint32_t least = least_of(&told->y);
        from = fmaxf(from, rank_value(max(least, rank_bits(-FLT_MAX))));
      }
      told = gather(from);
      if (room(told)) {
        int n = 0;
        for (int q = 0; q < parts; q++) n += (int)told[q].x;
        if (part == 0) finish(told, n, k, p, u);
        return;
      }
    }
    inv_bin = fminf(SMP_BINS / (SMP_SPAN * t), FLT_MAX);
    plain = floor_ == -FLT_MAX && lowest > -FLT_MAX && inv_bin > 0.f;
    __syncthreads();
    double mass = 0.0;
    uint32_t kept = 0;
    uint64_t end = 0;       // the last place that is kept, where that is known
    float y[SMP_MINE], last;
    bool known = false;     // whether mass and kept are
    if (k) {
      measure<true>(y, last);
      if ((uint32_t)k < __float_as_uint(last)) {
        const SmpFound f = search(SMP_COUNT, (double)k, y);
        mass = f.mass, kept = f.count, end = f.place;
        known = true;
      }
      all_sync();  // the histogram has been read
    }
    measure<false>(y, last);
    if (!known && at_once(p, u, y, last, mass, kept)) return;
    if (p < 1.f) {
      const SmpFound f = search(SMP_REACH, (double)p * mass, y);
      if (!known || f.count < kept) mass = f.mass, kept = f.count, end = f.place;
    }
    SmpFound f = search(SMP_PASS, u * mass, y);
    if (f.count > kept) f.place = end;  // by rounding alone
    if (part == 0 && tid == 0) answer((int)~(uint32_t)f.place, logprob(f.place, mass), kept);
  }
};

template <typename In, bool HELD>
__global__ void __launch_bounds__(SMP_THREADS, 2) sample_kernel(const __grid_constant__ IrisSample a) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ SmpShared sh;
  if (a.parts > 1) iris::cluster_sync();  // all blocks are there
  iris::grid_dep_wait();
  iris::grid_dep_launch();
  SmpRow<In, HELD> r(a, sh, smem);
  r.run();
}

constexpr int SMP_MOST = 170 * 1024;  // bytes of a block's part of a row, held
constexpr int SMP_PART = 75 * 1024;   // the same where two blocks are to fit an SM

template <typename In>
cudaError_t launch(IrisSample* a, int num_sms, cudaStream_t stream) {
  const int64_t bytes = (int64_t)a->vocab * (int64_t)sizeof(In) + 16;
  // Blocks on a row: as many as leave each no more than SMP_PART of it, so that two fit an SM (512 f32 rows of 151936, usual
  // settings 167 us, 201 with twice that; top-p alone 594 and 581), and more where each keeps 16 KB and the device has room
  // for them: for two blocks an SM up to four a row (48 bf16 rows of 32000 with top-p 24 us, 28 with one), for eight, of which
  // clusters reach seven eighths of the SMs, one (16 bf16 rows of 151936, usual settings 9.7 us, 11.4 with four; 32 rows 15.4 with
  // eight and two an SM, 12.2 with four).
  a->parts = 1;
  while (a->parts < SMP_PARTS &&
         (bytes > (int64_t)a->parts * SMP_PART ||
          (bytes > (int64_t)a->parts * 16384 &&
           (int64_t)a->rows * a->parts * 2 <= (a->parts < 4 ? 2 * num_sms : num_sms * 7 / 8))))
    a->parts *= 2;
  const int64_t vecs = (bytes + 15) / 16, held = (vecs + a->parts - 1) / a->parts * 16;
  const bool fits = held <= SMP_MOST;
  a->held_bytes = fits ? (int)((held + 127) / 128 * 128) : 0;
  const size_t smem = (size_t)a->held_bytes + SMP_WORK;
  const dim3 grid((unsigned)a->rows * a->parts);
  auto kernel = fits ? sample_kernel<In, true> : sample_kernel<In, false>;
  if (a->parts == 1) return iris::launch_overlapped(kernel, grid, dim3(SMP_THREADS), smem, stream, *a);
  return iris::launch_cluster_overlapped(kernel, grid, dim3(SMP_THREADS), smem, a->parts, stream, *a);
}

}  // namespace

extern "C" cudaError_t iris_sample_init(void) {
  const void* k[] = {(const void*)sample_kernel<float, true>, (const void*)sample_kernel<float, false>,
                     (const void*)sample_kernel<__nv_bfloat16, true>, (const void*)sample_kernel<__nv_bfloat16, false>};
  for (int i = 0; i < 4; i++) {
    const cudaError_t e = cudaFuncSetAttribute(k[i], cudaFuncAttributeMaxDynamicSharedMemorySize, (i % 2 ? 0 : SMP_MOST) + SMP_WORK);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

extern "C" cudaError_t iris_launch_sample(IrisSample* a, int f32, int num_sms, cudaStream_t stream) {
  return f32 ? launch<float>(a, num_sms, stream) : launch<__nv_bfloat16>(a, num_sms, stream);
}
