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
// With top-k of up to SMP_TOP, or where min-p leaves few, the tokens above a bound
// (which k of the threads' own largest reach) are few: one block puts them in order
// and has the answer.  Else a histogram over the distance from m, in parts of
// SMP_SPAN / SMP_BINS of t, says to 2^-14 (large vocabularies: less closely) how the sum grows along the line
// (each value adds its weight relative to its bin's, a whole number of 16 bits, so
// that no order of additions shows); a pass over the row adds up exactly what
// stands ahead of the bins in which the number is crossed and collects their
// tokens, some hundreds, which one block puts in order.  Where they are too many
// (equal logits, high temperatures) the bins are cut further, each time into 16,
// with exact sums, until few are left, or tokens of one value, of which the id decides.
// Weights and sums are 64-bit: a token is taken by where a sum of 100000 weights
// ends, and with 32 bits one row in a hundred would take its neighbour.
constexpr int SMP_THREADS = 512, SMP_WARPS = SMP_THREADS / 32, SMP_PARTS = 8;
constexpr int SMP_LIST = 1024;  // tokens put in order: two a thread
constexpr int SMP_TOP = 512;    // largest top-k whose tokens are looked for through a bound
constexpr int SMP_BINS = 2048;  // four a thread
constexpr float SMP_SPAN = 24.f;      // (m - x) / t that the bins cover; the last one holds all that is below
constexpr int SMP_CUT = 16, SMP_CUTTERS = 64;  // bins of a closer look, threads that fill bins of their own
static_assert(SMP_BINS == 4 * SMP_THREADS && SMP_LIST == 2 * SMP_THREADS && SMP_CUT == SMP_WARPS, "shares of a thread, and warp");

struct SmpSums {  // of the closer bins, from each block of the cluster
  double mass[SMP_PARTS][SMP_CUT];
  uint32_t count[SMP_PARTS][SMP_CUT];
};

struct SmpFound {
  uint64_t place;
  double mass;     // of the line up to and with it
  uint32_t count;
};

struct SmpExact {  // of a block
  double all, ahead;      // sums of all tokens, of those ahead of the window
  uint32_t n_all, n_ahead, n;  // tokens: all, ahead, in the window
};

struct SmpShared {
  SmpSums next[2];             // in turn, so that one round's may be read while the next one's come
  SmpExact exact[2][SMP_PARTS];
  uint32_t one[2][SMP_PARTS];  // a number from each block
  SmpExact parts[SMP_WARPS];   // of a block's warps
  double scan[SMP_WARPS];
  float fscan[SMP_WARPS];
  uint32_t iscan[SMP_WARPS];
  double root[64];             // 2^(i / 64)
  SmpFound found;
  uint32_t n, lo, hi;
};

// shared memory besides the row: the histogram, the sums along the bins, and the list, in whose place the closer bins stand
constexpr int SMP_HIST = SMP_BINS * 4, SMP_ALONG = SMP_BINS * 4;
constexpr int SMP_TAIL = SMP_CUT * SMP_CUTTERS * (8 + 4);
constexpr int SMP_WORK = SMP_HIST + SMP_ALONG + SMP_TAIL;
static_assert(SMP_TAIL >= SMP_LIST * 8 && SMP_ALONG >= SMP_LIST * 8 && SMP_HIST >= SMP_LIST * 8, "the lists fit");

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
  float m, floor_, cut_off;  // cut_off: what lies further under m weighs nothing, e^-620
  double top, inv_t, rate;   // rate: 64 log2(e) / t
  float inv_bin;
  float unit;                // of the histogram's weights, so that a block's tokens in one bin stay within 32 bits
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
  __device__ float* along() const { return reinterpret_cast<float*>(work() + SMP_HIST); }  // sums up to and with a bin, or counts
  __device__ uint64_t* list() const { return reinterpret_cast<uint64_t*>(work() + SMP_HIST + SMP_ALONG); }
  __device__ uint64_t* own_list() const { return reinterpret_cast<uint64_t*>(along()); }  // before there are sums; again for what is in order
  __device__ double* line() const { return reinterpret_cast<double*>(hist()); }           // when there is no histogram
  __device__ double* cut_mass() const { return reinterpret_cast<double*>(list()); }
  __device__ uint32_t* cut_count() const { return reinterpret_cast<uint32_t*>(cut_mass() + SMP_CUT * SMP_CUTTERS); }

  __device__ void all_sync() const {
    __syncwarp();
    if (parts > 1) iris::cluster_sync();
    else __syncthreads();
  }
  template <typename T>
  __device__ T* at(T* p, int rank) const { return parts > 1 ? iris::cluster_map(p, (uint32_t)rank) : p; }
  // this block's number, the same in all threads, to all of them; the numbers of the blocks after the barrier
  __device__ const uint32_t* tell(uint32_t v) {
    uint32_t* to = sh.one[turn++ & 1];
    if (tid < parts) *at(to + part, tid) = v;
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
    const double z = ((double)y - top) * rate;
    const double shifted = z + 0x1.8p52;
    const int n = __double2loint(shifted);
    const double r = z - (shifted - 0x1.8p52);
    double p = fma(r, c * c * c * c / 24, c * c * c / 6);
    p = fma(r, p, c * c / 2);
    p = fma(r, p, c);
    p = fma(r, p, 1.0) * sh.root[n & 63];
    const double w = __hiloint2double(__double2hiint(p) + (n >> 6) * (1 << 20), __double2loint(p));
    return m - y > cut_off ? 0.0 : w;
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
  __device__ uint32_t block_sum(uint32_t v) {
    v = __reduce_add_sync(0xffffffffu, v);
    if (tid % 32 == 0) sh.iscan[tid / 32] = v;
    __syncthreads();
    v = __reduce_add_sync(0xffffffffu, tid % 32 < SMP_WARPS ? sh.iscan[tid % SMP_WARPS] : 0u);
    __syncthreads();
    return v;
  }
  __device__ static double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  }
  // sum of what the threads ahead have
  __device__ uint32_t scan_count(uint32_t v, uint32_t* total) {
    uint32_t incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, incl, o);
      if (tid % 32 >= o) incl += y;
    }
    if (tid % 32 == 31) sh.iscan[tid / 32] = incl;
    __syncthreads();
    uint32_t before = incl - v;
    *total = 0;
    for (int w = 0; w < SMP_WARPS; w++) {
      if (w < tid / 32) before += sh.iscan[w];
      *total += sh.iscan[w];
    }
    __syncthreads();
    return before;
  }
  __device__ float scan_float(float v) {
    float incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float y = __shfl_up_sync(0xffffffffu, incl, o);
      if (tid % 32 >= o) incl += y;
    }
    if (tid % 32 == 31) sh.fscan[tid / 32] = incl;
    __syncthreads();
    float ahead = 0.f;
    for (int w = 0; w < tid / 32; w++) ahead += sh.fscan[w];
    __syncthreads();
    return ahead + (incl - v);
  }
  __device__ double scan_mass(double v) {
    double incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, incl, o);
      if (tid % 32 >= o) incl += y;
    }
    if (tid % 32 == 31) sh.scan[tid / 32] = incl;
    __syncthreads();
    const double before = incl - v;
    double ahead = 0;
    for (int w = 0; w < tid / 32; w++) ahead += sh.scan[w];
    __syncthreads();
    return ahead + before;
  }

  // ---- the row, its largest value (NaN if there is one); each thread's own largest in `own`, each warp's in sh.iscan
  __device__ uint32_t load(uint32_t& own) {
    float best = -INFINITY;
    constexpr int FLY = 10;  // 76 KB of a row in one round
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
    own = rank_bits(best);
    const uint32_t w = __reduce_max_sync(0xffffffffu, own);
    if (tid % 32 == 0) sh.iscan[tid / 32] = w;
    __syncthreads();
    const uint32_t* all = tell(__reduce_max_sync(0xffffffffu, sh.iscan[tid % SMP_WARPS]));
    uint32_t r = 0;
    for (int p = 0; p < parts; p++) r = max(r, all[p]);
    return r;
  }

  // ---- a value that `share` of this block's tokens reach, 0 if it may have fewer; sh.iscan as load() leaves it
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

  // ---- the tokens from `from` on, each block's in its own list; how many there are in the whole row (each block's in `all`)
  __device__ uint32_t gather(float from, const uint32_t*& all) {
    if (tid == 0) sh.n = 0;
    __syncthreads();
    vectors([&](const float* y, int id) {
      float most = y[0];
#pragma unroll
      for (int i = 1; i < VEC; i++) most = fmaxf(most, y[i]);
      if (most < from || *(volatile uint32_t*)&sh.n > SMP_LIST) return;  // none, or too many already
#pragma unroll
      for (int i = 0; i < VEC; i++)
        if (y[i] >= from) {
          const uint32_t n = atomicAdd(&sh.n, 1);
          if (n < SMP_LIST) own_list()[n] = place(rank_bits(y[i]), (uint32_t)(id + i));
        }
    });
    __syncthreads();
    all = tell(sh.n);
    uint32_t n = 0;
    for (int p = 0; p < parts; p++) n += min(all[p], SMP_LIST + 1);
    return n;
  }

  // ---- by the first block: list()[0, n) in order, largest first.  Few by counting how many are ahead of each, all threads
  // at it (n^2 steps); more by a bitonic sort, with what is missing to a power of two as 0.
  __device__ void put_in_order(int n) {
    uint64_t* l = list();
    __syncthreads();
    if (n <= 256) {
      int per = 2;  // threads to a token
      while (per < 32 && 2 * per * n <= SMP_THREADS) per *= 2;
      const int i = tid / per;
      const uint64_t mine = i < n ? l[i] : 0;
      int ahead = 0;
#pragma unroll 4
      for (int j = tid % per; j < n; j += per) ahead += l[j] > mine;
      for (int o = per / 2; o; o >>= 1) ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
      __syncthreads();
      if (i < n && tid % per == 0) l[ahead] = mine;
      __syncthreads();
      return;
    }
    int size = 512;
    while (size < n) size *= 2;
    for (int i = n + tid; i < size; i += SMP_THREADS) l[i] = 0;
    __syncthreads();
    for (int k = 2; k <= size; k *= 2)
      for (int j = k / 2; j; j /= 2) {
        // within 64 places a warp has them to itself
        if (j >= 32) __syncthreads();
        else __syncwarp();
        if (2 * tid < size) {
          const int i = 2 * (tid & ~(j - 1)) + (tid & (j - 1));
          const uint64_t p = l[i], q = l[i + j];
          if ((p < q) == ((i & k) == 0)) l[i] = q, l[i + j] = p;
        }
      }
    __syncthreads();
  }
  // weights of this thread's two tokens of the list
  __device__ void weights(int n, double w[2]) const {
#pragma unroll
    for (int j = 0; j < 2; j++) w[j] = 2 * tid + j < n ? weight(rank_value((uint32_t)(list()[2 * tid + j] >> 32))) : 0.0;
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

  // ---- all that can be kept is in list(): by the first block
  __device__ void finish(int n, int k, float p, double u) {
    put_in_order(n);
    if (k) n = min(n, k);
    double w[2];
    weights(n, w);
    const double before = scan_mass(w[0] + w[1]), c0 = before + w[0], c1 = c0 + w[1];
    double* sums = line();
    sums[2 * tid] = c0, sums[2 * tid + 1] = c1;
    __syncthreads();
    const double mass = sums[n - 1];
    uint32_t kept = n;
    if (p < 1.f) {
      const double goal = (double)p * mass;
      kept = max(block_sum((2 * tid < n && before < goal) + (2 * tid + 1 < n && c0 < goal)), 1u);
    }
    const double m_kept = sums[kept - 1], goal = u * m_kept;
    uint32_t pick = block_sum((2 * tid < kept && c0 <= goal) + (2 * tid + 1 < kept && c1 <= goal));
    const uint32_t heavy = block_sum((2 * tid < kept && w[0] > 0.0) + (2 * tid + 1 < kept && w[1] > 0.0));
    pick = min(pick, heavy - 1);  // the first one weighs 1
    if (tid == 0) answer((int)~(uint32_t)list()[pick], logprob(list()[pick], m_kept), kept);
  }

  // ---- how the line grows along the bins: along()[b] is the sum up to and with bin b, to near_ (or the count, a whole number)
  __device__ float distance(float y) const { return fminf(fminf(m - y, FLT_MAX) * inv_bin, SMP_BINS - 1); }
  __device__ static float nearest(float d) { return (d + 0x1.8p23f) - 0x1.8p23f; }  // whole number, ties to even
  __device__ float bin_of(float y) const { return nearest(distance(y)); }           // the bins are around whole numbers
  template <bool COUNTS>
  __device__ void measure() {
    uint32_t* h = hist();
    for (int i = tid; i < SMP_BINS; i += SMP_THREADS) h[i] = 0;
    __syncthreads();
    vectors([&](const float* y, int) {
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        const float d = distance(y[i]), b = nearest(d);
        const int at = __float_as_int(d + 0x1.8p23f) & (SMP_BINS - 1);
        if (COUNTS) {
          if (y[i] >= floor_) atomicAdd(h + at, 1u);
        } else {
          // unit e^-r for the way r behind the bin's middle, |r| <= 12 / 2048 (the series' next term is under 2^-24), as a
          // whole number
          const float r = (d - b) * (SMP_SPAN / SMP_BINS);
          const float w = fmaf(unit, r * fmaf(0.5f, r, -1.f), unit + 0x1p23f);
          if (y[i] >= floor_ && b < SMP_BINS - 1) atomicAdd(h + at, __float_as_uint(w) - 0x4B000000u);
        }
      }
    });
    all_sync();
    float mass[4];
    uint32_t n[4] = {0, 0, 0, 0};
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int p = 0; p < parts; p++) {
      const uint4 u = *reinterpret_cast<const uint4*>(at(h, p) + 4 * tid);
      if (COUNTS) n[0] += u.x, n[1] += u.y, n[2] += u.z, n[3] += u.w;
      else s[0] += (float)u.x, s[1] += (float)u.y, s[2] += (float)u.z, s[3] += (float)u.w;
    }
    if (COUNTS) {
      uint32_t all, before = scan_count(n[0] + n[1] + n[2] + n[3], &all);
#pragma unroll
      for (int j = 0; j < 4; j++) before += n[j], mass[j] = __uint_as_float(before);
    } else {
      const float one = exp2_approx(-kLog2e * SMP_SPAN / SMP_BINS * 4 * tid) / unit;
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] *= one * exp2_approx(-kLog2e * SMP_SPAN / SMP_BINS * j);
      float before = scan_float((s[0] + s[1]) + (s[2] + s[3]));
#pragma unroll
      for (int j = 0; j < 4; j++) before += s[j], mass[j] = before;
    }
    *reinterpret_cast<float4*>(along() + 4 * tid) = make_float4(mass[0], mass[1], mass[2], mass[3]);
    __syncthreads();
  }
  // Most that the tokens of the last bin, which was not measured, can weigh.
  __device__ double tail() const { return (double)a.vocab * exp2_approx(-kLog2e * SMP_SPAN * (SMP_BINS - 2) / SMP_BINS); }

  // ---- exact sums and counts of all tokens (all: else only the counts), of those ahead of bin b0, and the tokens of bins b0
  // .. b1 into the first block's list, as far as there is room
  __device__ SmpExact exactly(bool all, float b0, float b1, uint32_t& before) {
    if (tid == 0) sh.n = 0;
    all_sync();  // the first block's list is free, its count 0
    SmpExact e = {0.0, 0.0, 0, 0, 0};
    uint32_t* count = at(&sh.n, 0);
    uint64_t* to = at(list(), 0);
    vectors([&](const float* y, int id) {
      float b[VEC], first = 2 * SMP_BINS;
#pragma unroll
      for (int i = 0; i < VEC; i++) {
        b[i] = y[i] >= floor_ ? bin_of(y[i]) : 2 * SMP_BINS;
        e.n_all += b[i] < SMP_BINS;
        first = fminf(first, b[i]);
      }
      if (all || first < b0) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const double w = weight(y[i]);
          if (all) e.all += b[i] < SMP_BINS ? w : 0.0;
          if (b[i] < b0) e.ahead += w, e.n_ahead++;
        }
      }
      if (first <= b1) {
#pragma unroll
        for (int i = 0; i < VEC; i++)
          if (b[i] >= b0 && b[i] <= b1) {
            e.n++;
            const uint32_t k = atomicAdd(count, 1u);
            if (k < SMP_LIST) to[k] = place(rank_bits(y[i]), (uint32_t)(id + i));
          }
      }
    });
    auto over_lanes = [](SmpExact& v, int lanes) {
      for (int o = lanes / 2; o; o >>= 1) {
        v.all += __shfl_xor_sync(0xffffffffu, v.all, o);
        v.ahead += __shfl_xor_sync(0xffffffffu, v.ahead, o);
      }
    };
    over_lanes(e, 32);
    e.n_all = __reduce_add_sync(0xffffffffu, e.n_all);
    e.n_ahead = __reduce_add_sync(0xffffffffu, e.n_ahead);
    e.n = __reduce_add_sync(0xffffffffu, e.n);
    if (tid % 32 == 0) sh.parts[tid / 32] = e;
    __syncthreads();
    SmpExact* told = sh.exact[turn++ & 1];
    if (tid < 32) {
      SmpExact v = sh.parts[tid % SMP_WARPS];
      over_lanes(v, SMP_WARPS);
      if (tid >= SMP_WARPS) v.n_all = v.n_ahead = v.n = 0;
      v.n_all = __reduce_add_sync(0xffffffffu, v.n_all);
      v.n_ahead = __reduce_add_sync(0xffffffffu, v.n_ahead);
      v.n = __reduce_add_sync(0xffffffffu, v.n);
      if (tid < parts) *at(told + part, tid) = v;
    }
    all_sync();
    SmpExact r = {0.0, 0.0, 0, 0, 0};
    before = 0;
    for (int p = 0; p < parts; p++) {
      r.all += told[p].all, r.ahead += told[p].ahead;
      if (p < part) before += told[p].n;
      r.n_all += told[p].n_all, r.n_ahead += told[p].n_ahead, r.n += told[p].n;
    }
    return r;
  }

  __device__ static bool crosses(SmpKind kind, double mass, uint32_t count, double goal) {
    return kind == SMP_COUNT ? (double)count >= goal : kind == SMP_REACH ? mass >= goal : mass > goal;
  }

  // ---- the token at which the count or the sum crosses `goal`; before the sum of all tokens is known, share of it.  all:
  // gets that sum, and the number of tokens
  __device__ SmpFound search(SmpKind kind, double goal, double share, double* all, uint32_t* n_all) {
    // the first bin with which the number may be crossed, and the first with which it surely is
    if (tid == 0) sh.lo = sh.hi = SMP_BINS - 1;
    __syncthreads();
    const float4 four = *reinterpret_cast<const float4*>(along() + 4 * tid);
    const float y[5] = {tid ? along()[4 * tid - 1] : 0.f, four.x, four.y, four.z, four.w};
    double from = goal, to = goal;
    if (all) {
      const float last = along()[SMP_BINS - 1];
      from = share * last * (1.0 - near_), to = share * (last * (1.0 + near_) + tail());
    }
#pragma unroll
    for (int j = 0; j < 4; j++) {
      auto may = [&](float v) { return kind == SMP_COUNT ? (double)__float_as_uint(v) >= goal : v * (1.0 + near_) >= from; };
      auto must = [&](float v) { return kind == SMP_COUNT ? (double)__float_as_uint(v) >= goal : v * (1.0 - near_) > to; };
      const int b = 4 * tid + j;
      if (b < SMP_BINS - 1 && may(y[j + 1]) && !(b && may(y[j]))) sh.lo = b;
      if (b < SMP_BINS - 1 && must(y[j + 1]) && !(b && must(y[j]))) sh.hi = b;
    }
    __syncthreads();
    const float b0 = (float)sh.lo, b1 = (float)sh.hi;
    SmpWindow w;
    const SmpExact r = exactly(all != nullptr, b0, b1, w.before);
    if (all) *all = r.all, *n_all = r.n_all, goal = share * r.all;
    w.mass = r.ahead, w.ahead = r.n_ahead, w.count = r.n;
    if (w.count <= SMP_LIST) return among(kind, goal, w);
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
  __device__ SmpFound among(SmpKind kind, double goal, const SmpWindow& w) {
    if (part == 0) {
      put_in_order((int)w.count);
      double wt[2];
      weights((int)w.count, wt);
      const double before = scan_mass(wt[0] + wt[1]);
      const double c0 = w.mass + (before + wt[0]), c1 = w.mass + (before + wt[0] + wt[1]);
      const uint32_t i0 = 2 * tid, i1 = i0 + 1, n = w.count;
      uint32_t ahead = block_sum((i0 < n && !crosses(kind, c0, w.ahead + i0 + 1, goal)) +
                                 (i1 < n && !crosses(kind, c1, w.ahead + i1 + 1, goal)));
      ahead = min(ahead, n - 1);
      if (ahead / 2 == tid) {
        const SmpFound f = {list()[ahead], ahead % 2 ? c1 : c0, w.ahead + ahead + 1};
        for (int p = 0; p < parts; p++) *at(&sh.found, p) = f;
      }
    }
    all_sync();
    return sh.found;
  }

  // ---- a window of many tokens: exact sums over 16 bins of its ranks, the one with the crossing becomes the window
  __device__ SmpFound closer(SmpKind kind, double goal, SmpWindow w) {
    while (true) {
      all_sync();  // what was found, or listed, before has been read
      if (w.count <= SMP_LIST) {
        if (tid == 0) sh.n = 0;
        __syncthreads();
        uint64_t* to = at(list(), 0);
        each([&](float y, int id) {
          const uint32_t r = rank_bits(y);
          if (r - w.lo <= w.hi - w.lo) to[w.before + atomicAdd(&sh.n, 1)] = place(r, (uint32_t)id);
        });
        all_sync();
        return among(kind, goal, w);
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
    // 32 threads a bin
    const int b = tid / 32, i = tid % 32;
    double s = cut_mass()[b * SMP_CUTTERS + i] + cut_mass()[b * SMP_CUTTERS + 32 + i];
    const uint32_t n = __reduce_add_sync(0xffffffffu, cut_count()[b * SMP_CUTTERS + i] + cut_count()[b * SMP_CUTTERS + 32 + i]);
    s = warp_sum(s);
    if (i < parts) {
      *at(&to.mass[part][b], i) = s;
      *at(&to.count[part][b], i) = n;
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
    uint32_t own;
    const uint32_t most = load(own);
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
      const uint32_t* all = tell(block_max(first));
      if (part == 0 && tid == 0) {
        for (int q = 0; q < parts; q++) first = max(first, all[q]);
        answer((int)~first, 0.0, 1);
      }
      return;
    }
    top = m;
    inv_t = 1.0 / (double)t;
    rate = inv_t * (64 * 1.44269504088896340736);
    cut_off = 620.f * t;
    floor_ = -FLT_MAX;
    if (min_p >= 1.f) floor_ = m;
    else if (min_p > 0.f) floor_ = fmaxf(floor_, __double2float_ru(top + (double)t * log((double)min_p)));
    if ((k && k <= SMP_TOP) || min_p > 0.f) {
      float from = floor_;
      if (k && k <= SMP_TOP) {
        const uint32_t* all = tell(reached((k + parts - 1) / parts, own));
        uint32_t least = 0xFFFFFFFFu;
        for (int q = 0; q < parts; q++) least = min(least, all[q]);
        from = fmaxf(from, rank_value(max(least, rank_bits(-FLT_MAX))));
      }
      const uint32_t* all;
      const uint32_t n = gather(from, all);
      if (n <= SMP_LIST) {
        uint32_t before = 0;
        for (int q = 0; q < part; q++) before += all[q];
        for (uint32_t i = tid; i < all[part]; i += SMP_THREADS) at(list(), 0)[before + i] = own_list()[i];
        all_sync();
        if (part == 0) finish((int)n, k, p, u);
        return;
      }
    }
    inv_bin = fminf(SMP_BINS / (SMP_SPAN * t), FLT_MAX);
    __syncthreads();
    double mass = 0.0;
    uint32_t kept = 0;
    uint64_t last = 0;      // the last place that is kept, where that is known
    bool known = false;     // whether mass and kept are
    if (k) {
      measure<true>();
      if ((uint32_t)k < __float_as_uint(along()[SMP_BINS - 1])) {
        const SmpFound f = search(SMP_COUNT, (double)k, 0.0, nullptr, nullptr);
        mass = f.mass, kept = f.count, last = f.place;
        known = true;
      }
      all_sync();  // the histogram has been read
    }
    measure<false>();
    if (p < 1.f) {
      const SmpFound f = search(SMP_REACH, (double)p * mass, (double)p, known ? nullptr : &mass, &kept);
      if (f.count < kept) mass = f.mass, kept = f.count, last = f.place;
      known = true;
    }
    SmpFound f = search(SMP_PASS, u * mass, u, known ? nullptr : &mass, &kept);
    if (f.count > kept) f.place = last;  // by rounding alone
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

template <typename In>
cudaError_t launch(IrisSample* a, cudaStream_t stream) {
  const int64_t bytes = (int64_t)a->vocab * (int64_t)sizeof(In) + 16;
  // blocks on a row: as many as leave each 16 KB
  a->parts = 1;
  while (a->parts < SMP_PARTS && bytes > (int64_t)a->parts * 16384) a->parts *= 2;
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

extern "C" cudaError_t iris_launch_sample(IrisSample* a, int f32, cudaStream_t stream) {
  return f32 ? launch<float>(a, stream) : launch<__nv_bfloat16>(a, stream);
}
