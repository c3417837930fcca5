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
// and has the answer.  Else the sums are needed over the whole row: every
// thread adds up its values in 16 bins of its own (no atomics, always the same order), the bin in
// which the number is crossed is cut into 16 again, until SMP_LIST tokens are left
// to be put in order, or tokens of one value, of which the id decides.
// Weights and sums are 64-bit: a token is taken by where a sum of 100000 weights
// ends, and with 32 bits one row in a hundred would take its neighbour.
constexpr int SMP_THREADS = 256, SMP_WARPS = SMP_THREADS / 32, SMP_PARTS = 8, SMP_BINS = 16;
constexpr int SMP_LIST = 512;  // tokens put in order
constexpr int SMP_TOP = 256;   // largest top-k whose tokens are looked for through a bound
constexpr float SMP_SPAN = 24.f;  // (m - x) / t that the first bins cover; the last one holds all that is below

struct SmpSums {  // of the bins, from each block of the cluster
  double mass[SMP_PARTS][SMP_BINS];
  uint32_t count[SMP_PARTS][SMP_BINS];
};

struct SmpFound {
  uint64_t place;
  double mass;     // of the line up to and with it
  uint32_t count;
};

struct SmpShared {
  SmpSums first, next[2];      // next: in turn, so that one round's may be read while the next one's come
  uint32_t one[2][SMP_PARTS];  // a number from each block
  double scan[SMP_WARPS];
  uint32_t iscan[SMP_WARPS];
  SmpFound found;
  uint32_t n;
};

// shared memory besides the row: the bins; a list of places and its order in the same bytes
constexpr int SMP_WORK = SMP_BINS * SMP_THREADS * (8 + 2);
static_assert(SMP_WORK >= 2 * SMP_LIST * 8 + SMP_THREADS * 4, "the lists fit");

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
  float m, floor_;
  double top, inv_t;
  float inv_bin;
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
  }
  __device__ uint8_t* work() const { return smem + (HELD ? a.held_bytes : 0); }
  __device__ double* masses() const { return reinterpret_cast<double*>(work()); }
  __device__ uint16_t* counts() const { return reinterpret_cast<uint16_t*>(work() + SMP_BINS * SMP_THREADS * 8); }
  __device__ uint64_t* list() const { return reinterpret_cast<uint64_t*>(work()); }
  __device__ uint64_t* order() const { return list() + SMP_LIST; }
  __device__ uint32_t* owns() const { return reinterpret_cast<uint32_t*>(order() + SMP_LIST); }

  __device__ void all_sync() const {
    __syncwarp();
    if (parts > 1) iris::cluster_sync();
    else __syncthreads();
  }
  template <typename T>
  __device__ T* at(T* p, int rank) const { return parts > 1 ? iris::cluster_map(p, (uint32_t)rank) : p; }
  // this block's number, by thread 0, to all of them; the numbers of the blocks after the barrier
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
  template <typename F>
  __device__ void each(F f) const {
    for (int v = tid; v < nv; v += SMP_THREADS) {
      float y[VEC];
      vec_values<In>(vec(v), y);
#pragma unroll
      for (int i = 0; i < VEC; i++) f(y[i], first_id(v) + i);
    }
  }
  __device__ double weight(float y) const { return exp(((double)y - top) * inv_t); }

  // over the block, the same in all threads
  __device__ uint32_t block_max(uint32_t v) {
    v = __reduce_max_sync(0xffffffffu, v);
    if (tid % 32 == 0) sh.iscan[tid / 32] = v;
    __syncthreads();
    for (int w = 0; w < SMP_WARPS; w++) v = max(v, sh.iscan[w]);
    __syncthreads();
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
  __device__ double scan_mass(double v) {
    double incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, incl, o);
      if (tid % 32 >= o) incl += y;
    }
    if (tid % 32 == 31) sh.scan[tid / 32] = incl;
    __syncthreads();
    double before = incl - v;
    double ahead = 0;
    for (int w = 0; w < tid / 32; w++) ahead += sh.scan[w];
    __syncthreads();
    return ahead + before;
  }

  // ---- the row, its largest value; each thread's own largest stays in `own`
  __device__ uint32_t load(uint32_t& own) {
    float best = -INFINITY;
    bool nan = false;
    constexpr int FLY = 8;
    for (int b = tid; b < nv; b += FLY * SMP_THREADS) {
      uint4 u[FLY];
#pragma unroll
      for (int j = 0; j < FLY; j++) {
        const int v = b + j * SMP_THREADS;
        u[j] = v < nv ? row_vec(x, first_id(v), a.vocab) : make_uint4(0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u, 0xFF80FF80u);
        if (v >= nv && sizeof(In) == 4) u[j] = make_uint4(0xFF800000u, 0xFF800000u, 0xFF800000u, 0xFF800000u);
      }
#pragma unroll
      for (int j = 0; j < FLY; j++) {
        const int v = b + j * SMP_THREADS;
        if (HELD && v < nv) reinterpret_cast<uint4*>(smem)[v] = u[j];
        float y[VEC];
        vec_values<In>(u[j], y);
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          nan |= y[i] != y[i];
          best = fmaxf(best, y[i]);
        }
      }
    }
    own = rank_bits(nan ? NAN : best);
    const uint32_t* all = tell(block_max(own));
    uint32_t r = 0;
    for (int p = 0; p < parts; p++) r = max(r, all[p]);
    return r;
  }

  // ---- the tokens from `from` on, each block's in its own list; how many there are in the whole row (each block's in `all`)
  __device__ uint32_t gather(float from, const uint32_t*& all) {
    if (tid == 0) sh.n = 0;
    __syncthreads();
    each([&](float y, int id) {
      if (y >= from) {
        if (*(volatile uint32_t*)&sh.n > SMP_LIST) return;  // too many already
        const uint32_t n = atomicAdd(&sh.n, 1);
        if (n < SMP_LIST) order()[n] = place(rank_bits(y), (uint32_t)id);
      }
    });
    __syncthreads();
    all = tell(sh.n);
    uint32_t n = 0;
    for (int p = 0; p < parts; p++) n += min(all[p], SMP_LIST + 1);
    return n;
  }

  // ---- by the first block: list()[0, n) in order; a sum before each pair of tokens of this thread, their weights
  __device__ void put_in_order(int n, double w[2], double& before) {
    __syncthreads();
    uint64_t mine[2];
    int ahead[2] = {0, 0};
#pragma unroll
    for (int j = 0; j < 2; j++) mine[j] = tid + j * SMP_THREADS < n ? list()[tid + j * SMP_THREADS] : ~0ull;
#pragma unroll 4
    for (int i = 0; i < n; i++) {
      const uint64_t p = list()[i];
      ahead[0] += p > mine[0], ahead[1] += p > mine[1];
    }
#pragma unroll
    for (int j = 0; j < 2; j++)
      if (tid + j * SMP_THREADS < n) order()[ahead[j]] = mine[j];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 2; j++) w[j] = 2 * tid + j < n ? weight(rank_value((uint32_t)(order()[2 * tid + j] >> 32))) : 0.0;
    before = scan_mass(w[0] + w[1]);
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
    double w[2], before;
    if (k) {
      put_in_order(n, w, before);
      n = min(n, k);
      if (2 * tid >= n) w[0] = 0.0;
      if (2 * tid + 1 >= n) w[1] = 0.0;
      before = scan_mass(w[0] + w[1]);
    } else {
      put_in_order(n, w, before);
    }
    const double c0 = before + w[0], c1 = c0 + w[1];
    __shared__ double sums[SMP_LIST];
    sums[2 * tid] = c0, sums[2 * tid + 1] = c1;
    __syncthreads();
    const double mass = sums[n - 1];
    uint32_t kept = n;
    if (p < 1.f) {
      const double goal = (double)p * mass;
      uint32_t some;
      scan_count((2 * tid < n && before < goal) + (2 * tid + 1 < n && c0 < goal), &some);
      kept = max(some, 1u);
    }
    const double m_kept = sums[kept - 1], goal = u * m_kept;
    uint32_t pick, heavy;
    scan_count((2 * tid < kept && c0 <= goal) + (2 * tid + 1 < kept && c1 <= goal), &pick);
    scan_count((2 * tid < kept && w[0] > 0.0) + (2 * tid + 1 < kept && w[1] > 0.0), &heavy);
    pick = min(pick, heavy - 1);  // the first one weighs 1
    if (tid == 0) answer((int)~(uint32_t)order()[pick], logprob(order()[pick], m_kept), kept);
  }

  // ---- sums over bins of the tokens with ranks lo .. hi, in every block
  template <typename Bin>
  __device__ void bins(SmpSums& to, uint32_t lo, uint32_t hi, Bin bin) {
    double* mass = masses() + tid;
    uint16_t* count = counts() + tid;
#pragma unroll
    for (int b = 0; b < SMP_BINS; b++) mass[b * SMP_THREADS] = 0.0, count[b * SMP_THREADS] = 0;
    each([&](float y, int) {
      if (rank_bits(y) - lo <= hi - lo) {
        const int b = bin(y) * SMP_THREADS;
        mass[b] += weight(y);
        count[b]++;
      }
    });
    __syncthreads();
    // 16 threads a bin
    const int b = tid / 16, i = tid % 16;
    double s = 0.0;
    uint32_t n = 0;
    for (int j = i; j < SMP_THREADS; j += 16) s += masses()[b * SMP_THREADS + j], n += counts()[b * SMP_THREADS + j];
#pragma unroll
    for (int o = 8; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o), n += __shfl_xor_sync(0xffffffffu, n, o);
    if (i < parts) {
      *at(&to.mass[part][b], i) = s;
      *at(&to.count[part][b], i) = n;
    }
    all_sync();
  }

  __device__ static bool crosses(SmpKind kind, double mass, uint32_t count, double goal) {
    return kind == SMP_COUNT ? (double)count >= goal : kind == SMP_REACH ? mass >= goal : mass > goal;
  }
  // the bin of the window in which the number is crossed (rounding: else the last with a token), into w; its number
  __device__ int choose(const SmpSums& s, SmpKind kind, double goal, SmpWindow& w) const {
    int last = 0;
    SmpWindow at = w, hit = w;
    for (int b = 0; b < SMP_BINS; b++) {
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
  __device__ int first_bin(float y) const { return min(SMP_BINS - 1, (int)((m - y) * inv_bin)); }

  // ---- the token at which the count or the sum crosses `goal`
  __device__ SmpFound search(SmpKind kind, double goal) {
    SmpWindow w;
    w.mass = 0.0;
    w.ahead = 0;
    const int b1 = choose(sh.first, kind, goal, w);
    {
      // the ranks of this bin: the bins are monotone in the value
      const uint32_t least = rank_bits(floor_), most = rank_bits(m);
      uint32_t lo = least, hi = most;
      while (lo < hi) {  // smallest rank whose bin is b1 or an earlier one
        const uint32_t mid = lo + (hi - lo) / 2;
        if (first_bin(rank_value(mid)) <= b1) hi = mid;
        else lo = mid + 1;
      }
      w.lo = lo;
      hi = most;
      while (lo < hi) {  // largest whose bin is b1
        const uint32_t mid = hi - (hi - lo) / 2;
        if (first_bin(rank_value(mid)) >= b1) lo = mid;
        else hi = mid - 1;
      }
      w.hi = lo;
    }
    for (uint32_t round = 0;; round++) {
      if (w.count <= SMP_LIST) {
        __syncthreads();
        if (tid == 0) sh.n = 0;
        all_sync();  // the first block is done with its bins
        uint64_t* to = at(list(), 0);
        each([&](float y, int id) {
          const uint32_t r = rank_bits(y);
          if (r - w.lo <= w.hi - w.lo) to[w.before + atomicAdd(&sh.n, 1)] = place(r, (uint32_t)id);
        });
        all_sync();
        if (part == 0) {
          double wt[2], before;
          put_in_order((int)w.count, wt, before);
          const double c0 = w.mass + (before + wt[0]), c1 = w.mass + (before + wt[0] + wt[1]);
          const uint32_t i0 = 2 * tid, i1 = i0 + 1, n = w.count;
          uint32_t ahead;
          scan_count((i0 < n && !crosses(kind, c0, w.ahead + i0 + 1, goal)) + (i1 < n && !crosses(kind, c1, w.ahead + i1 + 1, goal)),
                     &ahead);
          ahead = min(ahead, n - 1);
          if (ahead / 2 == tid) {
            const SmpFound f = {order()[ahead], ahead % 2 ? c1 : c0, w.ahead + ahead + 1};
            for (int p = 0; p < parts; p++) *at(&sh.found, p) = f;
          }
        }
        all_sync();
        return sh.found;
      }
      if (w.lo == w.hi) {  // one value: the id decides
        all_sync();        // an earlier answer has been read
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
      const uint32_t range = w.hi - w.lo, hi = w.hi, shift = max(0, 28 - __clz(range));
      SmpSums& s = sh.next[turn++ & 1];
      bins(s, w.lo, w.hi, [&](float y) { return (int)((hi - rank_bits(y)) >> shift); });
      const int b = choose(s, kind, goal, w);
      w.hi = hi - ((uint32_t)b << shift);
      const uint64_t below = ((uint64_t)(b + 1) << shift) - 1;
      w.lo = below < hi - w.lo ? hi - (uint32_t)below : w.lo;
    }
  }

  __device__ void run() {
    const int row = blockIdx.x / parts;
    const float t = a.temperature ? a.temperature[row] : 1.f, p = a.top_p ? a.top_p[row] : 1.f;
    const float min_p = a.min_p ? a.min_p[row] : 0.f;
    int k = a.top_k ? a.top_k[row] : 0;
    if (k < 0 || k >= a.vocab) k = 0;
    double u = a.uniform[row];
    u = u > 0.0 ? fmin(u, 0x1.fffffffffffffp-1) : 0.0;
    uint32_t own;
    const uint32_t most = load(own);
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
    floor_ = -FLT_MAX;
    if (min_p >= 1.f) floor_ = m;
    else if (min_p > 0.f) floor_ = fmaxf(floor_, __double2float_ru(top + (double)t * log((double)min_p)));
    if ((k && k <= SMP_TOP) || min_p > 0.f) {
      float from = floor_;
      const int each_k = (k + parts - 1) / parts;
      if (k && k <= SMP_TOP) {
        // a value that each_k of this block's tokens reach, 0 if there are not so many threads with one
        owns()[tid] = own;
        __syncthreads();
        int ahead = 0;
        for (int i = 0; i < SMP_THREADS; i++) ahead += owns()[i] > own || (owns()[i] == own && i < tid);
        const uint32_t* all = tell(block_max(ahead >= each_k - 1 ? own : 0u));
        uint32_t least = 0xFFFFFFFFu;
        for (int q = 0; q < parts; q++) least = min(least, all[q]);
        from = fmaxf(from, rank_value(max(least, rank_bits(-FLT_MAX))));
      }
      const uint32_t* all;
      const uint32_t n = gather(from, all);
      if (n <= SMP_LIST) {
        uint32_t before = 0;
        for (int q = 0; q < part; q++) before += all[q];
        for (uint32_t i = tid; i < all[part]; i += SMP_THREADS) at(list(), 0)[before + i] = order()[i];
        all_sync();
        if (part == 0) finish((int)n, k, p, u);
        return;
      }
    }
    inv_bin = SMP_BINS / (SMP_SPAN * t);
    __syncthreads();
    bins(sh.first, rank_bits(floor_), most, [&](float y) { return first_bin(y); });
    double mass = 0.0;
    uint32_t kept = 0;
    for (int b = 0; b < SMP_BINS; b++)
      for (int q = 0; q < parts; q++) mass += sh.first.mass[q][b], kept += sh.first.count[q][b];
    uint64_t last = 0;  // the last place that is kept, where that is known
    if (k && (uint32_t)k < kept) {
      const SmpFound f = search(SMP_COUNT, (double)k);
      mass = f.mass, kept = f.count, last = f.place;
    }
    if (p < 1.f) {
      const SmpFound f = search(SMP_REACH, (double)p * mass);
      if (f.count < kept) mass = f.mass, kept = f.count, last = f.place;
    }
    SmpFound f = search(SMP_PASS, u * mass);
    if (f.count > kept) f.place = last;  // by rounding alone
    if (part == 0 && tid == 0) answer((int)~(uint32_t)f.place, logprob(f.place, mass), kept);
  }
};

template <typename In, bool HELD>
__global__ void __launch_bounds__(SMP_THREADS) sample_kernel(const __grid_constant__ IrisSample a) {
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
