// The pick of a token by chance: temperature, top-k, min-p and top-p, with the random numbers given.
//
// With M = max x (NaN counts as -inf) and w_i = exp((x_i - M) / temperature), the set drawn from is
//   K1 = the top_k largest x, of equal ones those of the lowest index;
//   K2 = the i of K1 with (x_i - M) / temperature >= ln(min_p);
//   K3 = of K2 in descending order (equal ones by index) the shortest run whose w add up to top_p of K2's,
// and the token is the first i of K3, by index, at which the sum of w reaches beyond u times K3's sum.
//
// All three cuts are thresholds on x plus a count of equal values taken by index, so no row is sorted, only a short
// list. A cluster of CTAs holds a row in shared memory and reads it from memory once. After its maximum:
//  - top-k (with or without the others): the j-th largest of the maxima of 256 groups of threads is at most
//    the j-th largest value, so that the values from it on hold the top j, and are hardly more. They go on a list in
//    one CTA, which sorts it, cuts it by prefix sums, sorts the rest by index and finds the token by prefix sums
//    again. The same with min-p alone: its threshold is known.
//  - top-p alone: a histogram of counts over 4096 equal parts of the value range gives the sums to a fraction of
//    a percent (and for a top-k of thousands the part of its cut), and with that the few parts in which the cut
//    must lie. One pass over the row then takes the exact sum of all w and, by stretch (a warp's run of indexes),
//    of those above these parts, whose own values go on the list; there the cut is found, then the stretch of the
//    token, and its warp finds the token in it.
//  - no filter: the stretches' sums, and one stretch again.
//  - whatever does not fit the list (thousands of equal values, top-p behind a top-k of thousands): histograms of counts and
//    exact sums, level by level, down to a single value.
//
// The sums decide between whole numbers: where a sum passes a border, another token follows. w is therefore
// computed in 64 bits and kept as a whole number of 2^-44ths, so that sums are exact in any order (and the
// result does not depend on the order of atomics). A weight is off by less than 0.6 of these (half of one by its
// rounding, 0.08 by the exponential), a sum of n of them by n times that.
//
// Bound by latency: the row's bytes are a few us at most, and the pipe of 64-bit arithmetic is busy for a tenth of the time where
// all weights are needed. By clock64, us of a row from the dependency wait on: one row of 151936, top-k 50 and top-p: the
// pass for the maximum 1.2, the search for the cut 1.4 to 1.8, the cluster 0.6, the pass for the list 1.0, collecting it 1.4, sorts and
// pick 4.5. 32 rows by top-p: maximum 2.5, cluster 1, counts 3.7, their sums over the cluster 2.2, the parts of the cut 2.4, the exact
// pass 9.7, collecting 1.4, sorts 2.8 (a list of 1024: 11), the token 1 or less. 64 rows in 32 bits: maximum 5.6, cut 1 to 2, the pass
// for the list from L2 6, collecting 1, sorts 2.7 to 6.5 (and where min-p lets more than 1024 in, the way by parts after that: 36).
#include "common.cuh"

#include <cfloat>

namespace {

constexpr int SM_THREADS = 1024;               // at most (see sample_go)
constexpr int SM_PARTS = 4096;                 // equal parts of the value range, SM_PER of them to a factor e of w
constexpr int SM_PER = 128;
constexpr int SM_GROUPS = 256;                 // groups of threads whose maxima bound the top-k cut
constexpr int SM_CTAS = 8;                     // CTAs of a cluster at most
constexpr int SM_FRACTION = 44;                // bits of a weight
constexpr int SM_MAX_ROWS = 1 << 24;
constexpr int SM_MAX_VOCAB = 1 << 19;          // (sums of so many stay below 2^63)
constexpr int SM_MOST = 1 << 17;               // values that a CTA gets at most (their 15-bit pieces add up in 32 bits)

typedef unsigned long long u64;

struct SampleArgs {
  const void* x;
  long long stride;
  const float* u;
  q_sampling_t s;
  int64_t* tokens;
  float* logprobs;
  int vocab, seg, resident;                    // seg: values of a warp's stretch, a multiple of a vector's
};

struct SampleShared {
  // slots that the CTAs of the cluster write into one another
  float top[SM_CTAS], cut[SM_CTAS], bottom[SM_CTAS];
  u64 sum[2][SM_CTAS];                         // (two of each: a round may begin while another CTA reads the last one's)
  unsigned count[2][SM_CTAS];
  u64 whole[SM_CTAS];                          // sums of all w (CTA 0)
  unsigned listed[2];                          // entries of the list (CTA 0), of the first and the second try
  int done;
  u64 last, start, goal, total;                // what the stretch of the token needs (see finish)
  int stretch;
  // this CTA's own
  unsigned base, found;
  u64 red[32];
  unsigned cred[32];
  u64 warp_sum[32];
  unsigned warp_equal[32];
  u64 above;
  unsigned inside;
  float group[SM_GROUPS];
  float part_sum[32], part_squares[32];
  double power[16];                            // 2^(j / 16)
  u64 list[SM_THREADS];                           // ~key << 32 | index, then index << 32 | rank
  u64 spare[SM_THREADS];                          // this CTA's entries before they are collected; scratch; weights
  u64 stretches[SM_CTAS * 32];                 // sums of all stretches (CTA 0)
  union {
    struct { unsigned count[SM_PARTS], all[SM_PARTS]; } parts;
    float parts_upto[SM_PARTS];                // (over the counts, once they are in registers)
    struct { unsigned count[SM_THREADS], mass[3][SM_THREADS], all_count[SM_THREADS]; u64 all_mass[SM_THREADS]; } level;
  };
};

constexpr size_t SM_SMEM_MAX = 227 * 1024;     // of a CTA: the above and the part of the row that it keeps, if that fits
constexpr size_t SM_FIXED = (sizeof(SampleShared) + 15) / 16 * 16;

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(shared_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void put32(const void* p, int rank, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at_rank(p, rank)), "r"(v) : "memory");
}
__device__ __forceinline__ void put64(const void* p, int rank, u64 v) {
  asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at_rank(p, rank)), "l"(v) : "memory");
}
__device__ __forceinline__ uint32_t get32(const void* p, int rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Whole numbers in the order of the values.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t b = __float_as_uint(x);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ ((key >> 31) ? 0x80000000u : 0xffffffffu));
}
// w = exp(z) in 2^-44ths, z = (x - M) / temperature <= 0, as 2^(n / 16) times exp(L r), L = ln(2) / 16, |r| <= 1 / 2;
// 2^(n / 16) from a table of sixteen. The Taylor series cut behind r^5 leaves up to E = (L / 2)^6 / 720 = 1.4e-13, 2.5
// units and always to one side. Its next term, E (2 r)^6, is therefore replaced by what differs from it by E T6(2 r) / 32, of
// the Chebyshev polynomial T6(y) = 32 y^6 - 48 y^4 + 18 y^2 - 1 (economization of a power series, C. Lanczos): a change of
// three coefficients, at most 4.5e-15 off to either side, 0.08 units.
struct Weigher {
  double top, rate;                            // M, 16 log2(e) / temperature
  float topf, floor;                           // M, and the (x - M) / 2 from which on w rounds to 0
  const double* power;
  __device__ __forceinline__ void start(float most, float temperature) {
    top = (double)most;
    topf = most;
    floor = -16.f * temperature;               // exp(-32) < 2^-46
  }
  // of a finite M and -64 <= z (anything else gives some number; no branches: the chains of several values run side by
  // side)
  __device__ __forceinline__ u64 plain(float x) const {
    constexpr double L = 0.69314718055994530942 / 16, H = L / 2, E = H * H * H * H * H * H / 720;
    const double t = ((double)x - top) * rate;
    const double big = 6755399441055744.0;                   // 1.5 * 2^52: adding it rounds to a whole number,
    const double sum = t + big;                              // which is then in the low bits
    const int n = __double2loint(sum);
    const double r = t - (sum - big);
    double p = L * L * L * L * L / 120;
    p = fma(p, r, L * L * L * L / 24 + E * (16 * 48.0 / 32));
    p = fma(p, r, L * L * L / 6);
    p = fma(p, r, L * L / 2 - E * (4 * 18.0 / 32));
    p = fma(p, r, L);
    p = fma(p, r, 1.0 + E / 32);
    const double q = power[n & 15];
    const double scale = __hiloint2double(__double2hiint(q) + (((n >> 4) + SM_FRACTION) << 20), __double2loint(q));
    // to a whole number: the sum with 2^52 has it in its low bits
    return (u64)__double_as_longlong(fma(p, scale, 4503599627370496.0)) & ((1ull << 52) - 1);
  }
  __device__ __forceinline__ u64 operator()(float x) const {
    const u64 w = plain(x);
    // (also of infinities; a whole difference can leave 32 bits where temperatures of 1e37 and more make it matter)
    return x == topf ? 1ull << SM_FRACTION : fmaf(0.5f, x, -0.5f * topf) > floor ? w : 0;
  }
};

// A 16-byte vector of logits: cleaned (NaN is -inf; -0 is 0: they compare equal, so their keys have to be), its
// largest value, and its values.
template <typename T> struct Vec;
template <> struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ __nv_bfloat162 two(uint32_t w) { return *reinterpret_cast<__nv_bfloat162*>(&w); }
  static __device__ __forceinline__ uint32_t bits(__nv_bfloat162 v) { return *reinterpret_cast<uint32_t*>(&v); }
  static __device__ __forceinline__ uint32_t clean(uint32_t w) {
    const __nv_bfloat162 zero = two(0u), lowest = two(0xff80ff80u);
    return bits(__hmax2(__hadd2_rn(two(w), zero), lowest));            // (the maximum with a NaN is the other)
  }
  static __device__ __forceinline__ uint4 clean(uint4 r) { return make_uint4(clean(r.x), clean(r.y), clean(r.z), clean(r.w)); }
  static __device__ __forceinline__ float most(uint4 r) {
    const uint32_t m = bits(__hmax2(__hmax2(two(r.x), two(r.y)), __hmax2(two(r.z), two(r.w))));
    return fmaxf(bf_lo(m), bf_hi(m));
  }
  static __device__ __forceinline__ void unpack(uint4 r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(w[i]); v[2 * i + 1] = bf_hi(w[i]); }
  }
  static __device__ __forceinline__ uint4 some(const bf16* p, int i, int n) {        // values i .. i + 7 of n; -inf outside
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      w[k] = 0;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int j = i + 2 * k + e;
        w[k] |= (j >= 0 && j < n ? (uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(p) + j) : 0xff80u) << (16 * e);
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ uint32_t clean(uint32_t w) { return __float_as_uint(fmaxf(__uint_as_float(w) + 0.f, -INFINITY)); }
  static __device__ __forceinline__ uint4 clean(uint4 r) { return make_uint4(clean(r.x), clean(r.y), clean(r.z), clean(r.w)); }
  static __device__ __forceinline__ float most(uint4 r) {
    return fmaxf(fmaxf(__uint_as_float(r.x), __uint_as_float(r.y)), fmaxf(__uint_as_float(r.z), __uint_as_float(r.w)));
  }
  static __device__ __forceinline__ void unpack(uint4 r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 some(const float* p, int i, int n) {
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) w[k] = i + k >= 0 && i + k < n ? __float_as_uint(__ldcg(p + i + k)) : 0xff800000u;
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
template <int WARPS>
__device__ __forceinline__ u64 block_add(u64 v, SampleShared& sh) {
  v = warp_add(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  const int lane = threadIdx.x & 31;
  return warp_add(lane < WARPS ? sh.red[lane] : 0);
}
// Inclusive prefix sums over the block's threads.
__device__ __forceinline__ void block_scan(u64& v, SampleShared& sh) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  __syncthreads();
  if (lane == 31) sh.red[warp] = v;
  __syncthreads();
  v += warp_add(lane < warp ? sh.red[lane] : 0);
}

// The same and a sort over the first `size` threads (a power of two, 32 .. SM_THREADS), whose warps alone call.
__device__ __forceinline__ void some_sync(int size) {
  if (size == 32) __syncwarp();
  else asm volatile("bar.sync 1, %0;" ::"r"(size) : "memory");
}
__device__ __forceinline__ u64 some_scan(u64 v, int size, SampleShared& sh, u64& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 t = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += t;
  }
  if (size == 32) {
    total = __shfl_sync(0xffffffffu, v, 31);
    return v;
  }
  some_sync(size);
  if (lane == 31) sh.red[warp] = v;
  some_sync(size);
  const u64 w = lane * 32 < size ? sh.red[lane] : 0;
  total = warp_add(w);
  return v + warp_add(lane < warp ? w : 0);
}
// Ascending bitonic sort, one number per thread.
__device__ __forceinline__ u64 some_sort(u64 v, int size, u64* scratch) {
  const int t = threadIdx.x;
  for (int k = 2; k <= size; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      u64 o;
      if (j >= 32) {
        some_sync(size);
        scratch[t] = v;
        some_sync(size);
        o = scratch[t ^ j];
      } else {
        o = __shfl_xor_sync(0xffffffffu, v, j);
      }
      const bool low = ((t & j) == 0) == ((t & k) == 0);     // keeps the smaller of the pair
      v = (o < v) == low ? o : v;
    }
  }
  return v;
}

// THREADS: also the most entries of the list and the bins of a histogram level.
template <typename T, int THREADS>
__global__ void __launch_bounds__(THREADS, 1)
k_sample(const SampleArgs a) {
  constexpr int WARPS = THREADS / 32;
  constexpr int VEC = Vec<T>::N;
  extern __shared__ __align__(16) unsigned char smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  uint4* slice = reinterpret_cast<uint4*>(smem + SM_FIXED);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int row = blockIdx.x / ctas;
  if (tid == 0) { sh.listed[0] = 0; sh.listed[1] = 0; sh.done = 0; sh.found = 0; }
  if (tid < 16) sh.power[tid] = exp2(tid / 16.0);
  // (waited for before the first store into another CTA's memory)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();

  // ---- this warp's stretch of the row. Vectors lie on 16-byte boundaries of memory: the row begins `head`
  // values into its first one, what lies outside it counts as -inf.
  const T* x = reinterpret_cast<const T*>(a.x) + (long long)row * a.stride;
  const int head = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int begin = (int)(rank * WARPS + warp) * a.seg - head;      // index of the stretch's first value
  uint4* mine = slice + (size_t)warp * a.seg / VEC;
  auto raw = [&](int o) {                      // vector at value o of the stretch from memory
    const int i = begin + o;
    return i >= 0 && i + VEC <= a.vocab ? __ldcg(reinterpret_cast<const uint4*>(x + i)) : Vec<T>::some(x, i, a.vocab);
  };
  auto vector = [&](int o) { return a.resident ? mine[o / VEC] : Vec<T>::clean(raw(o)); };     // ... cleaned
  constexpr int STEP = 32 * VEC;
  constexpr int SIDE = 4;                      // weights computed side by side

  // ---- maximum; the row's settings while the first values are on their way
  constexpr int AHEAD = 4;
  uint4 first[AHEAD];
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) {
    const int o = lane * VEC + q * STEP;
    first[q] = o < a.seg ? raw(o) : make_uint4(0, 0, 0, 0);
  }
  float temperature = a.s.d_temperature ? __ldcg(a.s.d_temperature + row) : a.s.temperature;
  int top_k = a.s.d_top_k ? __ldcg(a.s.d_top_k + row) : a.s.top_k;
  const float top_p = a.s.d_top_p ? __ldcg(a.s.d_top_p + row) : a.s.top_p;
  float min_p = a.s.d_min_p ? __ldcg(a.s.d_min_p + row) : a.s.min_p;
  const float u = __ldcg(a.u + row);
  const bool by_p = top_p > 0.f && top_p < 1.f;                      // (NaN: off)
  if (!(temperature > 0.f) || top_p <= 0.f) top_k = 1;               // the largest alone
  if (!(temperature > 0.f)) temperature = 1.f;
  if (top_k <= 0 || top_k >= a.vocab) top_k = 0;
  const bool by_min = min_p > 0.f && temperature < INFINITY;         // (NaN: off; at an infinite temperature all weigh the same)
  min_p = fminf(min_p, 1.f);
  Weigher weigh;
  weigh.rate = 16 * 1.4426950408889634074 / (double)temperature;
  weigh.power = sh.power;
  const double min_z = by_min ? (double)temperature * log((double)min_p) : -INFINITY;

  float best = -INFINITY;
#pragma unroll
  for (int q = 0; q < AHEAD; ++q) {
    const int o = lane * VEC + q * STEP;
    if (o < a.seg) {
      const uint4 r = Vec<T>::clean(first[q]);
      if (a.resident) mine[o / VEC] = r;
      best = fmaxf(best, Vec<T>::most(r));
    }
  }
  for (int o0 = lane * VEC + AHEAD * STEP; o0 < a.seg; o0 += AHEAD * STEP) {
    uint4 r[AHEAD];
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) r[q] = o0 + q * STEP < a.seg ? raw(o0 + q * STEP) : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int q = 0; q < AHEAD; ++q) {
      const int o = o0 + q * STEP;
      if (o < a.seg) {
        r[q] = Vec<T>::clean(r[q]);
        if (a.resident) mine[o / VEC] = r[q];
        best = fmaxf(best, Vec<T>::most(r[q]));
      }
    }
  }
#pragma unroll
  for (int o = 1; o < THREADS / SM_GROUPS; o <<= 1) best = fmaxf(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (tid % (THREADS / SM_GROUPS) == 0) sh.group[tid / (THREADS / SM_GROUPS)] = best;
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  // how many of this CTA's groups have to have a maximum from the cut on, so that all CTAs' make up the top k
  const int want = (top_k + (int)ctas - 1) / (int)ctas;
  const bool bounded = top_k > 0 && want <= SM_GROUPS * 15 / 16;
  if (warp == 0) {
    constexpr int EACH = SM_GROUPS / 32;
    float most = -INFINITY;
    uint32_t k[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      const float g = sh.group[lane + 32 * i];
      most = fmaxf(most, g);
      k[i] = key_of(g);
    }
    most = warp_max(most);
    float cut = -INFINITY;
    if (bounded) {
      uint32_t lo = key_of(-INFINITY), hi = key_of(most);              // (at lo all groups count)
      while (lo < hi) {
        const uint32_t mid = lo + (hi - lo) / 2 + ((hi - lo) & 1u);
        int n = 0;
#pragma unroll
        for (int i = 0; i < EACH; ++i) n += __popc(__ballot_sync(0xffffffffu, k[i] >= mid));
        if (n >= want) {
          lo = mid;
          if (n <= want + (want >> 3)) break;  // near enough
        } else {
          hi = mid - 1;
        }
      }
      cut = value_of(lo);
    }
    if (lane < (int)ctas) {
      put32(&sh.top[rank], lane, __float_as_uint(most));
      put32(&sh.cut[rank], lane, __float_as_uint(cut));
    }
  }
  cluster_sync();
  float top = sh.top[0], cut = sh.cut[0];
  for (int c = 1; c < (int)ctas; ++c) { top = fmaxf(top, sh.top[c]); cut = fminf(cut, sh.cut[c]); }
  if (top == -INFINITY) {                      // no token can be drawn
    if (rank == 0 && tid == 0) { a.tokens[row] = -1; a.logprobs[row] = -INFINITY; }
    return;
  }
  weigh.start(top, temperature);
  const double least = (double)top + min_z;    // x from which min-p lets a value in
  const float least_f = by_min ? __double2float_ru(least) : -INFINITY;      // (the next number of 32 bits: the same for x)
  auto let_in = [&](float v) { return v > -INFINITY && v >= least_f; };

  // the token at which the sums pass this much of `total`: the last that weighs anything for u of 1 and more
  auto goal_of = [&](u64 total) {
    const u64 g = __double2ull_rd((u > 0.f ? (double)u : 0.0) * (double)total);
    return g < total ? g : total - 1;
  };
  auto answer = [&](int index, float v, u64 total) {
    a.tokens[row] = index;
    const double z = v == top ? 0.0 : ((double)v - (double)top) / (double)temperature;
    a.logprobs[row] = (float)(z - log((double)total * (1.0 / (1ull << SM_FRACTION))));
  };
  // sums over the cluster's CTAs, of a number of each thread's
  int round = 0;
  auto cluster_add = [&](u64 v, unsigned c, u64& all, unsigned& count) {
    v = block_add<WARPS>(v, sh);
    const u64 n = block_add<WARPS>((u64)c, sh);
    if (tid < (int)ctas) {
      put64(&sh.sum[round & 1][rank], tid, v);
      put32(&sh.count[round & 1][rank], tid, (unsigned)n);
    }
    cluster_sync();
    all = 0;
    count = 0;
    for (int k = 0; k < (int)ctas; ++k) { all += sh.sum[round & 1][k]; count += sh.count[round & 1][k]; }
    ++round;
  };
  auto push = [&](float v, int index) {        // onto this CTA's part of the list
    const unsigned p = atomicAdd(&sh.found, 1u);
    if (p < THREADS) sh.spare[p] = (u64)(~key_of(v)) << 32 | (unsigned)index;
  };
  auto collect = [&](int which) {              // the parts into CTA 0's list
    __syncthreads();
    const unsigned found = sh.found;
    if (tid == 0) {
      unsigned b;
      asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(b) : "r"(at_rank(&sh.listed[which], 0)), "r"(found) : "memory");
      sh.base = b;
    }
    __syncthreads();
    if (tid == 0) sh.found = 0;                // (every thread has read it)
    if (tid < (int)min(found, (unsigned)THREADS) && sh.base + tid < THREADS) put64(&sh.list[sh.base + tid], 0, sh.spare[tid]);
    cluster_sync();
  };
  auto list_size = [](unsigned n) { int s = 32; while (s < (int)n) s <<= 1; return s; };

  // ---- the list of the top k, or of what min-p lets in
  if (bounded || by_min) {
    const float from = fmaxf(cut, least_f);
    for (int o = lane * VEC; o < a.seg; o += STEP) {
      const uint4 r = vector(o);
      if (Vec<T>::most(r) >= from) {
        float v[VEC];
        Vec<T>::unpack(r, v);
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (v[j] >= from && v[j] > -INFINITY) push(v[j], begin + o + j);
      }
    }
    collect(0);
    if (rank == 0) {
      const unsigned n = sh.listed[0];
      const int size = list_size(n);
      const bool done = n <= THREADS;          // (it holds the top k, or all that min-p lets in, and those among them)
      if (done && tid < size) {
        const u64 entry = some_sort(tid < (int)n ? sh.list[tid] : ~0ull, size, sh.spare);
        const float v = value_of(~(uint32_t)(entry >> 32));
        bool in = tid < (int)n && (top_k == 0 || tid < top_k) && let_in(v);
        const u64 w = in ? weigh(v) : 0;
        u64 total;
        if (by_p) {
          const u64 upto = some_scan(w, size, sh, total);
          in = in && (double)(upto - w) < (double)top_p * (double)total;
        }
        // the set is a run at the head of the list; by index, each with its rank to find its weight
        some_sync(size);
        sh.spare[tid] = in ? w : 0;
        const u64 s = some_sort(in ? (entry & 0xffffffffull) << 32 | (unsigned)tid : ~0ull, size, sh.list);
        const int place = s == ~0ull ? tid : (int)(s & 0xffffffffull);
        some_sync(size);
        const u64 ws = s == ~0ull ? 0 : sh.spare[place];
        const u64 sums = some_scan(ws, size, sh, total);
        const u64 goal = goal_of(total);
        if (sums > goal && sums - ws <= goal) sh.base = (unsigned)place;
        some_sync(size);
        if (tid == (int)sh.base) answer((int)(entry & 0xffffffffull), v, total);
      }
      if (warp == 0 && lane < (int)ctas) put32(&sh.done, lane, done ? 1u : 0u);
    }
    cluster_sync();
    if (sh.done) return;
  }

  // ---- top-p or a large top-k alone (min-p first, where it let too many in)
  // (parts_per is finite, and values whose difference from the largest leaves 32 bits weigh nothing)
  if ((by_p ? top_k == 0 : top_k > 0) && top < INFINITY && temperature > 1e-36f && temperature < 1e30f) {
    const float parts_per = (float)SM_PER / temperature;
    auto part_of = [&](float v) { return v == top ? 0 : min(SM_PARTS - 1, (int)((top - v) * parts_per)); };
    for (int i = tid; i < SM_PARTS; i += THREADS) sh.parts.count[i] = 0;
    __syncthreads();
    for (int o = lane * VEC; o < a.seg; o += STEP) {
      float v[VEC];
      Vec<T>::unpack(vector(o), v);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (let_in(v[j])) atomicAdd(&sh.parts.count[part_of(v[j])], 1u);
    }
    // every CTA adds its share of the parts over all CTAs and hands the sums to all
    cluster_sync();
    const int per = SM_PARTS / (int)ctas;
    for (int i = tid; i < per; i += THREADS) {
      const int part = (int)rank * per + i;
      unsigned c[SM_CTAS];
#pragma unroll
      for (int r = 0; r < SM_CTAS; ++r) c[r] = r < (int)ctas ? get32(&sh.parts.count[part], r) : 0;
#pragma unroll
      for (int r = 1; r < SM_CTAS; ++r) c[0] += c[r];
#pragma unroll
      for (int r = 0; r < SM_CTAS; ++r)
        if (r < (int)ctas) put32(&sh.parts.all[part], r, c[0]);
    }
    cluster_sync();
    // the parts up to each: their number of values (top-k), or what they weigh, about
    constexpr int EACH = SM_PARTS / THREADS;
    float own[EACH], upto = 0.f, squares = 0.f;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      const float w = by_p ? exp2f(-(EACH * tid + e + 0.5f) * (1.44269504f / SM_PER)) : 1.f;
      own[e] = (float)sh.parts.all[EACH * tid + e] * w;        // (numbers up to 2^19 are exact)
      upto += own[e];
      squares += own[e] * own[e];
    }
    float mine_upto = upto;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const float t = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += t;
    }
    squares = warp_sum(squares);
    if (lane == 31) { sh.part_sum[warp] = upto; sh.part_squares[warp] = squares; }
    __syncthreads();                           // (also: the counts are in registers, the sums may lie over them)
    const float about = warp_sum(lane < WARPS ? sh.part_sum[lane] : 0.f);
    squares = warp_sum(lane < WARPS ? sh.part_squares[lane] : 0.f);
    upto += warp_sum(lane < warp ? sh.part_sum[lane] : 0.f) - mine_upto;
#pragma unroll
    for (int e = 0; e < EACH; ++e) {
      upto += own[e];
      sh.parts_upto[EACH * tid + e] = upto;
    }
    __syncthreads();
    auto reached = [&](float goal) {           // first part with at least so much up to it
      int lo = 0, hi = SM_PARTS - 1;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sh.parts_upto[mid] >= goal) hi = mid; else lo = mid + 1;
      }
      return lo;
    };
    // A part's values lie anywhere in it: its sum is off by 1 / SM_PER / sqrt(12) of itself in the root mean square, all
    // sums by that times the root of the parts' squares. Four times as much either side; where that should not
    // do, the exact sums say so. (Counts are exact.)
    int part0, part1;
    unsigned wanted = 0;                       // top-k: values of the part that belong to the set
    if (by_p) {
      const float margin = 1e-5f * about + 4 * 0.2887f / SM_PER * sqrtf(squares);
      part0 = reached(top_p * about - margin);
      part1 = reached(top_p * about + margin);
    } else {
      part0 = part1 = reached((float)top_k);
      wanted = (unsigned)top_k - (part0 > 0 ? (unsigned)sh.parts_upto[part0 - 1] : 0u);
    }
    // values in these parts: on the list if they fit it
    auto values_in = [&](int from, int to) {
      unsigned n = 0;
      for (int i = from + lane; i <= to; i += 32) n += sh.parts.all[i];
      return __reduce_add_sync(0xffffffffu, n);
    };
    bool fits = values_in(part0, part1) <= THREADS;
    const float from_part = (float)part0;
    const float to_part = !fits ? from_part : part1 == SM_PARTS - 1 ? INFINITY : (float)(part1 + 1);
    // The smallest value that may have a weight: the sum's rounding is a value's own, at most twice as far below M. (With it
    // weights need no checks of their ends: 32 x 151936 bf16, top-p, with them / so, 40.2 / 38.2 us.)
    const float alive_from = fmaxf(fmaxf(top + 2.f * weigh.floor, -FLT_MAX), least_f);
    u64 sum = 0, above = 0;
    for (int o = lane * VEC; o < a.seg; o += STEP) {
      float v[VEC];
      Vec<T>::unpack(vector(o), v);
#pragma unroll
      for (int j0 = 0; j0 < VEC; j0 += SIDE) {
        u64 w[SIDE];
        bool listed = false;
#pragma unroll
        for (int j = 0; j < SIDE; ++j) w[j] = weigh.plain(v[j0 + j]);
#pragma unroll
        for (int j = 0; j < SIDE; ++j) {
          const float at = (top - v[j0 + j]) * parts_per;      // (part_of is its whole part)
          const bool alive = v[j0 + j] >= alive_from, over = at < from_part;
          if (alive) sum += w[j];
          if (alive && over) above += w[j];
          listed |= !over && at < to_part;
        }
        if (listed) {
#pragma unroll
          for (int j = 0; j < SIDE; ++j) {
            const float at = (top - v[j0 + j]) * parts_per;
            if (let_in(v[j0 + j]) && at >= from_part && at < to_part) push(v[j0 + j], begin + o + j0 + j);
          }
        }
      }
    }
    if (!fits && by_p && part1 - part0 < 32) {
      // Too many: with the exact sum above them, the parts' own bounds leave fewer in doubt.
      u64 all, over;
      unsigned unused;
      cluster_add(sum, 0, all, unused);
      cluster_add(above, 0, over, unused);
      const double share = (double)top_p * (double)all, unit = (double)(1ull << SM_FRACTION);
      // lane i: what the parts up to part0 + i weigh at most and at least
      const int part = part0 + lane;
      const double c = part <= part1 ? (double)sh.parts.all[part] * unit : 0.0;
      double most = c * exp(-(double)part / SM_PER), fewest = c * exp(-(part + 1.0) / SM_PER);
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double m = __shfl_up_sync(0xffffffffu, most, o), f = __shfl_up_sync(0xffffffffu, fewest, o);
        if (lane >= o) { most += m; fewest += f; }
      }
      const unsigned may = __ballot_sync(0xffffffffu, (double)over + most * (1 + 1e-5) >= share);
      const unsigned must = __ballot_sync(0xffffffffu, (double)over + fewest * (1 - 1e-5) >= share);
      const int from = part0 + (may ? __ffs(may) - 1 : 31), to = must ? part0 + __ffs(must) - 1 : part1;
      fits = from <= to && values_in(from, min(to, part1)) <= THREADS;
      if (fits) {
        for (int o = lane * VEC; o < a.seg; o += STEP) {
          float v[VEC];
          Vec<T>::unpack(vector(o), v);
#pragma unroll
          for (int j = 0; j < VEC; ++j) {
            if (!let_in(v[j])) continue;
            const int part = part_of(v[j]);
            if (part < part0 || part > to) continue;
            if (part < from) above += weigh(v[j]);
            else push(v[j], begin + o + j);
          }
        }
      }
    }
    above = warp_add(above);
    if (lane == 0) put64(&sh.stretches[rank * WARPS + warp], 0, above);
    sum = block_add<WARPS>(sum, sh);
    if (tid == 0) put64(&sh.whole[rank], 0, sum);
    collect(1);
    if (rank == 0) {
      const unsigned n = sh.listed[1];
      const int size = list_size(n);
      bool done = n <= THREADS && n > 0;
      if (done && tid < size) {
        u64 all = 0, above = 0;
        for (int c = 0; c < (int)ctas; ++c) all += sh.whole[c];
        for (int i = lane; i < (int)ctas * WARPS; i += 32) above += sh.stretches[i];
        above = warp_add(above);
        const double share = (double)top_p * (double)all;
        const u64 entry = some_sort(tid < (int)n ? sh.list[tid] : ~0ull, size, sh.spare);
        const float v = value_of(~(uint32_t)(entry >> 32));
        const u64 w = tid < (int)n ? weigh(v) : 0;
        u64 listed;
        const u64 upto = some_scan(w, size, sh, listed);
        if (by_p) done = (double)above < share && (double)(above + listed) >= share;
        if (done) {
          const bool in = tid < (int)n && (by_p ? (double)(above + upto - w) < share : tid < (int)wanted);
          // the set: all from its last value on (of equal ones up to its index)
          const bool next_in = tid + 1 < (int)n && (by_p ? (double)(above + upto) < share : tid + 1 < (int)wanted);
          if (in && !next_in) { sh.last = entry; sh.total = above + upto; }
          if (in) atomicAdd(&sh.stretches[((unsigned)(entry & 0xffffffffull) + head) / a.seg], w);
          some_sync(size);
          if (warp == 0) {
            // the stretch of the token: prefix sums, a lane taking several stretches
            const u64 total = sh.total, goal = goal_of(total);
            const int stretches = (int)ctas * WARPS, each = (stretches + 31) / 32;
            u64 mine_sum = 0;
            for (int i = 0; i < each; ++i)
              if (lane * each + i < stretches) mine_sum += sh.stretches[lane * each + i];
            u64 s = mine_sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const u64 t = __shfl_up_sync(0xffffffffu, s, o);
              if (lane >= o) s += t;
            }
            if (s > goal && s - mine_sum <= goal) {
              u64 at = s - mine_sum;
              int c = lane * each;
              while (at + sh.stretches[c] <= goal) at += sh.stretches[c++];
              const int owner = c / WARPS;
              put64(&sh.last, owner, sh.last);
              put64(&sh.start, owner, at);
              put64(&sh.goal, owner, goal);
              put64(&sh.total, owner, total);
              for (int r = 0; r < (int)ctas; ++r) put32(&sh.stretch, r, (uint32_t)c);
            }
          }
        }
      }
      if (warp == 0 && lane < (int)ctas) put32(&sh.done, lane, done ? 1u : 0u);
    }
    cluster_sync();
    if (sh.done) {
      if (sh.stretch == (int)(rank * WARPS + warp)) {
        const u64 last = sh.last, goal = sh.goal, total = sh.total;
        u64 s = sh.start;
        for (int o0 = 0; o0 < a.seg; o0 += STEP) {
          const int o = o0 + lane * VEC;
          float v[VEC];
          if (o < a.seg) {
            Vec<T>::unpack(vector(o), v);
          } else {
#pragma unroll
            for (int j = 0; j < VEC; ++j) v[j] = -INFINITY;
          }
          auto weight = [&](int j) {
            const u64 entry = (u64)(~key_of(v[j])) << 32 | (unsigned)(begin + o + j);
            return v[j] > -INFINITY && entry <= last ? weigh(v[j]) : 0ull;
          };
          u64 ls = 0;
#pragma unroll
          for (int j = 0; j < VEC; ++j) ls += weight(j);
          u64 is = ls;
#pragma unroll
          for (int q = 1; q < 32; q <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, is, q);
            if (lane >= q) is += t;
          }
          const unsigned here = __ballot_sync(0xffffffffu, s + is > goal);
          if (here != 0) {
            if (lane == __ffs(here) - 1) {
              u64 at = s + is - ls;
#pragma unroll
              for (int j = 0; j < VEC; ++j) {
                const u64 w = weight(j);
                if (at <= goal && at + w > goal) answer(begin + o + j, v[j], total);
                at += w;
              }
            }
            break;
          }
          s += __shfl_sync(0xffffffffu, is, 31);
        }
      }
      return;
    }
  }

  // ---- thresholds: the set is the values of a key above `edge`, and the first `ties` of key `edge`, as far as
  // min-p lets them in
  uint32_t edge = key_of(-INFINITY);
  unsigned ties = 0;
  auto above_edge = [&](float v) { return key_of(v) > edge && v >= least_f; };
  auto values = [&](int o, float (&v)[VEC]) {  // -inf past the stretch
    if (o < a.seg) {
      Vec<T>::unpack(vector(o), v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = -INFINITY;
    }
  };
  if (top_k > 0 || by_p) {
    float bottom = INFINITY;
    u64 all = 0;
    unsigned candidates = 0, mine_in = 0;
    for (int o = lane * VEC; o < a.seg; o += 32 * VEC) {
      float v[VEC];
      values(o, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j)
        if (above_edge(v[j])) { bottom = fminf(bottom, v[j]); ++mine_in; }
    }
    bottom = -warp_max(-bottom);
    __syncthreads();
    if (lane == 0) sh.cred[warp] = __float_as_uint(bottom);
    __syncthreads();
    bottom = -warp_max(lane < WARPS ? -__uint_as_float(sh.cred[lane]) : -INFINITY);
    if (tid < (int)ctas) put32(&sh.bottom[rank], tid, __float_as_uint(bottom));
    cluster_add(0, mine_in, all, candidates);
    bottom = sh.bottom[0];
    for (int c = 1; c < (int)ctas; ++c) bottom = fminf(bottom, sh.bottom[c]);

    // Finds the key at which a count (`by_count`: the first `need` values) or a sum (`share`) of the values above the
    // edge is reached, the count and sum above that key, and how many values have it. The first level cuts the
    // values into equal parts, the next ones a part's keys.
    const float scale = (float)(THREADS - 1) / (top - bottom);          // (inf or 0 apart: handled as one part)
    const bool whole = !(scale > 0.f && scale < INFINITY);
    auto part_of = [&](float v) { return whole ? 0 : min(THREADS - 1, (int)((top - v) * scale)); };
    auto descend = [&](bool by_count, u64 need, double share, uint32_t& key, u64& above, unsigned& inside) {
      int part = -1, shift = 0;
      uint32_t low = key_of(bottom), high = key_of(top);
      above = 0;
      for (bool first = !whole;;) {
        if (!first) {
          shift = 0;
          while (((high - low) >> shift) >= THREADS) ++shift;
        }
        sh.level.count[tid] = 0;
#pragma unroll
        for (int e = 0; e < 3; ++e) sh.level.mass[e][tid] = 0;
        __syncthreads();
        for (int o = lane * VEC; o < a.seg; o += 32 * VEC) {
          float v[VEC];
          values(o, v);
#pragma unroll 1
          for (int j = 0; j < VEC; ++j) {
            if (!above_edge(v[j])) continue;
            int bin;
            if (first) {
              bin = part_of(v[j]);
            } else {
              const uint32_t k = key_of(v[j]);
              if (k < low || k > high || (part >= 0 && part_of(v[j]) != part)) continue;
              bin = (int)((high - k) >> shift);
            }
            atomicAdd(&sh.level.count[bin], 1u);
            if (!by_count) {
              // 15 bits at a time: up to 2^17 values of a CTA add up in 32 (64-bit atomics on shared memory
              // take 0.7 to 2.3 cycles each, 32-bit ones 0.1 to 0.2)
              const u64 w = weigh(v[j]);
#pragma unroll
              for (int e = 0; e < 3; ++e) atomicAdd(&sh.level.mass[e][bin], (unsigned)(w >> (15 * e)) & 0x7fffu);
            }
          }
        }
        cluster_sync();
        // every CTA adds its share of the bins over all CTAs and hands the sums to all
        const int per = THREADS / (int)ctas;
        if (tid < per) {
          const int bin = (int)rank * per + tid;
          unsigned c = 0;
          u64 m = 0;
          for (int r = 0; r < (int)ctas; ++r) {
            c += get32(&sh.level.count[bin], r);
#pragma unroll
            for (int e = 0; e < 3; ++e) m += (u64)get32(&sh.level.mass[e][bin], r) << (15 * e);
          }
          for (int r = 0; r < (int)ctas; ++r) { put32(&sh.level.all_count[bin], r, c); put64(&sh.level.all_mass[bin], r, m); }
        }
        cluster_sync();
        const u64 own = by_count ? sh.level.all_count[tid] : sh.level.all_mass[tid];
        u64 upto = own;
        block_scan(upto, sh);
        const bool short_of = by_count ? above + upto < need : (double)(above + upto) < share;
        const int bin = min(__syncthreads_count(short_of), THREADS - 1);
        if (tid == bin) { sh.above = above + upto - own; sh.inside = sh.level.all_count[tid]; }
        __syncthreads();
        above = sh.above;
        inside = sh.inside;
        if (first) {
          first = false;
          part = bin;
          // the keys of a part, with room for the rounding of part_of
          const double width = 1.0 / (double)scale;
          const float to = __double2float_ru((double)top - bin * width * (1.0 - 1e-6));
          const float at = __double2float_rd((double)top - (bin + 1) * width * (1.0 + 1e-6));
          if (bin > 0) high = min(high, key_of(to));
          if (bin < THREADS - 1) low = max(low, key_of(at));
        } else {
          high -= (uint32_t)bin << shift;
          if (shift == 0) { key = high; return; }
          low = max(low, high - ((1u << shift) - 1u));
        }
      }
    };
    uint32_t key;
    u64 above;
    unsigned inside;
    if (top_k > 0 && candidates > (unsigned)top_k) {
      descend(true, (u64)top_k, 0.0, key, above, inside);
      edge = key;
      ties = (unsigned)((u64)top_k - above);
    }
    if (by_p) {
      u64 sum = 0;
      for (int o = lane * VEC; o < a.seg; o += 32 * VEC) {
        float v[VEC];
        values(o, v);
#pragma unroll 4
        for (int j = 0; j < VEC; ++j)
          if (above_edge(v[j])) sum += weigh(v[j]);
      }
      u64 strict;
      cluster_add(sum, 0, strict, candidates);
      u64 w = ties ? weigh(value_of(edge)) : 0;
      const double share = (double)top_p * (double)(strict + ties * w);
      above = strict;
      inside = ties;
      if ((double)strict >= share) {
        descend(false, 0, share, key, above, inside);
        edge = key;
        w = weigh(value_of(edge));
      }
      // the fewest of the equal values that reach the share
      unsigned j = w ? (unsigned)fmin((double)inside, fmax(1.0, ceil((share - (double)above) / (double)w))) : inside;
      while (j > 1 && (double)(above + (j - 1) * w) >= share) --j;
      while (j < inside && (double)(above + j * w) < share) ++j;
      ties = j;
    }
  }

  // ---- the token: sums of the warps' stretches, of the CTAs, then one warp goes through its stretch
  const u64 tie_weight = ties ? weigh(value_of(edge)) : 0;
  auto weight_of = [&](float v) {
    const u64 w = weigh(v);
    return above_edge(v) ? w : 0ull;
  };
  u64 sum = 0;
  unsigned equal = 0;
  for (int o = lane * VEC; o < a.seg; o += 32 * VEC) {
    float v[VEC];
    values(o, v);
#pragma unroll
    for (int j0 = 0; j0 < VEC; j0 += SIDE) {
      u64 w[SIDE];
#pragma unroll
      for (int j = 0; j < SIDE; ++j) w[j] = weigh(v[j0 + j]);
#pragma unroll
      for (int j = 0; j < SIDE; ++j) sum += above_edge(v[j0 + j]) ? w[j] : 0;
    }
    if (ties) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) equal += key_of(v[j]) == edge ? 1u : 0u;
    }
  }
  sum = warp_add(sum);
  equal = __reduce_add_sync(0xffffffffu, equal);
  __syncthreads();
  if (lane == 0) { sh.warp_sum[warp] = sum; sh.warp_equal[warp] = equal; }
  u64 total;
  unsigned equals;
  cluster_add(lane == 0 ? sum : 0, lane == 0 ? equal : 0, total, equals);
  const int last = (round - 1) & 1;
  u64 before = 0;
  unsigned equal_before = 0;
  for (int c = 0; c < (int)rank; ++c) { before += sh.sum[last][c]; equal_before += sh.count[last][c]; }
  total += (u64)min(ties, equals) * tie_weight;
  const u64 goal = goal_of(total);
  // inclusive sums over the warps, the same in every warp
  u64 ws = lane < WARPS ? sh.warp_sum[lane] : 0;
  unsigned we = lane < WARPS ? sh.warp_equal[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const u64 ts = __shfl_up_sync(0xffffffffu, ws, o);
    const unsigned te = __shfl_up_sync(0xffffffffu, we, o);
    if (lane >= o) { ws += ts; we += te; }
  }
  auto upto = [&](u64 s, unsigned e) { return s + (u64)min(ties, e) * tie_weight; };
  const unsigned past = __ballot_sync(0xffffffffu, upto(before + ws, equal_before + we) > goal);
  if (upto(before, equal_before) <= goal && past != 0 && warp == __ffs(past) - 1) {
    u64 s = before + __shfl_sync(0xffffffffu, ws, warp) - sum;
    unsigned e = equal_before + __shfl_sync(0xffffffffu, we, warp) - equal;
    for (int o0 = 0; o0 < a.seg; o0 += 32 * VEC) {
      const int o = o0 + lane * VEC;
      float v[VEC];
      values(o, v);
      u64 ls = 0;
      unsigned le = 0;
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        ls += weight_of(v[j]);
        le += ties && key_of(v[j]) == edge ? 1u : 0u;
      }
      u64 is = ls;
      unsigned ie = le;
#pragma unroll
      for (int q = 1; q < 32; q <<= 1) {
        const u64 ts = __shfl_up_sync(0xffffffffu, is, q);
        const unsigned te = __shfl_up_sync(0xffffffffu, ie, q);
        if (lane >= q) { is += ts; ie += te; }
      }
      const unsigned here = __ballot_sync(0xffffffffu, upto(s + is, e + ie) > goal);
      if (here != 0) {
        if (lane == __ffs(here) - 1) {
          u64 rs = s + is - ls;
          unsigned re = e + ie - le;
#pragma unroll 1
          for (int j = 0; j < VEC; ++j) {
            rs += weight_of(v[j]);
            re += ties && key_of(v[j]) == edge ? 1u : 0u;
            if (upto(rs, re) > goal) {
              answer(begin + o + j, v[j], total);
              break;
            }
          }
        }
        break;
      }
      s += __shfl_sync(0xffffffffu, is, 31);
      e += __shfl_sync(0xffffffffu, ie, 31);
    }
  }
}

// (The limit is the kernel's, not the launch's: one that never moves cannot be lowered by another shape's launch, or by
// one of another thread.)
template <typename T, int THREADS>
cudaError_t sample_room() {
  static size_t done[64] = {0};
  return q_ensure_smem(k_sample<T, THREADS>, SM_SMEM_MAX, done);
}

// Clusters of a size that the current device holds at once, a CTA to an SM (a cluster stays inside one GPC, so this is
// less than the SMs would allow), asked once per device.
int sample_resident(int ctas) {
  static int cached[64][SM_CTAS + 1];
  const int dev = q_device_index();
  if (dev < 0) return 132 / ctas;
  int& n = cached[dev][ctas];
  if (n == 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas);
    cfg.blockDim = dim3(SM_THREADS);
    cfg.dynamicSmemBytes = SM_SMEM_MAX;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    int got = 0;
    cudaError_t e = sample_room<bf16, SM_THREADS>();
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&got, k_sample<bf16, SM_THREADS>, &cfg);
    if (e != cudaSuccess) { cudaGetLastError(); got = 132 / ctas; }
    n = got > 0 ? got : -1;
  }
  return n;
}

// Values of a warp's stretch: whole vectors; a row that is not aligned may begin anywhere in its first one.
template <typename T>
int sample_seg(int vocab, bool aligned, int ctas, int threads) {
  constexpr int VEC = Vec<T>::N;
  const int vectors = ctas * (threads / 32) * VEC;
  return (vocab + (aligned ? 0 : VEC - 1) + vectors - 1) / vectors * VEC;
}

// How a row is dealt out; most values that a CTA gets.
struct SamplePlan { int ctas, threads, seg; };
template <typename T>
int sample_most(int vocab, bool aligned, int ctas, int threads) {
  const int room = sample_seg<T>(vocab, aligned, ctas, threads) * (threads / 32);
  return room < vocab ? room : vocab;
}

template <typename T>
SamplePlan sample_plan(int rows, int vocab, bool aligned) {
  // CTAs of a row: as many as leave all rows' clusters resident, while a CTA has a few thousand values. Not more where
  // a CTA's part then does not fit its shared memory: 64 rows of 151936 in 32 bits with 4 CTAs in two waves / 2
  // CTAs that read the row from L2 in each pass, us: top-k 33 / 23, top-p 71 / 62.
  SamplePlan p;
  p.ctas = 1;
  while (p.ctas < SM_CTAS && vocab / (p.ctas * 2) >= 3000 && rows <= sample_resident(p.ctas * 2)) p.ctas *= 2;
  // (Stretches are rounded up to whole vectors: a CTA may get more than its share of the row. Aligned rows of 2^17, 2^18 and
  // 2^19 just do with as few CTAs: 64 rows of 2^18 in 16 bits with 2 CTAs / 4 in two waves, us: top-k 20 / 31, min-p 17 / 23,
  // but top-p 276 / 194.)
  while (sample_most<T>(vocab, aligned, p.ctas, SM_THREADS) > SM_MOST) p.ctas *= 2;
  // Fewer threads meet faster, more hide the latency of the 64-bit arithmetic. 512 / 1024 threads, us: 1 row of 151936
  // (19000 a CTA) top-p 22.7 / 25.1, 7 of 32003 top-k 10.7 / 11.4; 32 of 151936 (38000 a CTA) top-p 35.5 / 34.1.
  p.threads = vocab / p.ctas < 24000 ? 512 : SM_THREADS;
  p.seg = sample_seg<T>(vocab, aligned, p.ctas, p.threads);
  return p;
}

template <typename T, int THREADS>
int sample_launch(SampleArgs a, int rows, int ctas, cudaStream_t stream) {
  const size_t slice = (size_t)a.seg * (THREADS / 32) * sizeof(T);
  a.resident = SM_FIXED + slice <= SM_SMEM_MAX;      // (otherwise every pass reads the row again, from L2)
  const size_t bytes = SM_FIXED + (a.resident ? slice : 0);
  Q_CHECK_CUDA((sample_room<T, THREADS>()));
  Q_CHECK_CUDA(q_launch_cluster(k_sample<T, THREADS>, dim3((unsigned)rows * ctas), dim3(THREADS), bytes, stream, (unsigned)ctas, a));
  return Q_OK;
}

template <typename T>
int sample_go(SampleArgs a, int rows, cudaStream_t stream) {
  const bool aligned = (uintptr_t)a.x % 16 == 0 && (rows == 1 || a.stride % Vec<T>::N == 0);
  const SamplePlan p = sample_plan<T>(rows, a.vocab, aligned);
  a.seg = p.seg;
  return p.threads == 512 ? sample_launch<T, 512>(a, rows, p.ctas, stream) : sample_launch<T, 1024>(a, rows, p.ctas, stream);
}

}  // namespace

extern "C" int q_sample_tokens_plan(int fp32, int rows, int vocab, int aligned, int* ctas, int* values) {
  const char* who = "q_sample_tokens_plan";
  Q_CHECK_ARG(ctas && values, "%s: null pointer", who);
  Q_CHECK_ARG(rows >= 1 && rows <= SM_MAX_ROWS && vocab >= 1 && vocab <= SM_MAX_VOCAB,
              "%s: %d rows of %d values (1 to 2^24 rows of up to %d)", who, rows, vocab, SM_MAX_VOCAB);
  const bool al = aligned != 0;
  const SamplePlan p = fp32 ? sample_plan<float>(rows, vocab, al) : sample_plan<bf16>(rows, vocab, al);
  *ctas = p.ctas;
  *values = fp32 ? sample_most<float>(vocab, al, p.ctas, p.threads) : sample_most<bf16>(vocab, al, p.ctas, p.threads);
  return Q_OK;
}

extern "C" int q_sample_tokens(const void* d_logits, int fp32, int64_t row_stride, const float* d_uniform,
                               const q_sampling_t* sampling, int64_t* d_tokens, float* d_logprobs, int rows, int vocab,
                               void* stream) {
  const char* who = "q_sample_tokens";
  Q_CHECK_ARG(d_logits && d_uniform && sampling && d_tokens && d_logprobs, "%s: null pointer", who);
  Q_CHECK_ARG(rows >= 1 && rows <= SM_MAX_ROWS && vocab >= 1 && vocab <= SM_MAX_VOCAB,
              "%s: %d rows of %d values (1 to 2^24 rows of up to %d)", who, rows, vocab, SM_MAX_VOCAB);
  Q_CHECK_ARG(row_stride >= 0, "%s: negative row stride", who);
  Q_CHECK_ARG(sampling->d_temperature || sampling->temperature >= 0.f, "%s: temperature is negative or NaN", who);
  Q_CHECK_ARG((sampling->d_top_p || sampling->top_p == sampling->top_p) && (sampling->d_min_p || sampling->min_p == sampling->min_p),
              "%s: top_p or min_p is NaN", who);
  Q_CHECK_ALIGN(d_logits, (fp32 ? 4 : 2), who); Q_CHECK_ALIGN(d_uniform, 4, who);
  Q_CHECK_ALIGN(d_tokens, 8, who); Q_CHECK_ALIGN(d_logprobs, 4, who);
  Q_CHECK_ALIGN(sampling->d_temperature, 4, who); Q_CHECK_ALIGN(sampling->d_top_k, 4, who);
  Q_CHECK_ALIGN(sampling->d_top_p, 4, who); Q_CHECK_ALIGN(sampling->d_min_p, 4, who);
  SampleArgs a = {};
  a.x = d_logits;
  a.stride = row_stride;
  a.u = d_uniform;
  a.s = *sampling;
  a.tokens = d_tokens;
  a.logprobs = d_logprobs;
  a.vocab = vocab;
  return fp32 ? sample_go<float>(a, rows, (cudaStream_t)stream) : sample_go<bf16>(a, rows, (cudaStream_t)stream);
}
