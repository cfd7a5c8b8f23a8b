// The pick of a token by chance: temperature, top-k, min-p and top-p, with the random numbers given.
//
// With M = max x (NaN counts as -inf) and w_i = exp((x_i - M) / temperature), the set drawn from is
//   K1 = the top_k largest x, of equal ones those of the lowest index;
//   K2 = the i of K1 with (x_i - M) / temperature >= ln(min_p);
//   K3 = of K2 in descending order (equal ones by index) the shortest run whose w add up to top_p of K2's,
// and the token is the first i of K3, by index, at which the sum of w reaches beyond u times K3's sum.
//
// All three cuts are thresholds on x plus a count of equal values taken by index, so nothing is sorted but a
// short list. A cluster of CTAs holds a row in shared memory and reads it from memory once:
//   1. the row's maximum, and a lower bound of the cut: the j-th largest of the threads' maxima is at most
//      the j-th largest value, so that all values from it on hold the top j, and are hardly more than that;
//   2. those values go on a list in one CTA (and where top-p has no top-k or min-p before it, the sum of all w
//      is taken). If the list decides - it is short enough, and holds the whole set - it is sorted there, cut by
//      prefix sums, sorted by index, and the token is found by prefix sums again;
//   3. otherwise (a nucleus of thousands, no filter at all) the thresholds come from histograms of counts
//      and sums, level by level, and the token from the sums of the warps' stretches of the row.
//
// The sums decide between whole numbers: where a sum passes a border, another token follows. w is therefore
// computed in 64 bits and kept as a whole number of 2^-44ths, so that sums are exact in any order (and the
// result does not depend on the order of atomics). The error of a sum of n of them is below n 2^-45.
//
// Bound by latency for few rows (a chain of cluster barriers), by the 64-bit exponentials where all of them are
// needed; the row's bytes are a few us at most.
#include "common.cuh"

namespace {

constexpr int SM_THREADS = 1024, SM_WARPS = 32;
constexpr int SM_LIST = 1024;                  // entries of the sorted list: one per thread
constexpr int SM_BINS = 1024;                  // bins of a histogram level: one per thread
constexpr int SM_CTAS = 8;                     // CTAs of a cluster at most
constexpr int SM_FRACTION = 44;                // bits of a weight
constexpr int SM_MAX_VOCAB = 1 << 19;          // (sums of so many stay below 2^63)
constexpr size_t SM_SLICE = 184 * 1024;        // most bytes of a row's part that a CTA keeps

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
  unsigned listed;                             // entries of the list (CTA 0)
  int done;
  // this CTA's own
  unsigned base, found;
  u64 red[SM_WARPS];
  unsigned cred[SM_WARPS];
  u64 warp_sum[SM_WARPS];
  unsigned warp_equal[SM_WARPS];
  u64 total, above;
  unsigned inside;
  int place;
  u64 list[SM_LIST];                           // ~key << 32 | index, then index << 32 | rank
  u64 spare[SM_LIST];                          // this CTA's entries before they are collected; scratch; weights
  unsigned bin_count[SM_BINS];                 // a histogram level
  u64 bin_mass[SM_BINS];
  unsigned all_count[SM_BINS];                 // ... over the cluster
  u64 all_mass[SM_BINS];
};

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
__device__ __forceinline__ u64 get64(const void* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at_rank(p, rank)) : "memory");
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
// A logit as it takes part: NaN is -inf, -0 is 0 (they compare equal, so their keys have to be).
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }

// w = exp(z) in 2^-44ths, z = (x - M) / temperature <= 0: 2^n times the Taylor series of exp in 64 bits, of which
// eleven terms leave 7e-13 at |r| <= ln(2) / 2.
struct Weigher {
  double top, rate;                            // M, log2(e) / temperature
  float topf;
  __device__ __forceinline__ u64 operator()(float x) const {
    if (x == topf) return 1ull << SM_FRACTION;
    const double t = ((double)x - top) * rate;
    if (!(t > -(double)(SM_FRACTION + 2))) return 0;         // (also -inf, and 0 * inf)
    const double big = 6755399441055744.0;                   // 1.5 * 2^52: adding it rounds to a whole number
    const double n = (t + big) - big;
    const double r = (t - n) * 0.69314718055994530942;
    double p = 1.0 / 3628800;
    p = fma(p, r, 1.0 / 362880);
    p = fma(p, r, 1.0 / 40320);
    p = fma(p, r, 1.0 / 5040);
    p = fma(p, r, 1.0 / 720);
    p = fma(p, r, 1.0 / 120);
    p = fma(p, r, 1.0 / 24);
    p = fma(p, r, 1.0 / 6);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    // times 2^(n + 44), then to a whole number: the sum with 2^52 has it in its low bits
    const double scale = __hiloint2double((1023 + SM_FRACTION + (int)n) << 20, 0);
    return (u64)__double_as_longlong(fma(p, scale, 4503599627370496.0)) & ((1ull << 52) - 1);
  }
};

template <typename T> struct Vec;
template <> struct Vec<bf16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(uint4 r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { v[2 * i] = bf_lo(w[i]); v[2 * i + 1] = bf_hi(w[i]); }
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[8]) {        // (values that were bf16)
    return make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
  }
  static __device__ __forceinline__ float load(const bf16* p) {
    return __uint_as_float((uint32_t)__ldcg(reinterpret_cast<const unsigned short*>(p)) << 16);
  }
};
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(uint4 r, float (&v)[4]) {
    v[0] = __uint_as_float(r.x); v[1] = __uint_as_float(r.y); v[2] = __uint_as_float(r.z); v[3] = __uint_as_float(r.w);
  }
  static __device__ __forceinline__ uint4 pack(const float (&v)[4]) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  }
  static __device__ __forceinline__ float load(const float* p) { return __ldcg(p); }
};

__device__ __forceinline__ u64 warp_add(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 block_add(u64 v, SampleShared& sh) {
  v = warp_add(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh.red[threadIdx.x >> 5] = v;
  __syncthreads();
  return warp_add(sh.red[threadIdx.x & 31]);
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

// Ascending bitonic sort of the first `n` (a power of two, 32..1024) numbers, one per thread; all threads call.
__device__ __forceinline__ u64 block_sort(u64 v, int n, u64* scratch) {
  const int t = threadIdx.x;
  for (int k = 2; k <= n; k <<= 1) {
    for (int j = k >> 1; j > 0; j >>= 1) {
      const bool low = ((t & j) == 0) == ((t & k) == 0);     // keeps the smaller of the pair
      u64 o;
      if (j >= 32) {
        __syncthreads();
        if (t < n) scratch[t] = v;
        __syncthreads();
        o = t < n ? scratch[t ^ j] : v;
      } else {
        o = __shfl_xor_sync(0xffffffffu, v, j);
      }
      v = (o < v) == low ? o : v;
    }
  }
  return v;
}

template <typename T>
__global__ void __launch_bounds__(SM_THREADS, 1)
k_sample(const SampleArgs a) {
  constexpr int VEC = Vec<T>::N;
  extern __shared__ __align__(16) unsigned char smem[];
  SampleShared& sh = *reinterpret_cast<SampleShared*>(smem);
  uint4* slice = reinterpret_cast<uint4*>(smem + (sizeof(SampleShared) + 15) / 16 * 16);

  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank, ctas;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(ctas));
  const int row = blockIdx.x / ctas;
  if (tid == 0) { sh.listed = 0; sh.done = 0; sh.found = 0; }
  // (waited for before the first store into another CTA's memory)
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  pdl_wait();
  pdl_launch_dependents();

  // ---- the row's settings
  float temperature = a.s.d_temperature ? __ldcg(a.s.d_temperature + row) : a.s.temperature;
  int top_k = a.s.d_top_k ? __ldcg(a.s.d_top_k + row) : a.s.top_k;
  const float top_p = a.s.d_top_p ? __ldcg(a.s.d_top_p + row) : a.s.top_p;
  float min_p = a.s.d_min_p ? __ldcg(a.s.d_min_p + row) : a.s.min_p;
  const float u = __ldcg(a.u + row);
  const bool by_p = top_p > 0.f && top_p < 1.f;                      // (NaN: off)
  if (!(temperature > 0.f) || top_p <= 0.f) top_k = 1;               // the largest alone
  if (!(temperature > 0.f)) temperature = 1.f;
  if (top_k <= 0 || top_k >= a.vocab) top_k = 0;
  if (!(min_p > 0.f)) min_p = 0.f;
  min_p = fminf(min_p, 1.f);

  // ---- this warp's stretch of the row. Vectors lie on 16-byte boundaries of memory: the row begins `head`
  // values into its first one, what lies outside it counts as -inf.
  const T* x = reinterpret_cast<const T*>(a.x) + (long long)row * a.stride;
  const int head = (int)(((uintptr_t)x & 15) / sizeof(T));
  const int begin = (int)(rank * SM_WARPS + warp) * a.seg - head;      // index of the stretch's first value
  uint4* mine = slice + (size_t)warp * a.seg / VEC;
  auto fetch = [&](int o, float (&v)[VEC]) {   // values o .. o + VEC - 1 of the stretch from memory
    const int i = begin + o;
    if (i >= 0 && i + VEC <= a.vocab) {
      Vec<T>::unpack(__ldcg(reinterpret_cast<const uint4*>(x + i)), v);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = i + j >= 0 && i + j < a.vocab ? Vec<T>::load(x + i + j) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < VEC; ++j) v[j] = clean(v[j]);
  };
  auto values = [&](int o, float (&v)[VEC]) {  // ... or from this CTA's copy; -inf past the stretch
    if (o >= a.seg) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) v[j] = -INFINITY;
    } else if (a.resident) {
      Vec<T>::unpack(mine[o / VEC], v);
    } else {
      fetch(o, v);
    }
  };

  // ---- 1. maximum
  float best = -INFINITY;
  for (int o0 = lane * VEC; o0 < a.seg; o0 += 4 * 32 * VEC) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int o = o0 + q * 32 * VEC;
      if (o < a.seg) {
        float v[VEC];
        fetch(o, v);
        if (a.resident) mine[o / VEC] = Vec<T>::pack(v);
#pragma unroll
        for (int j = 0; j < VEC; ++j) best = fmaxf(best, v[j]);
      }
    }
  }
  float block_best = warp_max(best);
  if (lane == 0) sh.cred[warp] = __float_as_uint(block_best);
  __syncthreads();
  block_best = warp_max(__uint_as_float(sh.cred[lane]));

  // ---- the CTA's lower bound of the cut: at least `want` of its threads have a maximum from it on
  const int ranks = top_k > 0 ? top_k : by_p ? SM_LIST / 3 : 0;
  const int want = (ranks + (int)ctas - 1) / (int)ctas;
  float cut = -INFINITY;
  if (want > 0 && want <= SM_THREADS / 2) {
    uint32_t lo = key_of(-INFINITY), hi = key_of(block_best);          // (at lo all threads count)
    const uint32_t own = key_of(best);
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2 + ((hi - lo) & 1u);
      const int n = __syncthreads_count(own >= mid);
      if (n >= want) {
        lo = mid;
        if (n <= want + (want >> 2)) break;    // near enough
      } else {
        hi = mid - 1;
      }
    }
    cut = value_of(lo);
  }
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (tid < (int)ctas) {
    put32(&sh.top[rank], tid, __float_as_uint(block_best));
    put32(&sh.cut[rank], tid, __float_as_uint(cut));
  }
  cluster_sync();
  float top = sh.top[0];
  cut = sh.cut[0];
  for (int c = 1; c < (int)ctas; ++c) { top = fmaxf(top, sh.top[c]); cut = fminf(cut, sh.cut[c]); }
  if (top == -INFINITY) {                      // no token can be drawn
    if (rank == 0 && tid == 0) { a.tokens[row] = -1; a.logprobs[row] = -INFINITY; }
    return;
  }

  Weigher weigh;
  weigh.top = (double)top;
  weigh.topf = top;
  weigh.rate = 1.4426950408889634074 / (double)temperature;
  // x from which min-p lets a value in
  const bool by_min = min_p > 0.f;
  const double least = by_min ? fma((double)temperature, log((double)min_p), (double)top) : -INFINITY;
  const bool plain = top_k == 0 && !by_p && !by_min;

  // the token at which the sums pass this much of `total`: the last that weighs anything for u of 1 and more
  auto goal_of = [&](u64 total) {
    const u64 g = __double2ull_rd((u > 0.f ? (double)u : 0.0) * (double)total);
    return g < total ? g : total - 1;
  };
  auto answer = [&](int index, float v, u64 total) {
    a.tokens[row] = index;
    const double z = v == top ? 0.0 : ((double)v - (double)top) / (double)temperature;
    a.logprobs[row] = (float)(z - log((double)total / (double)(1ull << SM_FRACTION)));
  };
  // sums over the cluster's CTAs, of a number of each thread's
  int round = 0;
  auto cluster_add = [&](u64 v, unsigned c, u64& all, unsigned& count) {
    v = block_add(v, sh);
    const u64 n = block_add((u64)c, sh);
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

  // ---- 2. the list
  if (!plain) {
    // everything from `from` on; for top-p alone the sum of all that min-p lets in
    const float from = fmaxf(cut, by_min ? __double2float_rd(least) : -INFINITY);
    const bool sum_all = by_p && top_k == 0;
    u64 sum = 0;
    for (int o = lane * VEC; o < a.seg; o += 32 * VEC) {
      float v[VEC];
      values(o, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        if (v[j] >= from && v[j] > -INFINITY) {
          const unsigned p = atomicAdd(&sh.found, 1u);
          if (p < SM_LIST) sh.spare[p] = (u64)(~key_of(v[j])) << 32 | (unsigned)(begin + o + j);
        }
      }
      if (sum_all) {
#pragma unroll
        for (int j = 0; j < VEC; ++j)
          if (!by_min || (double)v[j] >= least) sum += weigh(v[j]);
      }
    }
    if (sum_all) sum = block_add(sum, sh);
    __syncthreads();
    const unsigned found = sh.found;
    if (tid == 0) {
      unsigned b;
      asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(b) : "r"(at_rank(&sh.listed, 0)), "r"(found) : "memory");
      sh.base = b;
      put64(&sh.sum[1][rank], 0, sum);
    }
    __syncthreads();
    if (tid < (int)min(found, (unsigned)SM_LIST) && sh.base + tid < SM_LIST) put64(&sh.list[sh.base + tid], 0, sh.spare[tid]);
    cluster_sync();
    if (rank == 0) {
      const unsigned n = sh.listed;
      bool done = n <= SM_LIST;
      if (done) {
        int size = 32;
        while (size < (int)n) size <<= 1;
        const u64 entry = block_sort(tid < (int)n ? sh.list[tid] : ~0ull, size, sh.spare);
        const float v = value_of(~(uint32_t)(entry >> 32));
        bool in = tid < (int)n && (top_k == 0 || tid < top_k) && (!by_min || (double)v >= least);
        const u64 w = in ? weigh(v) : 0;
        u64 upto = w;
        block_scan(upto, sh);
        if (tid == SM_THREADS - 1) sh.total = upto;
        __syncthreads();
        if (by_p) {
          const u64 listed = sh.total;
          u64 all = listed;
          if (sum_all) {
            all = 0;
            for (int c = 0; c < (int)ctas; ++c) all += sh.sum[1][c];
          }
          const double share = (double)top_p * (double)all;
          done = (double)listed >= share;      // else the set goes on below the list
          in = in && (double)(upto - w) < share;
        }
        if (done) {
          // the set is a run at the head of the list; by index, each with its rank to find its weight
          const int k = __syncthreads_count(in);
          sh.spare[tid] = w;
          size = 32;
          while (size < k) size <<= 1;
          const u64 s = block_sort(in ? (entry & 0xffffffffull) << 32 | (unsigned)tid : ~0ull, size, sh.list);
          const int place = (int)(s & 0xffffffffull);
          __syncthreads();
          u64 sums = tid < k ? sh.spare[place] : 0;
          block_scan(sums, sh);
          if (tid == SM_THREADS - 1) sh.total = sums;
          __syncthreads();
          const u64 total = sh.total, goal = goal_of(total);
          const int chosen = __syncthreads_count(tid < k && sums <= goal);
          if (tid == chosen) sh.place = place;
          __syncthreads();
          if (tid == sh.place) answer((int)(entry & 0xffffffffull), v, total);
        }
      }
      if (tid < (int)ctas) put32(&sh.done, tid, done ? 1u : 0u);
    }
    cluster_sync();
    if (sh.done) return;
  }

  // ---- 3. thresholds: the set is the values of a key above `edge`, and the first `ties` of key `edge`, as far as
  // min-p lets them in
  uint32_t edge = key_of(-INFINITY);
  unsigned ties = 0;
  auto above_edge = [&](float v) { return key_of(v) > edge && (!by_min || (double)v >= least); };
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
    bottom = -warp_max(-__uint_as_float(sh.cred[lane]));
    if (tid < (int)ctas) put32(&sh.bottom[rank], tid, __float_as_uint(bottom));
    cluster_add(0, mine_in, all, candidates);
    bottom = sh.bottom[0];
    for (int c = 1; c < (int)ctas; ++c) bottom = fminf(bottom, sh.bottom[c]);

    // Finds the key at which a count (`by_count`: the first `need` values) or a sum (`share`) of the values above the
    // edge is reached, the count and sum above that key, and how many values have it. The first level cuts the
    // values into equal parts, the next ones a part's keys.
    const float scale = (float)(SM_BINS - 1) / (top - bottom);          // (inf or 0 apart: handled as one part)
    const bool whole = !(scale > 0.f && scale < INFINITY);
    auto part_of = [&](float v) { return whole ? 0 : min(SM_BINS - 1, (int)((top - v) * scale)); };
    auto descend = [&](bool by_count, u64 need, double share, uint32_t& key, u64& above, unsigned& inside) {
      int part = -1, shift = 0;
      uint32_t low = key_of(bottom), high = key_of(top);
      above = 0;
      for (bool first = !whole;;) {
        if (!first) {
          shift = 0;
          while (((high - low) >> shift) >= SM_BINS) ++shift;
        }
        sh.bin_count[tid] = 0;
        sh.bin_mass[tid] = 0;
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
            atomicAdd(&sh.bin_count[bin], 1u);
            if (!by_count) atomicAdd(&sh.bin_mass[bin], weigh(v[j]));
          }
        }
        cluster_sync();
        // every CTA adds its share of the bins over all CTAs and hands the sums to all
        const int per = SM_BINS / (int)ctas;
        if (tid < per) {
          const int bin = (int)rank * per + tid;
          unsigned c = 0;
          u64 m = 0;
          for (int r = 0; r < (int)ctas; ++r) { c += get32(&sh.bin_count[bin], r); m += get64(&sh.bin_mass[bin], r); }
          for (int r = 0; r < (int)ctas; ++r) { put32(&sh.all_count[bin], r, c); put64(&sh.all_mass[bin], r, m); }
        }
        cluster_sync();
        const u64 own = by_count ? sh.all_count[tid] : sh.all_mass[tid];
        u64 upto = own;
        block_scan(upto, sh);
        const bool short_of = by_count ? above + upto < need : (double)(above + upto) < share;
        const int bin = min(__syncthreads_count(short_of), SM_BINS - 1);
        if (tid == bin) { sh.above = above + upto - own; sh.inside = sh.all_count[tid]; }
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
          if (bin < SM_BINS - 1) low = max(low, key_of(at));
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
  auto weight_of = [&](float v) { return above_edge(v) ? weigh(v) : 0ull; };
  u64 sum = 0;
  unsigned equal = 0;
  for (int o = lane * VEC; o < a.seg; o += 32 * VEC) {
    float v[VEC];
    values(o, v);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      sum += weight_of(v[j]);
      equal += ties && key_of(v[j]) == edge ? 1u : 0u;
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
  u64 ws = sh.warp_sum[lane];
  unsigned we = sh.warp_equal[lane];
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

template <typename T>
int sample_go(const SampleArgs& args, int rows, cudaStream_t stream) {
  constexpr int VEC = Vec<T>::N;
  SampleArgs a = args;
  int sms = q_sm_count();
  if (sms <= 0) sms = 148;
  // CTAs of a row: what fills the SMs once, as long as a CTA keeps a few thousand values; more where a
  // CTA's part would not fit its shared memory
  auto seg_of = [&](int ctas) {
    const long long stretches = (long long)ctas * SM_WARPS;
    return (int)((a.vocab + VEC - 1 + stretches * VEC - 1) / (stretches * VEC)) * VEC;
  };
  int ctas = 1;
  while (ctas < SM_CTAS && rows * ctas * 2 <= sms && a.vocab / (ctas * 2) >= 4096) ctas *= 2;
  while (ctas < SM_CTAS && (size_t)seg_of(ctas) * SM_WARPS * sizeof(T) > SM_SLICE) ctas *= 2;
  a.seg = seg_of(ctas);
  const size_t slice = (size_t)a.seg * SM_WARPS * sizeof(T);
  a.resident = slice <= SM_SLICE;              // (otherwise every pass reads the row again)
  const size_t bytes = (sizeof(SampleShared) + 15) / 16 * 16 + (a.resident ? slice : 0);
  static size_t done[64] = {0};
  Q_CHECK_CUDA(q_ensure_smem(k_sample<T>, bytes, done));
  Q_CHECK_CUDA(q_launch_cluster(k_sample<T>, dim3((unsigned)rows * ctas), dim3(SM_THREADS), bytes, stream, (unsigned)ctas, a));
  return Q_OK;
}

}  // namespace

extern "C" int q_sample_tokens(const void* d_logits, int fp32, int64_t row_stride, const float* d_uniform,
                               const q_sampling_t* sampling, int64_t* d_tokens, float* d_logprobs, int rows, int vocab,
                               void* stream) {
  const char* who = "q_sample_tokens";
  Q_CHECK_ARG(d_logits && d_uniform && sampling && d_tokens && d_logprobs, "%s: null pointer", who);
  Q_CHECK_ARG(rows >= 1 && rows <= (1 << 24) && vocab >= 1 && vocab <= SM_MAX_VOCAB,
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
