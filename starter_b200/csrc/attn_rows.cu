// Attention of a few query rows per kv head (1-8 tokens per sequence, at most 32 rows) over a part of a
// paged cache: a sliding window with first tokens kept (sinks), and both halves of the attention of a
// batch that shares a prefix - few rows over the prefix, and every sequence's own keys, joined with the
// partial results of the prefix.
//
//   out = sum_j exp(s_j - m) v_j / sum_j exp(s_j - m),  s_j = scale q . k_j,  m = max_j s_j
//
// over the keys j that the row sees. A cluster of CTAs shares one (sequence, kv head): the pages that hold
// a visible key are dealt out evenly, every CTA keeps a running maximum, sum and weighted sum, and the parts
//   (m, l, O) (+) (m', l', O') = (M, e^(m-M) l + e^(m'-M) l', e^(m-M) O + e^(m'-M) O'),  M = max(m, m')
// are joined in the cluster's shared memory, in a fixed order.
//
// Bound by the bytes of the visible keys at long windows, by latencies at short ones (position -> pages ->
// keys -> join is a chain of memory round trips); hence one launch, and of a page only the rows somebody sees
// are copied: a window with 4 sinks brings 4 rows of its first page.
//
// Keys are the M dimension of the MMAs, a tile of 8 query rows the N dimension: S^T = K Q^T, O^T = V^T P^T,
// as in the decode attention, so that few rows leave no accumulator empty. Four warps share a tile of 64 keys, 16
// keys each; RG such groups take a row tile each, DG of them a key tile each. (With the row tiles in one warp's
// registers, four at most, a tile of 64 keys and 32 rows took 2.9 us: one warp a scheduler hides none of the MMAs'
// latency. As here 1.0 to 1.3.) Where 28 rows (6 sequences x 4 tokens x 7 heads, two tiles a CTA, cluster of five) spend their 10.2
// us, by clock64: position, queries and the first tile's arrival 2.2, the tiles 2.5, states of the warps to shared memory and
// the cluster's beginning 1.1, their join and the stores into the other CTAs 2.3, the barrier 0.9, the rows 1.2. Cast boundaries as there: fp32 scores and statistics, P rounded to bf16 for
// P V (the tensor cores' operand type), fp32 sums, one rounding of the result.
//
// Rows of a page that no query row sees may hold anything: their scores are replaced, their values cleared.
#include "mma.cuh"
#include "tc.cuh"
#include "attn_parts.cuh"

int* q_attn_status_addr();

namespace {

constexpr int ROW_TILE = Q_PAGE_TOKENS * 256;      // bytes of a K or V page tile
constexpr int ROW_STAGE = 2 * ROW_TILE;
constexpr int ROW_LD = 136;                        // floats of a row of the warps' merge area (rows on other banks)
constexpr int ROW_FAR = 0x7fffffff - 64;           // positions count up to this, so that their sums with T fit
constexpr int ROW_ALL = 0x7fffffff - 32;           // a window that holds every key of every such position
constexpr int MAX_SPLITS = 8;                      // CTAs of a cluster (the portable size)

struct RowsArgs {
  const bf16* q;
  const char* kpool;
  const char* vpool;
  const int32_t* table;
  const int32_t* pos;        // flat: the number of keys
  bf16* out;                 // final rows, or
  AttnParts parts;           // ... written (write_parts) or joined (parts.splits > 0)
  int pages_per_seq, pos_step, T, G, nq, nkv, window, sinks, share, stages;
  float scale_log2;
  bool flat;                 // every row sees keys [0, *pos): rows over a shared prefix
  bool write_parts;
  bool early;                // keys and queries are older than the launch before this one
};

// What a sequence's rows see, and in which pages it lies.
struct Seen {
  int pos, lim, low;         // position of row 0; newest visible key + 1; oldest key of the first row's window
  int sink_pages, window_page, pages;
};

__device__ __forceinline__ Seen seen_of(const RowsArgs& a, int b) {
  Seen s;
  const int room = a.pages_per_seq * Q_PAGE_TOKENS;
  int p = __ldcg(a.pos + (size_t)b * a.pos_step);
  if (a.flat) p = max(0, p) - a.T;                               // row T-1 is then the newest key
  // a position behind the pages sees what its window still holds of them; nothing outside the table is read
  s.pos = a.flat ? min(p, room - a.T) : min(max(p, -a.T), ROW_FAR);
  s.lim = min(max(s.pos + a.T, 0), room);
  s.low = a.flat ? 0 : min(max(0, s.pos - a.window + 1), s.lim);
  s.sink_pages = (min(a.sinks, s.lim) + Q_PAGE_TOKENS - 1) / Q_PAGE_TOKENS;
  s.window_page = max(s.sink_pages, s.low / Q_PAGE_TOKENS);
  s.pages = s.sink_pages + max(0, (s.lim + Q_PAGE_TOKENS - 1) / Q_PAGE_TOKENS - s.window_page);
  return s;
}
__device__ __forceinline__ int page_of(const Seen& s, int i) {
  return i < s.sink_pages ? i : i - s.sink_pages + s.window_page;
}

__device__ __forceinline__ void copy_rows(uint32_t dst, const char* src, uint32_t bytes, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t remote_addr(uint32_t local, int rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}

template <int RG, int DG, int BLOCKS>
__global__ void __launch_bounds__((4 * RG * DG + 1) * 32, BLOCKS)
k_attn_rows(RowsArgs a, int* status) {
  constexpr int DC = 4 * RG * DG;                  // consumer warps
  constexpr int SETS = 4;                          // accumulators of Q K^T: an MMA's result is ~280 cycles away
  extern __shared__ __align__(1024) unsigned char smem[];
  const int NS = a.stages;
  unsigned char* stages = smem;
  unsigned char* qtile = smem + NS * ROW_STAGE;                            // RG * 8 rows of 256 B
  uint64_t* bars = reinterpret_cast<uint64_t*>(qtile + RG * 8 * 256);      // full[NS], empty[NS]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(bars + 2 * NS);
  float* recv = reinterpret_cast<float*>(bars + 2 * NS + 2);               // [splits][share] sums, then [splits][R][2]

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int b = blockIdx.y / a.nkv, kh = blockIdx.y - b * a.nkv;
  const int R = a.T * a.G;
  const int rank = (int)cluster_rank(), S = (int)cluster_size();
  if (tid == 0) {
    for (int i = 0; i < NS; ++i) {
      mbar_init(smem_u32(&bars[i]), 1);
      mbar_init(smem_u32(&bars[NS + i]), 4 * RG);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  __syncthreads();
  // (waited for before the first store into another CTA's memory: that CTA has to be running)
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  if (!a.early) pdl_wait();      // position, table, queries and keys may come from the launch before
  // (after the wait: what follows may then read early whatever the launches before this one wrote)
  pdl_launch_dependents();

  const Seen seen = seen_of(a, b);
  // pages are dealt out evenly over all splits of the grid's row
  const int parts = gridDim.x, part = blockIdx.x;
  const int each = seen.pages / parts, more = seen.pages - each * parts;
  const int first = part * each + min(part, more);
  const int ntiles = each + (part < more ? 1 : 0);

  if (warp == DC) {
    // ---------------- producer ----------------
    const int32_t* table = a.table + (size_t)b * a.pages_per_seq;
    bool ok = true;
    int entry = 0, it = 0;
    for (; it < ntiles; ++it) {
      if ((it & 31) == 0) entry = it + lane < ntiles ? __ldcg(table + page_of(seen, first + it + lane)) : 0;
      const int page = __shfl_sync(0xffffffffu, entry, it & 31);
      const int s = it % NS;
      if (it >= NS) {
        const int landed = mbar_wait(smem_u32(&bars[NS + s]), ((it / NS) - 1) & 1, abort_flag) ? 1 : 0;
        ok = __all_sync(0xffffffffu, landed);
        if (!ok) {
          if (lane == 0) { atomicExch(status, 1); *abort_flag = 1; }
          break;
        }
      }
      if (lane == 0) {
        const int at = page_of(seen, first + it), base = at * Q_PAGE_TOKENS;
        int r0 = 0, r1 = min(Q_PAGE_TOKENS, seen.lim - base);
        if (at >= seen.sink_pages) r0 = max(0, seen.low - base);
        else if (seen.low >= base + Q_PAGE_TOKENS) r1 = min(r1, a.sinks - base);
        const uint32_t bytes = (uint32_t)(r1 - r0) * 256u;
        const size_t off = ((size_t)page * a.nkv + kh) * ROW_TILE + (size_t)r0 * 256;
        const uint32_t bar = smem_u32(&bars[s]), dst = smem_u32(stages) + s * ROW_STAGE + r0 * 256;
        mbar_expect_tx(bar, 2 * bytes);
        copy_rows(dst, a.kpool + off, bytes, bar);
        copy_rows(dst + ROW_TILE, a.vpool + off, bytes, bar);
      }
      __syncwarp();
    }
    // copies in flight land before the CTA may leave, also where a wait ran out
    if (lane == 0)
      for (int j = max(0, it - NS); j < it; ++j) mbar_wait_plain(smem_u32(&bars[j % NS]), (j / NS) & 1);
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  } else {
    // ---------------- consumers ----------------
    for (int c = tid; c < RG * 8 * 16; c += DC * 32) {
      const int r = c >> 4, ch = c & 15;
      uint4 v = make_uint4(0, 0, 0, 0);
      if (r < R) {
        const int t = r / a.G, g = r - t * a.G;
        v = __ldcg(reinterpret_cast<const uint4*>(a.q + ((size_t)(b * a.T + t) * a.nq + kh * a.G + g) * 128) + ch);
      }
      *reinterpret_cast<uint4*>(qtile + r * 256 + ((ch ^ (r & 7)) << 4)) = v;
    }
    asm volatile("bar.sync 1, %0;" ::"n"(DC * 32) : "memory");

    const int g = lane >> 2, t4 = lane & 3;
    const int wk = warp & 3;                       // key quarter of the warp
    const int rg = (warp >> 2) % RG, tg = (warp >> 2) / RG;     // its row tile, and its tiles: tg, tg + DG, ..
    float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};   // rows 8 rg + 2 t4, + 1 (l: of this lane's keys)
    float oacc[8][4];                              // dims 16 d + g, 16 d + g + 8
    int lim_r[2], low_r[2];                        // what the row sees: [low, lim) and the sinks
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = 8 * rg + 2 * t4 + h, t = r / a.G;
      lim_r[h] = r >= R ? 0 : a.flat ? seen.lim : min(seen.pos + t + 1, seen.lim);
      low_r[h] = a.flat ? 0 : seen.pos + t + 1 - a.window;
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) oacc[d][0] = oacc[d][1] = oacc[d][2] = oacc[d][3] = 0.f;
    uint32_t qf[8][2];                             // Q^T fragments of the eight k steps
#pragma unroll
    for (int kp = 0; kp < 4; ++kp) {
      const int row = 8 * rg + (lane & 7), ch = 4 * kp + (lane >> 3);
      ldsm_x4(smem_u32(qtile) + row * 256 + ((ch ^ (row & 7)) << 4), qf[2 * kp][0], qf[2 * kp][1], qf[2 * kp + 1][0], qf[2 * kp + 1][1]);
    }
    for (int it = tg; it < ntiles; it += DG) {
      const int s = it % NS;
      const int landed = mbar_wait(smem_u32(&bars[s]), (it / NS) & 1, abort_flag) ? 1 : 0;
      if (!__all_sync(0xffffffffu, landed)) {
        if (lane == 0) { atomicExch(status, 2); *abort_flag = 1; }
        break;
      }
      unsigned char* kt = stages + s * ROW_STAGE;
      unsigned char* vt = kt + ROW_TILE;
      const int key0 = page_of(seen, first + it) * Q_PAGE_TOKENS + wk * 16;
      if (key0 < seen.lim && (key0 + 16 > seen.low || key0 < a.sinks)) {
        if (key0 + 16 > seen.lim || (key0 < seen.low && key0 + 16 > a.sinks)) {
          // values that no row sees are cleared: 0 * garbage could be NaN in P V (the warps of the other row tiles
          // write the same zeros)
          for (int i = lane; i < 16 * 16; i += 32) {
            const int key = key0 + (i >> 4);
            if (key >= seen.lim || (key < seen.low && key >= a.sinks))
              *reinterpret_cast<uint4*>(vt + (wk * 16 + (i >> 4)) * 256 + ((i & 15) << 4)) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        const uint32_t k_base = smem_u32(kt), v_base = smem_u32(vt);
        float sset[SETS][4];
#pragma unroll
        for (int q = 0; q < SETS; ++q) sset[q][0] = sset[q][1] = sset[q][2] = sset[q][3] = 0.f;
        const int arow = wk * 16 + (lane & 7) + 8 * ((lane >> 3) & 1);
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          uint32_t a0, a1, a2, a3;
          const int ch = 2 * ks + (lane >> 4);
          ldsm_x4(k_base + arow * 256 + ((ch ^ (arow & 7)) << 4), a0, a1, a2, a3);
          mma16816(sset[ks % SETS], a0, a1, a2, a3, qf[ks][0], qf[ks][1]);
        }
        // every row sees all 16 keys: nothing to mask
        const bool open = key0 + 16 <= (a.flat ? seen.lim : seen.pos + 1) &&
                          (a.flat || key0 > seen.pos + a.T - 1 - a.window || key0 + 16 <= a.sinks);
        float sc[4];                             // (key g, row 2 t4), (g, 2 t4 + 1), (g + 8, 2 t4), (g + 8, 2 t4 + 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float v = ((sset[0][e] + sset[1][e]) + (sset[2][e] + sset[3][e])) * a.scale_log2;
          if (!open) {
            const int key = key0 + g + 8 * (e >> 1);
            v = key < lim_r[e & 1] && (key >= low_r[e & 1] || key < a.sinks) ? v : -INFINITY;
          }
          sc[e] = v;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float mx = fmaxf(sc[h], sc[2 + h]);
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
          const float m_new = fmaxf(m_run[h], mx);
          const float m_safe = m_new == -INFINITY ? 0.f : m_new;
          const float resc = exp2f(m_run[h] - m_safe);               // exp2(-inf) = 0 on the first keys
          sc[h] = exp2f(sc[h] - m_safe);
          sc[2 + h] = exp2f(sc[2 + h] - m_safe);
          l_run[h] = l_run[h] * resc + (sc[h] + sc[2 + h]);
          m_run[h] = m_new;
#pragma unroll
          for (int d = 0; d < 8; ++d) { oacc[d][h] *= resc; oacc[d][2 + h] *= resc; }
        }
        const uint32_t pb0 = transpose8x8(pack_bf16(sc[0], sc[1])), pb1 = transpose8x8(pack_bf16(sc[2], sc[3]));
        const int mi = lane >> 3, vrow = wk * 16 + 8 * (mi >> 1) + (lane & 7);
#pragma unroll
        for (int d = 0; d < 8; ++d) {
          uint32_t v0, v1, v2, v3;
          const int ch = 2 * d + (mi & 1);
          ldsm_x4_t(v_base + vrow * 256 + ((ch ^ (vrow & 7)) << 4), v0, v1, v2, v3);
          mma16816(oacc[d], v0, v1, v2, v3, pb0, pb1);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bars[NS + s]));
    }
    // join the warps' states of a row through shared memory (the R real rows), over the ring: every copy has
    // landed, since every tile was waited for
    asm volatile("bar.sync 1, %0;" ::"n"(DC * 32) : "memory");
    constexpr int STATES = 4 * DG;                           // of a row
    float* mo = reinterpret_cast<float*>(stages);            // [STATES][R][ROW_LD]
    float* mml = mo + STATES * R * ROW_LD;                   // [STATES][R][2]
    if (*abort_flag == 0) {
      const int state = tg * 4 + wk;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float l = l_run[h];
        l += __shfl_xor_sync(0xffffffffu, l, 4);
        l += __shfl_xor_sync(0xffffffffu, l, 8);
        l += __shfl_xor_sync(0xffffffffu, l, 16);
        const int r = 8 * rg + 2 * t4 + h;
        if (r < R) {
          float* dst = mo + (state * R + r) * ROW_LD + g;
#pragma unroll
          for (int d = 0; d < 8; ++d) { dst[16 * d] = oacc[d][h]; dst[16 * d + 8] = oacc[d][2 + h]; }
          if (g == 0) {
            mml[(state * R + r) * 2] = m_run[h];
            mml[(state * R + r) * 2 + 1] = l;
          }
        }
      }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(DC * 32) : "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const int d = tid & 127;
    for (int r = tid >> 7; r < R && *abort_flag == 0; r += RG * DG) {
      float mw[STATES], Mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < STATES; ++w) { mw[w] = mml[(w * R + r) * 2]; Mx = fmaxf(Mx, mw[w]); }
      const float Ms = Mx == -INFINITY ? 0.f : Mx;
      float Lsum = 0.f, O = 0.f;
#pragma unroll
      for (int w = 0; w < STATES; ++w) {
        const float wt = exp2f(mw[w] - Ms);
        Lsum += wt * mml[(w * R + r) * 2 + 1];
        O += wt * mo[(w * R + r) * ROW_LD + d];
      }
      // to the CTA that joins this row: slot `rank` of its receive area
      const int owner = r % S, at = r / S;
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(remote_addr(smem_u32(recv), owner) +
                   (uint32_t)(rank * a.share + at * 128 + d) * 4u), "f"(O) : "memory");
      if (d < S)           // the row's maximum and sum go to every CTA of the cluster (thread d -> CTA d)
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(remote_addr(smem_u32(recv), d) +
                     (uint32_t)(S * a.share + (rank * R + r) * 2) * 4u), "f"(Mx), "f"(Lsum) : "memory");
    }
  }
  // everything this CTA joins is in its own memory behind the barrier: no remote reads, and no second
  // barrier before it may leave
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (a.early) pdl_wait();       // the prefix's partial rows are complete
  // a warp joins a row: rank, rank + S, ..
  const float* rml = recv + S * a.share;
  const int psplits = a.parts.splits > 0 && !a.write_parts ? parts_used(a.parts) : 0;
  for (int at = warp; rank + at * S < R; at += DC + 1) {
    const int r = rank + at * S;
    const int t = r / a.G, hg = r - t * a.G;
    const size_t prow = (size_t)(b * a.T + t) * a.G + hg;
    // all of the prefix's first parts are asked for at once, with their maxima and sums
    constexpr int AHEAD = RG == 1 && BLOCKS < 4 ? 16 : 8;
    float4 o[AHEAD];
    if (psplits > 0)
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        o[j] = j < psplits ? __ldcg(reinterpret_cast<const float4*>(a.parts.o + a.parts.row(j, kh, prow) * 128) + lane)
                           : make_float4(0.f, 0.f, 0.f, 0.f);
    float2 ml = make_float2(-INFINITY, 0.f);
    if (lane < S) ml = *reinterpret_cast<const float2*>(rml + (lane * R + r) * 2);
    float2 pml[2] = {make_float2(-INFINITY, 0.f), make_float2(-INFINITY, 0.f)};      // parts lane and lane + 32
#pragma unroll
    for (int e = 0; e < 2; ++e)
      if (lane + 32 * e < psplits) pml[e] = __ldcg(a.parts.ml + a.parts.row(lane + 32 * e, kh, prow));
    float Mx = warp_max(fmaxf(ml.y > 0.f ? ml.x : -INFINITY,
                              fmaxf(pml[0].y > 0.f ? pml[0].x : -INFINITY, pml[1].y > 0.f ? pml[1].x : -INFINITY)));
    if (Mx == -INFINITY) Mx = 0.f;
    const float w = ml.y > 0.f ? exp2f(ml.x - Mx) : 0.f;
    const float pw[2] = {pml[0].y > 0.f ? exp2f(pml[0].x - Mx) : 0.f, pml[1].y > 0.f ? exp2f(pml[1].x - Mx) : 0.f};
    // NaN (a NaN among the visible keys) is carried on
    float l = (ml.y == ml.y ? w * ml.y : ml.y) + (pml[0].y == pml[0].y ? pw[0] * pml[0].y : pml[0].y) +
              (pml[1].y == pml[1].y ? pw[1] * pml[1].y : pml[1].y);
    l = warp_sum(l);
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float f, float4 x) { O.x += f * x.x; O.y += f * x.y; O.z += f * x.z; O.w += f * x.w; };
    for (int s = 0; s < S; ++s)
      add(__shfl_sync(0xffffffffu, w, s), *reinterpret_cast<const float4*>(recv + s * a.share + at * 128 + 4 * lane));
    if (psplits > 0)
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) add(__shfl_sync(0xffffffffu, pw[0], j), o[j]);
    for (int s0 = AHEAD; s0 < psplits; s0 += AHEAD) {
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        o[j] = s0 + j < psplits ? __ldcg(reinterpret_cast<const float4*>(a.parts.o + a.parts.row(s0 + j, kh, prow) * 128) + lane)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const float lo = __shfl_sync(0xffffffffu, pw[0], (s0 + j) & 31), hi = __shfl_sync(0xffffffffu, pw[1], (s0 + j) & 31);
        add(s0 + j < 32 ? lo : hi, o[j]);
      }
    }
    if (a.write_parts) {
      const size_t row = a.parts.row(blockIdx.x / S, kh, prow);
      *(reinterpret_cast<float4*>(a.parts.o + row * 128) + lane) = O;
      if (lane == 0) a.parts.ml[row] = make_float2(Mx, l);
    } else {
      const float inv = l > 0.f ? 1.f / l : l == 0.f ? 0.f : l;
      uint2 packed;
      packed.x = pack_bf16(O.x * inv, O.y * inv);
      packed.y = pack_bf16(O.z * inv, O.w * inv);
      *reinterpret_cast<uint2*>(a.out + ((size_t)(b * a.T + t) * a.nq + kh * a.G + hg) * 128 + 4 * lane) = packed;
    }
  }
}

// How a launch splits: row tiles, tile groups, CTAs of a cluster, clusters of a (sequence, kv head), ring stages.
struct RowsPlan { int rg, dg, per_sm, splits, clusters, stages, share; size_t smem; };

typedef void (*rows_kernel)(RowsArgs, int*);
rows_kernel rows_form(const RowsPlan& p) {
  if (p.rg == 4) return k_attn_rows<4, 1, 1>;
  if (p.rg == 2) return k_attn_rows<2, 1, 2>;
  return p.dg == 3 ? k_attn_rows<1, 3, 1> : p.per_sm == 4 ? k_attn_rows<1, 1, 4> : k_attn_rows<1, 1, 3>;
}

size_t rows_smem(const RowsPlan& p, int rows) {
  return (size_t)p.stages * ROW_STAGE + p.rg * 8 * 256 + 16 * p.stages + 16 + (size_t)(p.splits * p.share + p.splits * rows * 2) * 4;
}

// Fills in the ring and the sizes for `each` pages a split.
void rows_sizes(RowsPlan& p, int rows, long long each) {
  p.stages = p.rg == 4 ? 6 : p.per_sm == 4 ? 1 : p.per_sm == 3 ? 2 : 3;
  const int need = (4 * p.dg * rows * (ROW_LD + 2) * 4 + ROW_STAGE - 1) / ROW_STAGE;       // the warps' states lie over the ring
  if (each < p.stages) p.stages = each < 1 ? 1 : (int)each;
  if (p.dg == 3) p.stages = 3;                    // a stage always belongs to the same group, which tracks its parity
  if (p.stages < need) p.stages = need;
  p.share = (rows + p.splits - 1) / p.splits * 128;
  p.smem = rows_smem(p, rows);
}

// Lets a form have any plan's shared memory: the limit is the kernel's, not the launch's, and one that never moves
// cannot be lowered by another shape's launch, or by one of another thread.
constexpr size_t ROW_SMEM_MAX = 227 * 1024;
cudaError_t rows_room(const RowsPlan& p) {
  static size_t done[5][64] = {{0}};
  return q_ensure_smem(rows_form(p), ROW_SMEM_MAX, done[p.rg == 4 ? 3 : p.rg == 2 ? 2 : p.dg == 3 ? 1 : p.per_sm == 4 ? 4 : 0]);
}

// Clusters of a form that the current device holds at once (a cluster stays inside one GPC, so this is less than
// the SMs would allow), asked once per device.
int rows_resident(const RowsPlan& p) {
  static int cached[64][4][MAX_SPLITS + 1];
  const int form = p.rg == 4 ? 3 : p.rg == 2 ? 2 : p.dg == 3 ? 1 : 0;
  const int dev = q_device_index(), per_sm = form == 0 || form == 2 ? 2 : 1;
  if (dev < 0) return per_sm * 148 / p.splits;
  int& n = cached[dev][form][p.splits];
  if (n == 0) {
    RowsPlan full = p;
    rows_sizes(full, 8 * p.rg, 1 << 20);
    const rows_kernel k = rows_form(full);
    int got = 0;
    cudaError_t e = rows_room(full);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(p.splits);
    cfg.blockDim = dim3((4 * p.rg * p.dg + 1) * 32);
    cfg.dynamicSmemBytes = full.smem;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = p.splits; at[0].val.clusterDim.y = 1; at[0].val.clusterDim.z = 1;
    cfg.attrs = at; cfg.numAttrs = 1;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveClusters(&got, k, &cfg);
    if (e != cudaSuccess) { cudaGetLastError(); got = per_sm * 148 / p.splits; }
    n = got > 0 ? got : -1;
  }
  return n;
}

// vh: (sequence, kv head) pairs; pages: most pages a pair's rows can see. join: the splits merge in one
// cluster; otherwise the pages go to as many clusters as fill the SMs, by their number on a B200 (the
// caller's scratch goes by it, whichever device is current).
RowsPlan rows_plan(int vh, int rows, long long pages, bool join) {
  RowsPlan p = {};
  p.rg = rows <= 8 ? 1 : rows <= 16 ? 2 : 4;
  p.dg = 1;
  p.clusters = 1;
  const int most = pages < MAX_SPLITS ? (int)pages : MAX_SPLITS;
  p.splits = 1;
  if (join) {
    // as many splits as leave all clusters resident
    for (p.splits = most; p.splits > 1 && rows_resident(p) < vh; --p.splits) {}
    if (p.rg == 1 && p.splits == MAX_SPLITS && pages >= 3 * MAX_SPLITS) {
      // few heads and long windows: three groups of warps, a tile each, on an SM of their own
      p.dg = 3;
      if (rows_resident(p) < vh) p.dg = 1;
    }
  } else {
    const int per_sm = p.rg == 4 ? 1 : 2;
    p.splits = most < 4 ? most : 4;
    long long n = (long long)per_sm * 132 / ((long long)vh * p.splits);
    if (n > pages / p.splits) n = pages / p.splits;
    p.clusters = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
  }
  // More unsplit pairs than two for an SM: a ring of two stages leaves room for a third, one stage for a fourth, where
  // that saves the second wave. 32 / 8 heads, two to an SM / so, us: 50 sequences under a window of 512 28.6 / 22.4, 48
  // under 300 20.4 / 15.7; 64 under 512 31.5 / 30.3, 64 x 333 keys 21.7 / 20.0, 64 under 1024 49.3 / 49.4.
  if (p.rg == 1 && p.dg == 1 && p.splits == 1 && vh > 2 * 148 && vh <= 4 * 148) p.per_sm = vh <= 3 * 148 ? 3 : 4;
  rows_sizes(p, rows, (pages + (long long)p.splits * p.clusters - 1) / ((long long)p.splits * p.clusters));
  return p;
}

int rows_launch(const RowsPlan& p, RowsArgs& a, int vh, const char* who, cudaStream_t stream) {
  int* status = q_attn_status_addr();
  if (!status) { q_set_error("%s: could not locate the device status word", who); return Q_ERR_CUDA; }
  a.share = p.share;
  a.stages = p.stages;
  const rows_kernel k = rows_form(p);
  Q_CHECK_CUDA(rows_room(p));
  Q_CHECK_CUDA(q_launch_cluster(k, dim3(p.splits * p.clusters, vh), dim3((4 * p.rg * p.dg + 1) * 32), p.smem, stream,
                                (unsigned)p.splits, a, status));
  return Q_OK;
}

int check_rows(const char* who, const void* d_q, const q_kv_layout_t* kv, const int32_t* d_pos, const void* d_out,
               int batch, int T, int n_q_heads) {
  Q_CHECK_ARG(d_q && kv && d_pos && d_out, "%s: null pointer", who);
  Q_CHECK_ARG(kv->d_kpool && kv->d_vpool && kv->d_block_table && kv->pages_per_seq >= 1 && kv->n_kv_heads >= 1,
              "%s: incomplete KV layout", who);
  const int nkv = kv->n_kv_heads;
  Q_CHECK_ARG(batch >= 1 && T >= 1 && n_q_heads >= nkv && n_q_heads % nkv == 0, "%s: bad batch/T/heads", who);
  const int G = n_q_heads / nkv;
  Q_CHECK_ARG((long long)T * G <= 32, "%s: T*G = %lld exceeds 32 query rows per kv head", who, (long long)T * G);
  Q_CHECK_ARG((long long)batch * nkv <= 65535, "%s: too many (sequence, kv head) pairs", who);
  Q_CHECK_ARG(kv->pages_per_seq <= (1 << 24), "%s: too many pages per sequence", who);
  Q_CHECK_ALIGN(d_q, 16, who); Q_CHECK_ALIGN(kv->d_kpool, 16, who); Q_CHECK_ALIGN(kv->d_vpool, 16, who);
  Q_CHECK_ALIGN(d_out, 8, who); Q_CHECK_ALIGN(d_pos, 4, who); Q_CHECK_ALIGN(kv->d_block_table, 4, who);
  return Q_OK;
}

RowsArgs rows_args(const void* d_q, const q_kv_layout_t* kv, const int32_t* d_pos, int pos_per_seq, void* d_out,
                   int T, int n_q_heads, float scale) {
  RowsArgs a = {};
  a.q = (const bf16*)d_q;
  a.kpool = (const char*)kv->d_kpool;
  a.vpool = (const char*)kv->d_vpool;
  a.table = kv->d_block_table;
  a.pos = d_pos;
  a.pos_step = pos_per_seq ? 1 : 0;
  a.out = (bf16*)d_out;
  a.pages_per_seq = kv->pages_per_seq;
  a.nkv = kv->n_kv_heads;
  a.nq = n_q_heads;
  a.T = T;
  a.G = n_q_heads / kv->n_kv_heads;
  a.window = ROW_ALL;
  a.scale_log2 = scale * 1.4426950408889634f;
  return a;
}

}  // namespace

extern "C" int q_attention_window(const void* d_q, const q_kv_layout_t* kv, const int32_t* d_pos, int pos_per_seq,
                                  void* d_out, int batch, int T, int n_q_heads, int window, int sinks, float scale,
                                  void* stream) {
  const char* who = "q_attention_window";
  const int rc = check_rows(who, d_q, kv, d_pos, d_out, batch, T, n_q_heads);
  if (rc) return rc;
  Q_CHECK_ARG(window >= 1 && sinks >= 0, "%s: window %d / sinks %d", who, window, sinks);
  RowsArgs a = rows_args(d_q, kv, d_pos, pos_per_seq, d_out, T, n_q_heads, scale);
  a.window = window < ROW_ALL ? window : ROW_ALL;
  a.sinks = sinks;
  // most pages a sequence's rows can see: those of window + T - 1 consecutive keys, and the sinks'
  const long long all = kv->pages_per_seq;
  long long pages = ((long long)a.window + T - 2) / Q_PAGE_TOKENS + 2 + ((long long)a.sinks + Q_PAGE_TOKENS - 1) / Q_PAGE_TOKENS;
  if (pages > all) pages = all;
  const RowsPlan p = rows_plan(batch * kv->n_kv_heads, T * a.G, pages, true);
  return rows_launch(p, a, batch * kv->n_kv_heads, who, (cudaStream_t)stream);
}

namespace {

// How the prefix of a batch is split: few rows per kv head on k_attn_rows (clusters of CTAs, each leaving one
// part), more on the prompt attention's kernel (rows there fill tiles of 128).
struct SharedPlan { bool few; int parts, rows; RowsPlan plan; };

SharedPlan shared_plan(int batch, int T, int n_q_heads, int nkv, long long prefix_pages) {
  SharedPlan s;
  const int G = n_q_heads / nkv;
  s.rows = batch * T * G;
  s.few = s.rows <= 32;
  if (s.few) {
    s.plan = rows_plan(nkv, s.rows, prefix_pages, false);
    s.parts = s.plan.clusters;
  } else {
    constexpr int sms = 148;
    const int tokens = 128 / G, tiles = (batch * T + tokens - 1) / tokens, blocks = tiles == 1 ? 1 : (tiles + 1) / 2;
    long long n = sms / ((long long)nkv * blocks);
    if (n > (prefix_pages + 1) / 2) n = (prefix_pages + 1) / 2;
    s.parts = (int)(n < 1 ? 1 : n > 64 ? 64 : n);
  }
  return s;
}

bool shared_sizes(int batch, int T, int n_q_heads, int nkv, long long prefix_pages) {
  return batch >= 1 && T >= 1 && nkv >= 1 && n_q_heads >= nkv && n_q_heads % nkv == 0 && (long long)T * (n_q_heads / nkv) <= 32 &&
         (long long)batch * nkv <= 65535 && (long long)batch * T * (n_q_heads / nkv) <= (1 << 24) && prefix_pages >= 1 &&
         prefix_pages <= (1 << 23);
}

}  // namespace

extern "C" int64_t q_attention_shared_scratch_bytes(int batch, int T, int n_q_heads, int n_kv_heads, int prefix_pages) {
  if (!shared_sizes(batch, T, n_q_heads, n_kv_heads, prefix_pages)) return 0;
  const SharedPlan s = shared_plan(batch, T, n_q_heads, n_kv_heads, prefix_pages);
  return (int64_t)s.parts * n_kv_heads * s.rows * (128 + 2) * 4;
}

extern "C" int q_attention_shared(const void* d_q, const q_kv_layout_t* prefix, const int32_t* d_prefix_len,
                                  const q_kv_layout_t* kv, const int32_t* d_pos, int pos_per_seq, void* d_scratch,
                                  void* d_out, int batch, int T, int n_q_heads, float scale, void* stream) {
  const char* who = "q_attention_shared";
  int rc = check_rows(who, d_q, kv, d_pos, d_out, batch, T, n_q_heads);
  if (rc) return rc;
  Q_CHECK_ARG(prefix && d_prefix_len && d_scratch, "%s: null pointer", who);
  Q_CHECK_ARG(prefix->d_kpool && prefix->d_vpool && prefix->d_block_table, "%s: incomplete KV layout of the prefix", who);
  Q_CHECK_ARG(prefix->n_kv_heads == kv->n_kv_heads, "%s: prefix and sequences have different kv heads", who);
  const int nkv = kv->n_kv_heads;
  Q_CHECK_ARG(shared_sizes(batch, T, n_q_heads, nkv, prefix->pages_per_seq), "%s: too many rows or prefix pages", who);
  Q_CHECK_ALIGN(d_scratch, 16, who); Q_CHECK_ALIGN(d_prefix_len, 4, who); Q_CHECK_ALIGN(prefix->d_block_table, 4, who);
  Q_CHECK_ALIGN(prefix->d_kpool, 16, who); Q_CHECK_ALIGN(prefix->d_vpool, 16, who);
  const SharedPlan s = shared_plan(batch, T, n_q_heads, nkv, prefix->pages_per_seq);
  AttnParts parts = {};
  parts.o = (float*)d_scratch;
  parts.ml = reinterpret_cast<float2*>(parts.o + (size_t)s.parts * nkv * s.rows * 128);
  parts.splits = s.parts;
  parts.nkv = nkv;
  parts.rows = s.rows;
  if (s.few) {
    RowsArgs a = rows_args(d_q, prefix, d_prefix_len, 0, nullptr, batch * T, n_q_heads, scale);
    a.flat = true;
    a.write_parts = true;
    a.parts = parts;
    rc = rows_launch(s.plan, a, nkv, who, (cudaStream_t)stream);
  } else {
    rc = q_attention_parts_tc(d_q, prefix, d_prefix_len, parts.o, (float*)parts.ml, s.parts, batch * T, n_q_heads, scale,
                              stream);
    parts.keys = d_prefix_len;
    parts.tile = 128;
  }
  if (rc) return rc;
  // The sequences' own keys, under the prefix's launch: what they are made of is older than it, and the parts are
  // read at the end, behind the wait for it.
  RowsArgs a = rows_args(d_q, kv, d_pos, pos_per_seq, d_out, T, n_q_heads, scale);
  a.parts = parts;
  a.early = true;
  const RowsPlan p = rows_plan(batch * nkv, T * a.G, kv->pages_per_seq, true);
  return rows_launch(p, a, batch * nkv, who, (cudaStream_t)stream);
}
