// Causal attention over a whole prompt on the 5th-generation tensor cores (the prompt pass;
// reference: engine/prefill.py:45-52 calls the library's scaled-dot-product attention there).
//
// A work item is one (sequence, kv head, block of prompt tokens): two query tiles of 128 rows each
// (row = token, query head of the group: 128 / G tokens x G heads), which share every K/V tile of
// 128 keys (two pages). Per tile S = Q K^T (M = 128 query rows, N = 128 keys, fp32 in tensor
// memory), the softmax warps read their rows, write P as bf16 over S, and O += P V takes P from
// tensor memory and V from shared memory (keys are the K dimension there, so V is the operand whose
// other dimension is contiguous). Tensor memory is exactly S and O of the two query tiles.
//
// What bounds it: per query tile and key tile 16384 exponentials (16 per clock and SM: 1024 cycles)
// and 2 x 128 x 128 x 128 products (1024 cycles). Two query tiles let the tensor cores work on one
// while the softmax of the other runs; a CTA is persistent and starts the next item's first
// products under the current one's last softmax, since an item is only ~9 tiles long at 1-2 K keys.
//
// Warps 0-7 / 8-15: softmax and epilogue of query tile 0 / 1 (TILES = 1: all of one tile). Two (four) threads
// share a row (64 or 32 scores, then as many dims of O each) and exchange its maximum through shared memory: a step is a chain - scores,
// softmax, P V, next scores - and with one thread per row it took 4500 cycles, of which the softmax
// of 128 scores was more than half.
// Warp 16: producer lane. Warp 17: MMA issue; the whole warp walks the loop and one elected lane
// issues, so that descriptors live in uniform registers: an MMA of 128 x 128 x 16 takes 64 cycles,
// about what a single diverged lane needs to assemble its operands.
// O is rescaled only when some row of the warp has a new maximum. (In the causal form. Moving the maximum
// only after it had grown by 2^8 measured 367 against 390 us at 7000 tokens there, but the largest probability of a
// row is then no longer exactly 1 in bf16: error against fp64 2.1e-3 instead of 1.77e-3 where scores
// keep growing. The other two forms take that speed; what it costs them stands at the rescaling.) Cast boundaries as in attention.cu: fp32 scores and statistics, P rounded to bf16,
// fp32 accumulation, one rounding of the result.
//
// Tiles are read through tensor maps whose boxes undo the 256-byte row pitch of a page: a box of
// 64 rows x 64 dims lands as rows of 128 bytes, and the pages' own chunk swizzle (chunk ^ row & 7)
// is then the 128-byte swizzle the MMA descriptors name. Every wait is bounded.
//
// DEEP (one tile per CTA): the other half of tensor memory holds a second set of scores, so that those of the next
// key tile are there when the softmax of this one ends, and the tensor cores work under it; queries of the next item
// lie in the second tile's place. A step then waits for the softmax alone, not for the chain.
//
// Three forms (FORM) walk other keys with the same pipeline: CAUSAL (the prompt), WINDOW (the prompt under a
// sliding window with sinks: of the key tiles only those that hold a key some row of the item sees), PARTS (many
// rows over one range of keys that all of them see, cut into key splits whose m, l and O are left in 32 bits).
// In the last two any head count per kv head up to 32 is taken, k steps of 16 keys that nobody sees are left out
// of P V, and of a tile that nobody sees in one of its pages that page is not read.
#include "tc.cuh"
#include "attn_parts.cuh"

int* q_attn_status_addr();

namespace {

constexpr int AP_THREADS = 576;                            // 16 softmax warps, producer, MMA
constexpr int AP_KEYS = 128;                               // keys per tile
constexpr uint32_t AP_HALF = 128 * 128;                    // bytes of 128 rows x 64 dims
constexpr uint32_t AP_TILE = 2 * AP_HALF;                  // 128 rows x 128 dims
constexpr uint32_t AP_Q = 0, AP_K = 2 * AP_TILE, AP_V = AP_K + 2 * AP_TILE;
constexpr uint32_t AP_BARS = AP_V + 2 * AP_TILE;           // 192 KB in
constexpr uint32_t AP_RED = AP_BARS + 24 * 8 + 16;         // row exchange: [3][2 tiles x 2 or 4 parts][128] floats
constexpr size_t AP_SMEM = 1024 + AP_RED + 3 * 2 * 2 * 128 * 4;

enum { B_QF = 0, B_QE = 2, B_KF = 4, B_KE = 6, B_VF = 8, B_VE = 10, B_SF = 12, B_P = 14, B_OF = 18, B_OE = 20, B_PV = 22 };

struct AttnShape {
  int batch, T, G, gshift, nq, nkv, pages_per_seq;
  int tokens;        // prompt tokens per query tile: 128 / G
  int tiles;         // query tiles per work item: 2, or 1 where there are at most two for an SM
  int blocks;        // work items per (sequence, kv head)
  int items;
  int wide;          // the output is 32-byte aligned
  float scale_log2;
  int pos_step, window, sinks, room;     // WINDOW: positions per sequence, keys that the table's pages hold (PARTS: too)
  int far;                               // WINDOW: positions count up to it, so that their sums with T fit
  AttnParts parts;                       // PARTS
};

enum Form { CAUSAL, WINDOW, PARTS };

struct Item {
  int b, kh, q0, n, max_limit;
  int pos, low;                          // WINDOW: position of token 0, oldest key of the item's first window
  int sink_tiles, skip;                  // tile j is key tile j, + skip from sink_tiles on (PARTS: sink_tiles 0)
  int split;
};

__device__ __forceinline__ Item item_at(const AttnShape& sh, int w, int pos) {
  Item it;
  const int heads = sh.batch * sh.nkv;
  const int blk = w / heads, bh = w - blk * heads;
  it.b = bh / sh.nkv;
  it.kh = bh - it.b * sh.nkv;
  it.q0 = (sh.blocks - 1 - blk) * sh.tiles * sh.tokens;           // latest blocks (most keys) first
  it.max_limit = pos + min(it.q0 + sh.tiles * sh.tokens, sh.T);
  it.n = (it.max_limit + AP_KEYS - 1) / AP_KEYS;
  return it;
}
// `pos`: the position (CAUSAL), the number of keys (PARTS), nothing (WINDOW, where every sequence has its own).
template <int FORM>
__device__ __forceinline__ Item item_of_form(const AttnShape& sh, int w, int pos, const int32_t* pos_ptr) {
  if constexpr (FORM == CAUSAL) return item_at(sh, w, pos);
  Item it;
  if constexpr (FORM == WINDOW) {
    const int heads = sh.batch * sh.nkv;
    const int blk = w / heads, bh = w - blk * heads;
    it.b = bh / sh.nkv;
    it.kh = bh - it.b * sh.nkv;
    it.q0 = (sh.blocks - 1 - blk) * sh.tiles * sh.tokens;
    it.pos = min(max(__ldcg(pos_ptr + (size_t)it.b * sh.pos_step), 0), sh.far);
    it.max_limit = min(it.pos + min(it.q0 + sh.tiles * sh.tokens, sh.T), sh.room);
    it.low = max(0, it.pos + it.q0 - sh.window + 1);
    it.sink_tiles = (min(sh.sinks, it.max_limit) + AP_KEYS - 1) / AP_KEYS;
    // Nothing outside the table is read. A window that lies behind the pages still walks their last tile, of which
    // then no key is live and neither page is read: an item has one tile at least.
    const int last = (it.max_limit - 1) / AP_KEYS, first = max(it.sink_tiles, min(it.low / AP_KEYS, last));
    it.skip = first - it.sink_tiles;
    it.n = it.sink_tiles + max(0, last + 1 - first);
    it.split = 0;
  } else {
    // query blocks of a (split, kv head) next to one another: they share its keys in L2
    const int blk = w % sh.blocks, sk = w / sh.blocks;
    it.b = 0;
    it.split = sk / sh.nkv;
    it.kh = sk - it.split * sh.nkv;
    it.q0 = blk * sh.tiles * sh.tokens;
    it.max_limit = pos;
    it.pos = it.low = it.sink_tiles = 0;
    const int tiles = (pos + AP_KEYS - 1) / AP_KEYS, splits = min(sh.parts.splits, tiles);
    const int each = tiles / splits, more = tiles - each * splits;
    it.skip = it.split * each + min(it.split, more);
    it.n = each + (it.split < more ? 1 : 0);
  }
  return it;
}
// First key of an item's tile j.
template <int FORM>
__device__ __forceinline__ int key_base_of(const Item& it, int j) {
  if constexpr (FORM == CAUSAL) return j * AP_KEYS;
  return (j + (j >= it.sink_tiles ? it.skip : 0)) * AP_KEYS;
}
// The k steps (16 keys each) of a tile in which some row of the item sees a key.
template <int FORM>
__device__ __forceinline__ uint32_t live_steps(const AttnShape& sh, const Item& it, int key_base) {
  const int hi = min(AP_KEYS, it.max_limit - key_base);
  uint32_t live = (1u << ((hi + 15) >> 4)) - 1u;
  if (FORM == WINDOW && it.low > key_base) {
    const uint32_t near = 0xffu << (min(it.low - key_base, AP_KEYS) >> 4);
    const uint32_t far = (1u << ((min(max(sh.sinks - key_base, 0), AP_KEYS) + 15) >> 4)) - 1u;
    live &= near | far;
  }
  return live & 0xffu;
}
// The items of a CTA: rounds of gridDim.x, every other round backwards, so that the lengths (which
// fall with the item number) even out.
__device__ __forceinline__ int item_of(int round) {
  const int g = gridDim.x;
  return round * g + ((round & 1) ? g - 1 - (int)blockIdx.x : (int)blockIdx.x);
}

// The key tiles of a CTA's items in order.
template <int FORM>
struct Walk {
  Item it;
  int r, j;          // round of the item, tile of the item
  bool more;         // there is a tile here
  __device__ __forceinline__ void seek(const AttnShape& sh, int items, int pos, const int32_t* pos_ptr) {
    for (; r * (int)gridDim.x < items; ++r) {
      const int w = item_of(r);
      if (w < items) { it = item_of_form<FORM>(sh, w, pos, pos_ptr); j = 0; more = true; return; }
    }
    more = false;
  }
  __device__ __forceinline__ void next(const AttnShape& sh, int items, int pos, const int32_t* pos_ptr) {
    if (++j < it.n) return;
    ++r;
    seek(sh, items, pos, pos_ptr);
  }
};
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
// D[tmem] (+)= A[tmem] . B[smem desc]
__device__ __forceinline__ void tc_mma_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 columns of the warp's lanes; valid after tc_wait_ld and tc_pin32.
__device__ __forceinline__ void tc_ld32(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Keeps the compiler from using loaded registers before the wait.
__device__ __forceinline__ void tc_pin32(float* v) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]),
                      "+f"(v[i + 6]), "+f"(v[i + 7]));
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The lowest n bits (none for n <= 0, all from 32 on).
__device__ __forceinline__ uint32_t below(int n) { return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1u; }
// Two fp32 lanes per instruction, each rounded like the scalar one; and the largest of three.
__device__ __forceinline__ unsigned long long pair2(float a, float b) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpair2(unsigned long long r, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r));
}
__device__ __forceinline__ unsigned long long fma2(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ unsigned long long add2(unsigned long long a, unsigned long long b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int TILES, int FORM, bool DEEP>
__global__ void __launch_bounds__(AP_THREADS, 1)
k_attn_prompt(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
              const __grid_constant__ CUtensorMap vmap, const int32_t* __restrict__ block_table,
              const int32_t* __restrict__ pos_ptr, bf16* __restrict__ out, AttnShape sh, int* status) {
  static_assert(!DEEP || (TILES == 1 && FORM != CAUSAL), "one tile of the other forms");
  constexpr int WARPS = TILES == 2 ? 8 : 16;               // softmax warps of a query tile
  constexpr int PER_ROW = WARPS / 4, COLS = 128 / PER_ROW; // threads of a row, scores (and dims of O) of each
  extern __shared__ unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* smem = smem_raw + (base - raw);
  const uint32_t bars = base + AP_BARS;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + AP_BARS + 24 * 8);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  auto bar = [&](int kind, int i) { return bars + 8u * (uint32_t)(kind + i); };

  if (FORM == CAUSAL) pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
    for (int i = 0; i < 24; ++i) {
      const bool warps = i >= B_P && i < B_P + 4;          // half a tile's softmax warps arrive (all at the epilogue)
      mbar_init(bars + 8u * i, i >= B_OE && i < B_OE + 2 ? WARPS : warps ? WARPS / 2 : 1);
    }
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 16 && lane == 0) {
    prefetch_map(&qmap);
    prefetch_map(&kmap);
    prefetch_map(&vmap);
  }
  if (warp == 17) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // All 512 columns are this CTA's, so its tensor memory starts at column 0.
  constexpr uint32_t tmem = 0;
  // q, this pass's K/V rows, and also the position and the block table: a caller's own kernel before this
  // one may write those. All are requested at once, behind the wait: reading position and pages before
  // it, as the decode kernel does, gained 1 us in a prompt of 64 tokens (12 layers, 1128.7 / 1129.6 us).
  pdl_wait();
  // (the other forms' dependents may read early whatever the launches before this one wrote)
  if (FORM != CAUSAL) pdl_launch_dependents();
  int pos = FORM == WINDOW ? 0 : *reinterpret_cast<const volatile int32_t*>(pos_ptr);
  int items = sh.items;
  if (FORM == PARTS) {
    pos = min(max(pos, 0), sh.room);
    items = min(sh.parts.splits, (pos + AP_KEYS - 1) / AP_KEYS) * sh.nkv * sh.blocks;
  }
  // with fewer tiles than splits some CTAs have no item
  const bool idle = FORM == PARTS && item_of(0) >= items;
  int first_page[2] = {0, 0};
  if (FORM == CAUSAL && warp == 16) {                      // the grid has at most one CTA per item
    const volatile int32_t* table = block_table + (size_t)item_at(sh, item_of(0), 0).b * sh.pages_per_seq;
    first_page[0] = table[0];
    first_page[1] = table[min(1, sh.pages_per_seq - 1)];
  }

  if (warp == 16) {
    // ---------------- producer ----------------
    if (lane == 0) {
      uint32_t step = 0;                                   // K/V tiles requested so far
      uint32_t nitems = 0;
      bool ok = true;
      auto fail = [&]() { atomicExch(status, 7); *abort_flag = 1; ok = false; };
      if constexpr (DEEP) {
        // keys run one tile ahead of values: their place is free as soon as their scores are
        Walk<FORM> k, v;
        k.r = v.r = 0;
        k.seek(sh, items, pos, pos_ptr);
        v = k;
        uint32_t ksteps = 0, vsteps = 0;
        auto load = [&](const Walk<FORM>& at, bool values, uint32_t n) {
          const int key_base = key_base_of<FORM>(at.it, at.j), first = key_base / Q_PAGE_TOKENS;
          const uint32_t live = live_steps<FORM>(sh, at.it, key_base);
          const int32_t* table = block_table + (size_t)at.it.b * sh.pages_per_seq;
          const int p0 = live & 0x0fu ? 0 : 1, np = live & 0xf0u ? 2 : 1;      // a page that nobody sees is not read
          const int page0 = p0 == 0 ? __ldcg(table + first) : 0, page1 = np == 2 ? __ldcg(table + first + 1) : 0;
          const int s = n & 1;
          if (!mbar_wait(bar(values ? B_VE : B_KE, s), ((n >> 1) & 1) ^ 1, abort_flag)) { fail(); return; }
          const uint32_t full = bar(values ? B_VF : B_KF, s), dst = base + (values ? AP_V : AP_K) + s * AP_TILE;
          mbar_expect_tx(full, (uint32_t)(np - p0) * AP_HALF);
          for (int p = p0; p < np; ++p)
            for (int h = 0; h < 2; ++h)
              tma_load_4d(dst + h * AP_HALF + p * (AP_HALF / 2), values ? &vmap : &kmap, 0, h, 0,
                          (p ? page1 : page0) * sh.nkv + at.it.kh, full);
        };
        while (ok && v.more) {
          if (k.more) {
            if (k.j == 0) {
              const int slot = nitems & 1;
              if (!mbar_wait(bar(B_QE, slot), ((nitems >> 1) & 1) ^ 1, abort_flag)) { fail(); break; }
              mbar_expect_tx(bar(B_QF, slot), (uint32_t)(sh.tokens * sh.G) * 256u);
              for (int h = 0; h < 2; ++h)
                tma_load_3d(base + AP_Q + slot * AP_TILE + h * AP_HALF, &qmap, 64 * h, k.it.kh * sh.G,
                            k.it.b * sh.T + k.it.q0, bar(B_QF, slot));
              ++nitems;
            }
            load(k, false, ksteps);
            if (!ok) break;
            ++ksteps;
            k.next(sh, items, pos, pos_ptr);
          }
          if (ksteps < 2 && k.more) continue;              // (the first two tiles' keys go first)
          load(v, true, vsteps);
          if (!ok) break;
          ++vsteps;
          v.next(sh, items, pos, pos_ptr);
        }
        // copies in flight must land before the CTA may leave
        for (uint32_t i = 0; i < 2; ++i) {
          if (nitems > i) mbar_wait_plain(bar(B_QF, (nitems - 1 - i) & 1), ((nitems - 1 - i) >> 1) & 1);
          if (ksteps > i) mbar_wait_plain(bar(B_KF, (ksteps - 1 - i) & 1), ((ksteps - 1 - i) >> 1) & 1);
          if (vsteps > i) mbar_wait_plain(bar(B_VF, (vsteps - 1 - i) & 1), ((vsteps - 1 - i) >> 1) & 1);
        }
        nitems = 0;
      } else
      for (int r = 0; ok && r * (int)gridDim.x < items; ++r) {
        const int w = item_of(r);
        if (w >= items) continue;
        const Item it = item_of_form<FORM>(sh, w, pos, pos_ptr);
        for (int i = 0; ok && i < TILES; ++i) {
          if (!mbar_wait(bar(B_QE, i), (nitems & 1) ^ 1, abort_flag)) { fail(); break; }
          const int tok = it.b * sh.T + it.q0 + i * sh.tokens;
          mbar_expect_tx(bar(B_QF, i), FORM == CAUSAL ? AP_TILE : (uint32_t)(sh.tokens * sh.G) * 256u);
          for (int h = 0; h < 2; ++h)
            tma_load_3d(base + AP_Q + i * AP_TILE + h * AP_HALF, &qmap, 64 * h, it.kh * sh.G, tok, bar(B_QF, i));
        }
        const int32_t* table = block_table + (size_t)it.b * sh.pages_per_seq;
        const int npages = (it.max_limit + Q_PAGE_TOKENS - 1) / Q_PAGE_TOKENS;
        for (int j = 0; ok && j < it.n; ++j, ++step) {
          const int s = step & 1;
          const uint32_t parity = ((step >> 1) & 1) ^ 1;
          int np = min(2, npages - 2 * j), page0, page1, p0 = 0;
          if constexpr (FORM == CAUSAL) {
            page0 = step ? table[2 * j] : first_page[0];
            page1 = np < 2 ? 0 : step ? table[2 * j + 1] : first_page[1];
          } else {
            const int key_base = key_base_of<FORM>(it, j), at = key_base / Q_PAGE_TOKENS;
            const uint32_t live = live_steps<FORM>(sh, it, key_base);
            p0 = live & 0x0fu ? 0 : 1;                     // a page that nobody sees is not read, nor its table entry
            np = live & 0xf0u ? 2 : 1;
            page0 = p0 == 0 ? __ldcg(table + at) : 0;
            page1 = np == 2 ? __ldcg(table + at + 1) : 0;
          }
          for (int kv = 0; kv < 2; ++kv) {
            if (!mbar_wait(bar(kv ? B_VE : B_KE, s), parity, abort_flag)) { fail(); break; }
            const uint32_t full = bar(kv ? B_VF : B_KF, s);
            const uint32_t dst = base + (kv ? AP_V : AP_K) + s * AP_TILE;
            mbar_expect_tx(full, (uint32_t)(np - p0) * AP_HALF);
            for (int p = p0; p < np; ++p)
              for (int h = 0; h < 2; ++h)
                tma_load_4d(dst + h * AP_HALF + p * (AP_HALF / 2), kv ? &vmap : &kmap, 0, h, 0,
                            (p ? page1 : page0) * sh.nkv + it.kh, full);
          }
        }
        ++nitems;
      }
      // copies in flight must land before the CTA may leave
      for (int i = 0; i < 2; ++i) {
        if (nitems > 0 && i < TILES) mbar_wait_plain(bar(B_QF, i), (nitems - 1) & 1);
        if (step > (uint32_t)i) {
          const uint32_t last = ((step - 1 - i) >> 1) & 1;
          mbar_wait_plain(bar(B_KF, (step - 1 - i) & 1), last);
          mbar_wait_plain(bar(B_VF, (step - 1 - i) & 1), last);
        }
      }
      if (!ok) {                                           // ... also those of a step that was given up half-way
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) __nanosleep(1000);
      }
    }
  } else if (warp == 17) {
    // ---------------- MMA issuer ----------------
    {
      const uint32_t f16 = (1u << 4) | (1u << 7) | (1u << 10) | (16u << 17) | (8u << 24);   // 128 x 128, fp32 sums
      const uint32_t idesc_s = f16, idesc_pv = f16 | (1u << 16);      // V: the non-contracted dimension is contiguous
      const uint64_t q_desc = smem_desc(base + AP_Q), k_desc = smem_desc(base + AP_K);
      // V: leading offset = the other 64 dims, stride offset = the next 8 keys
      const uint64_t v_desc = (uint64_t)(((base + AP_V) & 0x3FFFFu) >> 4) | ((uint64_t)(AP_HALF >> 4) << 16) |
                              (64ull << 32) | (1ull << 46) | (2ull << 61);
      uint32_t kstep = 0, vstep = 0, nitems = 0;
      bool ok = true;
      auto wait = [&](uint32_t b, uint32_t parity) {
        const int landed = mbar_wait(b, parity, abort_flag) ? 1 : 0;
        if (!__all_sync(0xffffffffu, landed)) {
          if (elect_one()) { atomicExch(status, 8); *abort_flag = 1; }
          ok = false;
        }
        tc_fence_after();
        return ok;
      };
      auto scores = [&](int i) {                           // S_i = Q_i K^T of the K tile at kstep
        const uint64_t a = q_desc + (uint64_t)(i * (AP_TILE >> 4)), b = k_desc + (uint64_t)((kstep & 1) * (AP_TILE >> 4));
        if (!elect_one()) return;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t off = (uint32_t)(ks >> 2) * (AP_HALF >> 4) + (ks & 3) * 2;
          tc_mma(tmem + 128u * i, a + off, b + off, idesc_s, ks ? 1u : 0u);
        }
        tc_commit(bar(B_SF, i));
      };
      if constexpr (DEEP) {
        Walk<FORM> s, v;                                   // tiles of the next scores and the next products
        s.r = 0;
        s.seek(sh, items, pos, pos_ptr);
        v = s;
        uint32_t qitems = 0;                               // items whose queries have been waited for
        auto ahead = [&]() {                               // scores of the tile at s into the buffer of its parity
          if (s.j == 0) {
            if (!wait(bar(B_QF, qitems & 1), (qitems >> 1) & 1)) return;
            ++qitems;
          }
          if (!wait(bar(B_KF, kstep & 1), (kstep >> 1) & 1)) return;
          const uint32_t buf = kstep & 1, slot = (qitems - 1) & 1;
          const uint64_t a = q_desc + (uint64_t)(slot * (AP_TILE >> 4)), b = k_desc + (uint64_t)(buf * (AP_TILE >> 4));
          const bool last = s.j + 1 == s.it.n;
          if (elect_one()) {
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
              const uint32_t off = (uint32_t)(ks >> 2) * (AP_HALF >> 4) + (ks & 3) * 2;
              tc_mma(tmem + 128u * buf, a + off, b + off, idesc_s, ks ? 1u : 0u);
            }
            tc_commit(bar(B_SF, buf));
            tc_commit(bar(B_KE, buf));
            if (last) tc_commit(bar(B_QE, slot));
          }
          __syncwarp();
          ++kstep;
          s.next(sh, items, pos, pos_ptr);
        };
        for (int i = 0; i < 2 && ok && s.more; ++i) ahead();
        while (ok && v.more) {
          const uint32_t buf = vstep & 1, parity = (vstep >> 1) & 1;
          const int key_base = key_base_of<FORM>(v.it, v.j);
          const bool last = v.j + 1 == v.it.n;
          const uint32_t live = live_steps<FORM>(sh, v.it, key_base);
          if (!wait(bar(B_VF, buf), parity)) break;
          if (v.j == 0 && !wait(bar(B_OE, 0), (nitems & 1) ^ 1)) break;
          if (!wait(bar(B_P, 2 * buf), parity) || !wait(bar(B_P, 2 * buf + 1), parity)) break;
          const bool first = v.j == 0;
          v.next(sh, items, pos, pos_ptr);
          if (elect_one()) {
            const uint64_t b = v_desc + (uint64_t)(buf * (AP_TILE >> 4));
            if (live == 0xffu) {
#pragma unroll
              for (int ks = 0; ks < 8; ++ks)
                tc_mma_ta(tmem + 256u, tmem + 128u * buf + 8u * ks, b + (uint64_t)(ks * (2048 >> 4)), idesc_pv, (!first || ks) ? 1u : 0u);
            } else {
              uint32_t sum = first ? 0u : 1u;
#pragma unroll 1
              for (int ks = 0; ks < 8; ++ks) {
                if (!((live >> ks) & 1u)) continue;
                tc_mma_ta(tmem + 256u, tmem + 128u * buf + 8u * ks, b + (uint64_t)(ks * (2048 >> 4)), idesc_pv, sum);
                sum = 1u;
              }
            }
            // (nothing after the last tile's: nobody waits for it any more, and the arrival could find that the CTA has left)
            if (v.more) {
              tc_commit(bar(B_VE, buf));
              tc_commit(bar(B_PV, 0));
            }
            if (last) tc_commit(bar(B_OF, 0));
          }
          __syncwarp();
          ++vstep;
          if (last) ++nitems;
          if (s.more) ahead();
        }
        ok = false;                                        // (nothing is left)
      }
      int r = 0;
      if (DEEP || idle) ok = false;                        // (nothing is waited for)
      Item cur = {};
      if (ok) cur = item_of_form<FORM>(sh, item_of(0), pos, pos_ptr);      // the grid has at most one CTA per item
      for (int i = 0; i < TILES && ok; ++i) {
        if (!wait(bar(B_QF, i), 0) || (i == 0 && !wait(bar(B_KF, 0), 0))) break;
        scores(i);
        if (elect_one() && cur.n == 1) tc_commit(bar(B_QE, i));
        __syncwarp();
      }
      if (ok) {
        if (elect_one()) tc_commit(bar(B_KE, 0));
        ++kstep;
      }
      while (ok) {
        // the item after this one
        bool more = false;
        Item nxt = cur;
        for (++r; r * (int)gridDim.x < items; ++r) {
          const int w = item_of(r);
          if (w < items) { nxt = item_of_form<FORM>(sh, w, pos, pos_ptr); more = true; break; }
        }
        for (int j = 0; ok && j < cur.n; ++j) {
          const bool last = j + 1 == cur.n, ahead = !last || more;
          const int vs = vstep & 1;
          if (!wait(bar(B_VF, vs), (vstep >> 1) & 1)) break;
          for (int i = 0; i < TILES && ok; ++i) {
            if (j == 0 && !wait(bar(B_OE, i), (nitems & 1) ^ 1)) break;
            // P comes in two halves of 64 keys, from different warps
            if (!wait(bar(B_P, 2 * i), vstep & 1) || !wait(bar(B_P, 2 * i + 1), vstep & 1)) break;
            const int keys = cur.max_limit - key_base_of<FORM>(cur, j);  // in the last tile, k steps past the newest key are left out
            uint32_t live = 0;
            if (FORM == WINDOW) live = live_steps<FORM>(sh, cur, key_base_of<FORM>(cur, j));
            if (elect_one()) {
              if (FORM == WINDOW && live != 0xffu) {
                uint32_t sum = j ? 1u : 0u;
#pragma unroll 1
                for (int ks = 0; ks < 8; ++ks) {
                  if (!((live >> ks) & 1u)) continue;
                  tc_mma_ta(tmem + 256u + 128u * i, tmem + 128u * i + 8u * ks,
                            v_desc + (uint64_t)(vs * (AP_TILE >> 4) + ks * (2048 >> 4)), idesc_pv, sum);
                  sum = 1u;
                }
              } else if (keys >= AP_KEYS) {
#pragma unroll
                for (int ks = 0; ks < 8; ++ks)
                  tc_mma_ta(tmem + 256u + 128u * i, tmem + 128u * i + 8u * ks,
                            v_desc + (uint64_t)(vs * (AP_TILE >> 4) + ks * (2048 >> 4)), idesc_pv, (j | ks) ? 1u : 0u);
              } else {
#pragma unroll 1
                for (int ks = 0; 16 * ks < keys; ++ks)
                  tc_mma_ta(tmem + 256u + 128u * i, tmem + 128u * i + 8u * ks,
                            v_desc + (uint64_t)(vs * (AP_TILE >> 4) + ks * (2048 >> 4)), idesc_pv, (j | ks) ? 1u : 0u);
              }
            }
            __syncwarp();
            if (!ok) break;
            if (last && elect_one()) tc_commit(bar(B_OF, i));
            if (ahead) {
              if (i == 0 && !wait(bar(B_KF, kstep & 1), (kstep >> 1) & 1)) break;
              if (last && !wait(bar(B_QF, i), (nitems + 1) & 1)) break;
              scores(i);
              if (elect_one() && (last ? nxt.n == 1 : j + 2 == cur.n)) tc_commit(bar(B_QE, i));
              __syncwarp();
            }
          }
          if (!ok) break;
          // (not after the last tile: nobody waits for it any more, and the arrival could find that the
          // CTA has left)
          if (ahead && elect_one()) {
            tc_commit(bar(B_VE, vs));
            tc_commit(bar(B_KE, kstep & 1));
          }
          __syncwarp();
          ++vstep;
          if (ahead) ++kstep;
        }
        ++nitems;
        if (!more) break;
        cur = nxt;
      }
    }
  } else {
    // ---------------- softmax and epilogue: query tile `i`, half (a quarter) of a row per thread ----------------
    const int i = TILES == 2 ? warp >> 3 : 0, part = TILES == 2 ? (warp >> 2) & 1 : warp >> 2;
    const int row = tid & 127;
    float* red = reinterpret_cast<float*>(smem + AP_RED) + i * 256;        // [buffer * 512 + part * 128 + row]
    auto tile_sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(1 + i), "n"(WARPS * 32) : "memory"); };
    const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
    uint32_t s_addr = tmem + lanes + 128u * i + (uint32_t)(COLS * part), p_addr = tmem + lanes + 128u * i + (uint32_t)(COLS / 2 * part);
    const uint32_t o_addr = tmem + lanes + 256u + 128u * i + (uint32_t)(COLS * part);
    // A scale that is not positive (the maximum would sit elsewhere) is multiplied in first.
    const bool plain = sh.scale_log2 > 0.f;
    const float c = plain ? sh.scale_log2 : 1.f;
    uint32_t step = 0, nitems = 0;
    // A warp whose wait ran out keeps coming to the tile's barriers; at the item's end all its tile's
    // warps learn of it and leave together.
    bool broken = false;
    auto wait = [&](uint32_t b, uint32_t parity) {
      const int landed = broken || mbar_wait(b, parity, abort_flag) ? 1 : 0;
      if (!__all_sync(0xffffffffu, landed)) {
        if (lane == 0) { atomicExch(status, 9); *abort_flag = 1; }
        broken = true;
      }
      tc_fence_after();
    };
    for (int r = 0; r * (int)gridDim.x < items; ++r) {
      const int w = item_of(r);
      if (w >= items) continue;
      const Item it = item_of_form<FORM>(sh, w, pos, pos_ptr);
      // token and head of the row (128 rows hold `tokens` tokens of G heads; with an odd G the last rows are nobody's)
      const int tok = FORM == CAUSAL ? row >> sh.gshift : row / sh.G;
      const int t = it.q0 + i * sh.tokens + tok;
      const bool live_row = t < sh.T && (FORM == CAUSAL || tok < sh.tokens);
      int limit, free_keys, low = 0, free_from = 0;        // the row sees [low, limit) and the sinks
      if constexpr (FORM == CAUSAL) {
        limit = t < sh.T ? pos + t + 1 : 0;                // a row past the prompt sees nothing
        // keys that every row of this warp sees: tiles inside them need no mask
        const int t_first = it.q0 + i * sh.tokens + (((warp & 3) * 32) >> sh.gshift);
        const int t_last = it.q0 + i * sh.tokens + (((warp & 3) * 32 + 31) >> sh.gshift);
        free_keys = t_last < sh.T ? pos + t_first + 1 : 0;
      } else if constexpr (FORM == WINDOW) {
        limit = min(it.pos + t + 1, sh.room);
        low = max(0, it.pos + t + 1 - sh.window);
        free_keys = min(it.pos + it.q0 + i * sh.tokens + (warp & 3) * 32 / sh.G + 1, sh.room);
        free_from = it.pos + it.q0 + i * sh.tokens + ((warp & 3) * 32 + 31) / sh.G + 1 - sh.window;
      } else {
        limit = free_keys = pos;
      }
      float m = -INFINITY, l = 0.f;
      for (int j = 0; j < it.n; ++j, ++step) {
        const uint32_t buf = DEEP ? step & 1 : (uint32_t)i;
        if (DEEP) {
          s_addr = tmem + lanes + 128u * buf + (uint32_t)(COLS * part);
          p_addr = tmem + lanes + 128u * buf + (uint32_t)(COLS / 2 * part);
        }
        wait(bar(B_SF, buf), DEEP ? (step >> 1) & 1 : step & 1);
        float v[COLS];
        if constexpr (TILES == 2) {
          tc_ld32(s_addr, v);
          tc_ld32(s_addr + 32, v + 32);
          tc_wait_ld();
          tc_pin32(v);
          tc_pin32(v + 32);
        } else {
          float lo[16], hi[16];
          tc_ld16(s_addr, lo);
          tc_ld16(s_addr + 16, hi);
#pragma unroll
          for (int k = 0; k < 16; ++k) { v[k] = lo[k]; v[k + 16] = hi[k]; }
        }
        const int key_base = key_base_of<FORM>(it, j);
        if (!plain) {
#pragma unroll
          for (int k = 0; k < COLS; ++k) v[k] *= sh.scale_log2;
        }
        if (FORM == WINDOW) {
          if (key_base + AP_KEYS > free_keys || (key_base < free_from && key_base + AP_KEYS > sh.sinks)) {
            // a bit per score: with three comparisons each a tile took 1900 cycles more, of 3400
#pragma unroll
            for (int h = 0; h < COLS; h += 32) {
              const int at = key_base + COLS * part + h;
              const uint32_t seen = below(limit - at) & (~below(low - at) | below(sh.sinks - at));
#pragma unroll
              for (int k = 0; k < 32; ++k) v[h + k] = seen & (1u << k) ? v[h + k] : -INFINITY;
            }
          }
        } else if (key_base + AP_KEYS > free_keys) {
          const int vis = limit - key_base - COLS * part;
#pragma unroll
          for (int k = 0; k < COLS; ++k) v[k] = k < vis ? v[k] : -INFINITY;
        }
        if (FORM == WINDOW) {
          // V rows that no row of the item sees are cleared where their k step takes part in P V
          if (tid < 128 && (key_base + AP_KEYS > it.max_limit || key_base < it.low)) {
            const int key = key_base + tid;
            const bool stale = ((live_steps<FORM>(sh, it, key_base) >> (tid >> 4)) & 1u) &&
                               (key >= it.max_limit || (key < it.low && key >= sh.sinks));
            if (__any_sync(0xffffffffu, stale)) {
              wait(bar(B_VF, step & 1), (step >> 1) & 1);
              if (stale && !broken) {
                unsigned char* vt = smem + AP_V + (step & 1) * AP_TILE + tid * 128;
#pragma unroll
                for (int q = 0; q < 16; ++q)
                  *reinterpret_cast<uint4*>(vt + (q & 8 ? AP_HALF : 0u) + ((q & 7) << 4)) = make_uint4(0, 0, 0, 0);
              }
              asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
              __syncwarp();
            }
          }
        } else if (tid < 128 && key_base + AP_KEYS > it.max_limit && (it.max_limit & 15)) {
          // V rows past the newest key hold stale bits (0 * garbage could be NaN): clear those of its
          // k step before the first product with this tile may start
          wait(bar(B_VF, step & 1), (step >> 1) & 1);
          unsigned char* vt = smem + AP_V + (step & 1) * AP_TILE;
          const int live = it.max_limit - key_base;
          for (int q = tid; !broken && q < ((16 - live) & 15) * 16; q += 128) {
            const int kr = live + (q >> 4);
            *reinterpret_cast<uint4*>(vt + (q & 8 ? AP_HALF : 0u) + kr * 128 + ((q & 7) << 4)) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
        }
        float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
        for (int k = 4; k < COLS - 4; k += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], v[k + e], v[k + 4 + e]);
        float m_tile = max3(max3(mx[0], mx[1], mx[2]), mx[3], fmaxf(max3(v[COLS - 4], v[COLS - 3], v[COLS - 2]), v[COLS - 1]));
        // the row's other parts; this barrier also says that all of S is in registers, so that P may
        // overwrite it
        red[(step & 1) * 512 + part * 128 + row] = m_tile;
        tc_fence_before();
        tile_sync();
        tc_fence_after();
#pragma unroll
        for (int e = 1; e < PER_ROW; ++e) m_tile = fmaxf(m_tile, red[(step & 1) * 512 + (part ^ e) * 128 + row]);
        if (j == 0) {
          m = m_tile;
        } else {
          // (the other forms let it grow by 2^8 first: over few tiles some row of a warp has a new maximum in nearly
          // each, and reading and writing O took a quarter of a step. P is then at most 256, as exact in bf16 as up to
          // 1; only a row's largest is no longer exactly 1. At once / after 2^8, us: a prompt of 7000 tokens under a window
          // of 1024 176 / 165, under 4096 365 / 339, 3 x 701 50.5 / 48.0, 64 x 2 tokens over a prefix of 30001 82.8 / 77.9. Error
          // against fp64, relative 2-norm, of unit normals 2.12e-3 / 2.20e-3 (windows), 2.26e-3 / 2.33e-3 (prefixes); where
          // keys grow from 0.05 to 4 times that along the context 1.78e-3 / 2.19e-3 and 1.72e-3 / 2.09e-3, the largest error,
          // of the largest result, 2.3e-3 / 4.7e-3 and 2.1e-3 / 3.8e-3. The result's own rounding is 1.66e-3 of that.)
          if (__any_sync(0xffffffffu, FORM == CAUSAL ? m_tile > m : (m_tile - m) * c > 8.f)) {
            // the products up to the tile before are complete: this tile's scores came after them (DEEP: after those
            // of the tile before that, so that the parity of the last ones names them)
            if (DEEP) wait(bar(B_PV, 0), (step - 1) & 1);
            const float m_new = fmaxf(m, m_tile);
            const float f = m_new == m ? 1.f : ex2((m - m_new) * c);
            l *= f;
            m = m_new;
#pragma unroll 1
            for (int k = 0; k < COLS / 16; ++k) {
              float o[16];
              uint32_t u[16];
              tc_ld16(o_addr + 16 * k, o);
#pragma unroll
              for (int e = 0; e < 16; ++e) u[e] = __float_as_uint(o[e] * f);
              tc_st16(o_addr + 16 * k, u);
            }
            tc_wait_st();
          }
        }
        const float mc = m == -INFINITY ? 0.f : m * c;
        const unsigned long long c2 = pair2(c, c), mc2 = pair2(-mc, -mc);
        unsigned long long sum[2] = {0ull, 0ull};
#pragma unroll
        for (int h = 0; h < COLS / 32; ++h) {
          uint32_t p[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float a, b;
            unpair2(fma2(pair2(v[32 * h + 2 * k], v[32 * h + 2 * k + 1]), c2, mc2), a, b);
            a = ex2(a);
            b = ex2(b);
            sum[k & 1] = add2(sum[k & 1], pair2(a, b));
            p[k] = pack_bf16(a, b);
          }
          tc_st16(p_addr + 16 * h, p);
        }
        tc_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_P, 2 * buf + part / (PER_ROW / 2)));
        __syncwarp();
        float s_lo, s_hi;
        unpair2(add2(sum[0], sum[1]), s_lo, s_hi);
        l += s_lo + s_hi;
      }
      red[1024 + part * 128 + row] = l;
      int give_up;
      asm volatile(
          "{\n\t.reg .pred p, q;\n\t"
          "setp.ne.u32 q, %1, 0;\n\t"
          "barrier.cta.red.or.pred p, %2, %3, q;\n\t"
          "selp.u32 %0, 1, 0, p;\n\t}"
          : "=r"(give_up) : "r"((int)broken), "r"(1 + i), "n"(WARPS * 32) : "memory");
      if (give_up) break;
      {
        float all = red[1024 + row];                       // (in the same order in all threads of a row)
#pragma unroll
        for (int e = 1; e < PER_ROW; ++e) all += red[1024 + e * 128 + row];
        l = all;
      }
      wait(bar(B_OF, i), nitems & 1);
      if (broken) { ++nitems; continue; }
      if constexpr (FORM == PARTS) {
        const size_t prow = sh.parts.row(it.split, it.kh, (size_t)t * sh.G + (row - tok * sh.G));
        float* to = sh.parts.o + prow * 128 + COLS * part;
        if (live_row && part == 0) sh.parts.ml[prow] = make_float2(m * c, l);
#pragma unroll 1
        for (int k = 0; k < COLS / 16; ++k) {
          float o[16];
          tc_ld16(o_addr + 16 * k, o);
          if (live_row) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
              *reinterpret_cast<float4*>(to + 16 * k + 4 * q) = make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
          }
          __syncwarp();
        }
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar(B_OE, i));
        __syncwarp();
        ++nitems;
        continue;
      }
      const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);      // NaN stays NaN
      const bool none = FORM == WINDOW && l == 0.f;        // (O may never have been written)
      const int head = FORM == CAUSAL ? row & (sh.G - 1) : row - tok * sh.G;
      bf16* dst = out + (((size_t)it.b * sh.T + t) * sh.nq + it.kh * sh.G + head) * 128 + COLS * part;
#pragma unroll 1
      for (int k = 0; k < COLS / 16; ++k) {
        float o[16];
        tc_ld16(o_addr + 16 * k, o);
        if (live_row) {
          uint32_t u[8];
#pragma unroll
          for (int q = 0; q < 8; ++q) u[q] = none ? 0u : pack_bf16(o[2 * q] * inv, o[2 * q + 1] * inv);
          if (sh.wide) {
            asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                         ::"l"(dst + 16 * k), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]),
                         "r"(u[6]), "r"(u[7]) : "memory");
          } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) *reinterpret_cast<uint32_t*>(dst + 16 * k + 2 * q) = u[q];
          }
        }
        __syncwarp();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(bar(B_OE, i));
      __syncwarp();
      ++nitems;
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 17) {
    __syncwarp();
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
}

// What q_attention_prefill, its windowed form and the partial form share. FORM WINDOW and PARTS fill their own
// fields of `sh` before; d_out null for PARTS.
template <int FORM>
int prompt_launch(const char* who, AttnShape& sh, const void* d_q, const q_kv_layout_t* kv, const int32_t* d_pos,
                  void* d_out, int batch, int T, int n_q_heads, float scale, void* stream) {
  Q_CHECK_ARG(d_q && kv && d_pos && (d_out || FORM == PARTS), "%s: null pointer", who);
  Q_CHECK_ARG(kv->d_kpool && kv->d_vpool && kv->d_block_table && kv->pages_per_seq >= 1 &&
                  kv->n_kv_heads >= 1,
              "%s: incomplete KV layout", who);
  const int nkv = kv->n_kv_heads;
  Q_CHECK_ARG(batch >= 1 && batch <= 65535 && nkv <= 65535 && T >= 1 && n_q_heads >= nkv &&
                  n_q_heads % nkv == 0,
              "%s: bad batch/T/heads", who);
  const int G = n_q_heads / nkv;
  if (FORM == CAUSAL) {
    Q_CHECK_ARG(G <= 8 && (G & (G - 1)) == 0,
                "%s: %d query heads per kv head (1, 2, 4 or 8 supported)", who, G);
  } else {
    Q_CHECK_ARG(G <= 32, "%s: %d query heads per kv head exceed 32", who, G);
    Q_CHECK_ARG(kv->pages_per_seq <= (1 << 23), "%s: too many pages per sequence", who);
    Q_CHECK_ALIGN(d_pos, 4, who); Q_CHECK_ALIGN(kv->d_block_table, 4, who);
  }
  Q_CHECK_ALIGN(d_q, 16, who); Q_CHECK_ALIGN(d_out, 4, who);
  Q_CHECK_ALIGN(kv->d_kpool, 16, who); Q_CHECK_ALIGN(kv->d_vpool, 16, who);
  int* status = q_attn_status_addr();
  if (!status) { q_set_error("%s: could not locate the device status word", who); return Q_ERR_CUDA; }
  sh.batch = batch; sh.T = T; sh.G = G; sh.nq = n_q_heads; sh.nkv = nkv; sh.pages_per_seq = kv->pages_per_seq;
  sh.room = FORM == CAUSAL ? 0 : kv->pages_per_seq * Q_PAGE_TOKENS;
  sh.gshift = 0;
  while ((1 << sh.gshift) < G) ++sh.gshift;
  sh.tokens = 128 / G;
  // Two tiles of a CTA hide each other's latencies; one tile has all 16 softmax warps, four threads to a row, and a
  // shorter chain. Up to two tiles per SM the one is faster. One tile / two, us: 1 x 592 tokens 15.5 / 18.8, 1 x 1024
  // 22.8 / 26.4, 1 x 1184 (296 tiles) 28.8 / 30.7, 3 x 250 10.2 / 12.8, 9 x 128 10.2 / 10.5, but 1 x 1200 32.4 / 31.8,
  // 3 x 400 (312) 19.4 / 17.0, 2 x 701 26.9 / 22.8. (With half of the warps idle, one tile took 17.1 at 592.)
  // These are the causal form's; one tile of the other forms is DEEP. Windows, 32 / 8 heads, one / two, us: 1.7 row tiles per
  // SM (1 x 1024) 19.5 / 22.7, 2.0 (1 x 1184 behind 2000, window 1024) 36.2 / 62.5, 2.4 (2 x 701 behind 1000, 512) 39.8 / 47.3,
  // 3.6 (3 x 701) 51.6 / 48.0, 4.8 (4 x 701) 63.4 / 69.5, 7.1 (6 x 701) 101.9 / 91.3, 11.8 (1 x 7000, 1024) 182 / 165: up to
  // two and from six on the rule holds; between them it goes by how full the last round of items is, which the rule does not
  // look at. Prefixes, row tiles: 1 (32 x 16384) 25.8 / 32.8, 2 (64 x 16384) 34.0 / 37.8, 3 (96 x 16384) 45.6 / 54.1, 4 (64 x 2
  // over 4096) 27.9 / 32.3 but over 30001 86.3 / 78.0, 8 (128 x 2 over 8192) 69.3 / 69.6.
  const int sms = q_sm_count();
  const long long row_tiles = (T + sh.tokens - 1) / sh.tokens;
  if (FORM == PARTS) sh.tiles = row_tiles == 1 ? 1 : 2;
  else sh.tiles = row_tiles * batch * nkv <= 2ll * sms ? 1 : 2;
  sh.blocks = (int)((row_tiles + sh.tiles - 1) / sh.tiles);
  const long long items = (long long)sh.blocks * batch * nkv * (FORM == PARTS ? sh.parts.splits : 1);
  Q_CHECK_ARG(items < (1ll << 30) && (long long)batch * T < (1ll << 31), "%s: too many rows", who);
  sh.items = (int)items;
  sh.wide = ((uintptr_t)d_out & 31) == 0;
  sh.scale_log2 = scale * 1.4426950408889634f;
  CUtensorMap qmap, kmap, vmap;
  {
    const cuuint64_t dim[3] = {128, (cuuint64_t)n_q_heads, (cuuint64_t)batch * T};
    const cuuint64_t stride[2] = {256, (cuuint64_t)n_q_heads * 256};
    const cuuint32_t box[3] = {64, (cuuint32_t)G, (cuuint32_t)sh.tokens};
    int rc = tc_encode(&qmap, d_q, 3, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_128B, who);
    if (rc) return rc;
  }
  for (int i = 0; i < 2; ++i) {
    // (64 dims, half, token row, page x head): the number of pages is the caller's, bounded by memory
    const cuuint64_t dim[4] = {64, 2, Q_PAGE_TOKENS, 1u << 24};
    const cuuint64_t stride[3] = {128, 256, Q_PAGE_TOKENS * 256};
    const cuuint32_t box[4] = {64, 1, Q_PAGE_TOKENS, 1};
    int rc = tc_encode(i ? &vmap : &kmap, i ? kv->d_vpool : kv->d_kpool, 4, dim, stride, box, CU_TENSOR_MAP_SWIZZLE_NONE,
                       who);
    if (rc) return rc;
  }
  static size_t done[2][64] = {{0}};
  auto kern = sh.tiles == 2 ? k_attn_prompt<2, FORM, false> : k_attn_prompt<1, FORM, FORM != CAUSAL>;
  Q_CHECK_CUDA(q_ensure_smem(kern, AP_SMEM, done[sh.tiles - 1]));
  const int grid = sh.items < sms ? sh.items : sms;
  Q_CHECK_CUDA(q_launch(kern, dim3(grid), dim3(AP_THREADS), AP_SMEM, (cudaStream_t)stream, qmap, kmap, vmap,
                        kv->d_block_table, d_pos, (bf16*)d_out, sh, status));
  return Q_OK;
}

}  // namespace

extern "C" int q_attention_prefill(const void* d_q, const q_kv_layout_t* kv, const int32_t* d_pos,
                                   void* d_out, int batch, int T, int n_q_heads, float scale,
                                   void* stream) {
  AttnShape sh = {};
  return prompt_launch<CAUSAL>("q_attention_prefill", sh, d_q, kv, d_pos, d_out, batch, T, n_q_heads, scale, stream);
}

extern "C" int q_attention_window_prefill(const void* d_q, const q_kv_layout_t* kv, const int32_t* d_pos,
                                          int pos_per_seq, void* d_out, int batch, int T, int n_q_heads, int window,
                                          int sinks, float scale, void* stream) {
  const char* who = "q_attention_window_prefill";
  Q_CHECK_ARG(window >= 1 && sinks >= 0, "%s: window %d / sinks %d", who, window, sinks);
  AttnShape sh = {};
  sh.pos_step = pos_per_seq ? 1 : 0;
  Q_CHECK_ARG(T <= (1 << 30), "%s: %d tokens", who, T);
  sh.far = 0x7fffffff - 512 - (T > 0 ? T : 0);             // (a block of tokens ends at most 255 behind T)
  sh.window = window < 0x7fffffff - 512 ? window : 0x7fffffff - 512;
  sh.sinks = sinks;
  return prompt_launch<WINDOW>(who, sh, d_q, kv, d_pos, d_out, batch, T, n_q_heads, scale, stream);
}

int q_attention_parts_tc(const void* d_q, const q_kv_layout_t* kv, const int32_t* d_len, float* parts_o,
                         float* parts_ml, int splits, int tokens, int n_q_heads, float scale, void* stream) {
  AttnShape sh = {};
  sh.parts.o = parts_o;
  sh.parts.ml = reinterpret_cast<float2*>(parts_ml);
  sh.parts.keys = d_len;
  sh.parts.splits = splits;
  sh.parts.nkv = kv->n_kv_heads;
  sh.parts.rows = tokens * (n_q_heads / kv->n_kv_heads);
  sh.parts.tile = AP_KEYS;
  return prompt_launch<PARTS>("q_attention_shared", sh, d_q, kv, d_len, nullptr, 1, tokens, n_q_heads, scale, stream);
}
