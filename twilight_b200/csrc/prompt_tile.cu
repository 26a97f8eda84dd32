// Attention tiles of up to 256 query rows on the fifth-generation tensor cores: the part of prompt_attn and
// shared_prefix_attn whose segments have more than a few rows.
//
// A block (one per SM, persistent) works on one item at a time: two subtiles of 128 packed rows (tokens x query heads
// of one KV head) over one run of its pages, 128 keys (eight pages) a step.  Per subtile and step
//   S = Q K^T          tcgen05.mma, both operands in shared memory (128-byte swizzle), S in TMEM, fp32
//   P = 2^(S c - m)    one softmax thread per row: S from TMEM, running maximum and sum in registers, P back to TMEM
//   O += P V           tcgen05.mma, P from TMEM, V in shared memory as it lies in the cache (keys x channels)
// The two subtiles share K and V and alternate on the tensor cores: while one subtile's weights are computed, the
// other's products run.  An item of one subtile takes both places: they take its key tiles in turn, and their results
// are joined at the end.  TMEM (512 columns): S of both (P takes the place of S once it is read), O of both.
// The reference m of a row is only moved when its maximum has grown by more than 2^8, so O is rescaled a few times per row.  The
// largest weight is between 1 and 2^8 in bf16, between 2^7 and 2^15 in fp16 (see kTopWeight): n weights are off by at most n 2^-32 of
// the largest one altogether there.
//
// Warps: 0-3 and 4-7 softmax, 8 K pages, 11 V pages, 9 tensor-core issue, 10 work items (taken from a counter, two ahead).
// K has three 32 KiB stages, V two.  A page is ONE copy: seen as [groups of 8 rows][halves of 64 channels][8 rows][64] it
// lands as four swizzle atoms, equal halves 2 KiB apart for both operands.  (As two boxes per page, issued by one warp, the
// copies took 2700 clocks a step of K and V, more than its products: each costs its warp about 85.)
//
// Bound: two products of 128 x 128 x 128 (512 clocks each at the tensor peak) and 128 x 128 exponentials (1024 clocks of the
// special-function units) per subtile and step; with few rows per KV head, reading K and V.  8192 queries x 8192 keys, 32/8
// heads: 820 us, 1340 TFLOP/s (0.82 of the measured bf16 peak; causal 1230), a step of both subtiles in 3340 clocks.
#include <cuda.h>

#include <type_traits>

#include "prompt.cuh"

namespace twl {

constexpr int kTileThreads = 384;  // three warpgroups, the unit of the register split
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;  // (200: the same, 216: 1 % slower, 224: 5 %)
static_assert(2 * kSoftmaxRegs + kOtherRegs <= 3 * 168, "registers of the launch: 168 a thread at 384 threads");
constexpr int kKStages = 3, kVStages = 2, kStages = kKStages + kVStages;
constexpr int kStageBytes = 128 * kD * 2;      // 128 keys (or 128 query rows)
constexpr int kHalfBytes = kStageBytes / 2;    // 64 channels of 128 query rows
constexpr int kPageBytes = kPage * kD * 2, kAtom = 1024;
constexpr int kInfoSlots = 8;                  // key tiles whose positions are kept
constexpr uint32_t kWaitTries = 2000, kWaitNs = 500000;  // a wait gives up after about a second

struct alignas(64) TileParams {
  CUtensorMap tq, tk, tv;
  AttnParams a;
};

// One work item as every role of the block sees it; n_tiles < 0 ends the block.
struct Item {
  const int32_t* indices;  // the segment's part of its page table
  const int32_t* list;     // block list from the item's first page on, or null
  int64_t part0;           // partial row of its first token and query head 0, or -1
  int32_t tok0, ntok, kvh; // first token
  int32_t page0;           // first page (without a list)
  int32_t npages, len;     // of the segment
  int32_t limit0;          // last position the first token sees (all tokens, when not causal)
  int32_t n_pages;
  int32_t n_tiles;         // key tiles of the item
  int32_t steps[2];        // and of its two subtiles
  int32_t tail_page;       // page of the last key tile in which the sequence ends inside the page, or -1
  int32_t pair;            // one subtile in both places: key tile 2j + a is step j of place a
};

struct TileShared {
  uint64_t item_full[2], item_empty[2];
  uint64_t q_full, q_free, k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages];
  uint64_t s_full[2], p_half[2], p_full[2], o_full[2], pair[2], drain;
  Item items[2];
  uint32_t tmem;
  int32_t hi[kInfoSlots];      // largest position of the tile's keys, INT_MAX when a page is missing
  int32_t pos[kInfoSlots][8];  // position of every page's first key
  float2 ml[2][128];           // results of the two places of a pair
};
constexpr int kTileSmem = 2 * kStageBytes + kStages * kStageBytes + (int)sizeof(TileShared);
static_assert(kTileSmem <= 232448, "shared memory of a block");

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void mbar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(b)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
// Bounded wait for the completion of the phase with this parity; false when the limit ran out.  A thread that was refused
// goes on (with data that is not there yet) to the next all_ok of its warp, so that the warps stay together.
__device__ __forceinline__ bool mbar_wait(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{ .reg .pred p; .reg .u32 n; mov.u32 n, %3;\n"
      "W: mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n"
      "@p bra D;\n"
      "sub.u32 n, n, 1; setp.ne.u32 p, n, 0;\n"
      "@p bra W;\n"
      "D: selp.u32 %0, 1, 0, p; }"
      : "=r"(ok) : "r"(smem_u32(b)), "r"(parity), "n"(kWaitTries), "n"(kWaitNs) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(0xffffffffu, ok); }

__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* m, int group, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %2, %2, %3}], [%4];" ::"r"(
          dst),
      "l"(m), "r"(0), "r"(group), "r"(smem_u32(bar))
      : "memory");
}
__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap* m, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
      "l"(m), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// Shared-memory operand descriptor, 128-byte swizzle.  Rows of 128 bytes, eight rows to a swizzle atom (1024 bytes):
// `stride` is from one group of eight rows to the next, `lead` (operands whose rows are the K side) from one 64-element
// column block to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr & 0x3ffff) >> 4) | ((uint64_t)(lead >> 4) << 16) | ((uint64_t)(stride >> 4) << 32) |
         (1ull << 46) | (2ull << 61);
}
// Instruction descriptor: fp32 accumulators, 128 x 128, A and B of the model type, B's rows the N side or the K side.
template <typename T>
__device__ __forceinline__ constexpr uint32_t mma_desc(bool b_rows_are_k) {
  const uint32_t fmt = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_rows_are_k ? 1u : 0u) << 16) | (16u << 17) | (8u << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a),
      "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }" ::"r"(d), "r"(a),
      "l"(b), "r"(idesc), "r"((uint32_t)add)
      : "memory");
}
// One lane of the warp (always the same), in a form that the compiler knows to be a single thread: the operands of what
// it issues then stay in uniform registers.
__device__ __forceinline__ bool one_lane() {
  uint32_t p;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of the thread's TMEM lane.  The wait names the registers, so that nothing uses them before it.
__device__ __forceinline__ void tmem_ld32(float* r, uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]),
        "=f"(r[8]), "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]),
        "=f"(r[16]), "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]),
        "=f"(r[24]), "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_wait_ld32(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
      : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
        "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]),
        "+f"(r[16]), "+f"(r[17]), "+f"(r[18]), "+f"(r[19]), "+f"(r[20]), "+f"(r[21]), "+f"(r[22]), "+f"(r[23]),
        "+f"(r[24]), "+f"(r[25]), "+f"(r[26]), "+f"(r[27]), "+f"(r[28]), "+f"(r[29]), "+f"(r[30]), "+f"(r[31])
               :: "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
      "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
      "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]), "r"(addr)
      : "memory");
}
__device__ __forceinline__ float tile_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t tile_pack2(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t tile_pack2(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// (a NaN goes on: the row's reference, and with it the row, becomes NaN)
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max64(const float* x) {
  float m[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
  for (int c = 4; c < 60; c += 8)
#pragma unroll
    for (int e = 0; e < 4; ++e) m[e] = max3(m[e], x[c + e], x[c + 4 + e]);
  m[0] = max3(m[0], x[60], x[61]);
  m[1] = max3(m[1], x[62], x[63]);
  return max3(max3(m[0], m[1], m[2]), m[3], m[3]);
}
// 64 weights 2^(x scale - ref) of a row: their sum in 32 bits, and themselves rounded to the model type (half a step each, see above),
// in which they go to the tensor cores.  All on the special-function unit: with an eighth or a quarter of them by a polynomial
// on the multiply-add pipes, 8K x 8K with 32/8 heads took 848 instead of 823 us.
template <typename T>
__device__ __forceinline__ void weights(const float* x, uint64_t scale, uint64_t ref, uint64_t (&sum)[2], uint32_t (&w)[32]) {
#pragma unroll
  for (int e = 0; e < 32; ++e) {
    float a, b;
    f2_split(fma2(f2(x[2 * e], x[2 * e + 1]), scale, ref), a, b);
    a = tile_ex2(a);
    b = tile_ex2(b);
    sum[e & 1] = add2(sum[e & 1], f2(a, b));
    w[e] = tile_pack2(a, b, T());
  }
}

__device__ __forceinline__ Item load_item(const AttnParams& p, int i) {
  Item it;
  const int4 w = p.tile_list[i / p.Hkv];
  it.kvh = i % p.Hkv;
  const Segment s = p.segs[w.x];
  it.indices = (s.second ? p.indices2 : p.indices1) + s.kvbase;
  it.tok0 = s.tok0 + w.y;
  it.ntok = w.z;
  it.page0 = w.w * s.chunk_pages;  // (a chunk that is everything: number 0)
  it.npages = s.npages;
  it.len = s.len;
  it.limit0 = p.causal ? s.len - s.ntok + w.y : s.len - 1;
  it.part0 = s.pbase < 0 ? -1 : s.pbase + ((int64_t)w.w * s.ntok + w.y) * p.Hq;
  it.list = nullptr;
  int avail = 0;
  if (p.block_pages) {
    const int64_t slot = (int64_t)(s.tok0 / p.query_block + w.x + w.y / p.query_block) * p.Hkv + it.kvh;
    it.list = p.block_pages + slot * p.max_k + it.page0;
    avail = min(max(p.block_npages[slot], 0), p.max_k);
  }
  it.n_pages = 0;
#pragma unroll
  for (int a = 0; a < 2; ++a) {
    const int n = min(it.ntok - a * p.tok_tile, p.tok_tile);
    int pages = 0;
    if (n > 0) {
      if (!it.list) avail = pages_seen(s, w.y + a * p.tok_tile + n - 1, p.causal);
      pages = max(0, min(avail - it.page0, s.chunk_pages));
    }
    it.steps[a] = (pages + 7) >> 3;
    it.n_pages = max(it.n_pages, pages);
  }
  it.n_tiles = max(it.steps[0], it.steps[1]);
  it.tail_page = -1;
  if (it.n_pages > 0 && (s.len & (kPage - 1)) != 0 &&
      (it.list ? it.list[it.n_pages - 1] : it.page0 + it.n_pages - 1) == s.npages - 1)
    it.tail_page = (it.n_pages - 1) & 7;
  it.pair = it.ntok <= p.tok_tile && it.n_tiles > 1;
  if (it.pair) {
    it.steps[0] = (it.n_tiles + 1) >> 1;
    it.steps[1] = it.n_tiles >> 1;
  }
  return it;
}

template <typename T>
__global__ void __launch_bounds__(kTileThreads, 1) prompt_tile_kernel(const __grid_constant__ TileParams tp) {
  extern __shared__ __align__(1024) uint8_t smem[];  // swizzle atoms of 1024 bytes
  uint8_t* q_s = smem;
  uint8_t* kv_s = smem + 2 * kStageBytes;
  TileShared& sh = *reinterpret_cast<TileShared*>(smem + (2 + kStages) * kStageBytes);
  const AttnParams& p = tp.a;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    mbar_init(&sh.q_full, 1);
    mbar_init(&sh.q_free, 1);
    mbar_init(&sh.drain, 1);
    for (int i = 0; i < kKStages; ++i) {
      mbar_init(&sh.k_full[i], 1);
      mbar_init(&sh.k_empty[i], 1);
    }
    for (int i = 0; i < kVStages; ++i) {
      mbar_init(&sh.v_full[i], 1);
      mbar_init(&sh.v_empty[i], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&sh.item_full[a], 1);
      mbar_init(&sh.item_empty[a], 11);  // two of loads, tensor cores, eight softmax warps
      mbar_init(&sh.s_full[a], 1);
      mbar_init(&sh.p_half[a], 128);
      mbar_init(&sh.p_full[a], 128);
      mbar_init(&sh.o_full[a], 1);
      mbar_init(&sh.pair[a], 256);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // Everything from here on reads what earlier kernels wrote (the plan, page tables, lists; Q, K and V by TMA), and only this wait
  // makes that visible.  The kernel before is the row kernel, whose release lets the lines above run beside its last blocks.
  pdl_wait();
  bool ok = true;
  uint32_t n_item = 0;  // items so far: slot n_item & 1 of the two
  // The next item, copied out of its slot; false at the end (or when a wait ran out: ok is false then).
  const auto next_item = [&](Item& it) {
    const int s = n_item & 1;
    ok = all_ok(mbar_wait(&sh.item_full[s], (n_item >> 1) & 1));
    if (!ok) return false;
    it = sh.items[s];
    __syncwarp();
    if (lane == 0) mbar_arrive(&sh.item_empty[s]);
    ++n_item;
    return it.n_tiles >= 0;
  };
  if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));

  if (warp == 10) {
    // ---- work items ----
    const int n_items = p.hdr->tile_items * p.Hkv;
    for (int i = blockIdx.x;; ++n_item) {
      Item it;
      if (i < n_items)
        it = load_item(p, i);
      else
        it.n_tiles = -1;
      const int s = n_item & 1;
      ok = all_ok(mbar_wait(&sh.item_empty[s], ((n_item >> 1) & 1) ^ 1));
      if (!ok) break;
      if (lane == 0) {
        sh.items[s] = it;
        mbar_arrive(&sh.item_full[s]);
      }
      __syncwarp();
      if (i >= n_items) break;
      if (lane == 0) i = gridDim.x + atomicAdd(&p.hdr->next_tile, 1);
      i = __shfl_sync(0xffffffffu, i, 0);
    }
  } else if (warp == 8 || warp == 11) {
    // ---- loads: warp 8 Q and K, warp 11 V; lane l takes page l of a key tile ----
    const bool is_k = warp == 8;
    const int n_stages = is_k ? kKStages : kVStages;
    uint64_t* const full = is_k ? sh.k_full : sh.v_full;
    uint64_t* const empty = is_k ? sh.k_empty : sh.v_empty;
    uint8_t* const base = kv_s + (is_k ? 0 : kKStages * kStageBytes);
    const CUtensorMap* const map = is_k ? &tp.tk : &tp.tv;
    uint32_t stage = 0, round = 0, q_round = 0;
    uint32_t tiles = 0;  // key tiles so far, over all items
    const int gone = p.num_pages_total * p.Hkv * 2;  // a group of rows behind the pool: reads as zeros
    Item it;
    while (next_item(it)) {
      if (it.n_tiles == 0) continue;
      if (is_k) {
        const int subs = it.ntok > p.tok_tile ? 2 : 1;
        ok = all_ok(mbar_wait(&sh.q_free, (q_round & 1) ^ 1));
        if (!ok) break;
        ++q_round;
        if (lane == 0) {
          mbar_expect(&sh.q_full, (uint32_t)(subs * 2 * 64 * 2 * p.G * p.tok_tile));
          for (int a = 0; a < subs; ++a)
            for (int h = 0; h < 2; ++h)
              tma_3d(smem_u32(q_s) + a * kStageBytes + h * kHalfBytes, &tp.tq, h * 64, it.kvh * p.G,
                     it.tok0 + a * p.tok_tile, &sh.q_full);
        }
        __syncwarp();
      }
      const auto look_up = [&](int j, int& lp, int& phys) {
        const int at = 8 * j + lane;
        lp = -1;
        phys = -1;
        if (lane < 8 && at < it.n_pages) {
          lp = it.list ? it.list[at] : it.page0 + at;
          if (lp >= 0 && lp < it.npages) phys = it.indices[lp];
          if (phys < 0 || phys >= p.num_pages_total) {
            phys = -1;
            if (is_k) raise_flag(p.status, TWL_FLAG_BAD_INDEX);
          }
        }
      };
      int lp, phys;
      look_up(0, lp, phys);
      for (int t = 0; t < it.n_tiles; ++t) {
        const int group = phys < 0 ? gone : (phys * p.Hkv + it.kvh) * 2;
        const int pos = phys < 0 ? 0x7fffffff : lp * kPage;
        const int hi = __reduce_max_sync(0xffffffffu, lane >= 8 ? -1 : phys < 0 ? 0x7fffffff : pos + kPage - 1);
        look_up(t + 1, lp, phys);
        ok = all_ok(mbar_wait(&empty[stage], (round & 1) ^ 1));
        if (!ok) break;
        if (is_k) {
          // Room for K means that the scores of three tiles ago are done, and they were begun after the weights of at the
          // latest five tiles ago: of the eight slots of the info at most five are still read.
          const int slot = tiles++ & (kInfoSlots - 1);
          if (lane < 8) sh.pos[slot][lane] = pos;
          if (lane == 0) sh.hi[slot] = hi;
        }
        if (lane == 0) mbar_expect(&full[stage], kStageBytes);
        __syncwarp();
        if (lane < 8) tma_page(smem_u32(base + stage * kStageBytes) + lane * kPageBytes, map, group, &full[stage]);
        __syncwarp();
        if (++stage == (uint32_t)n_stages) {
          stage = 0;
          ++round;
        }
      }
      if (!ok) break;
    }
    if (!ok) {  // an early end: the copies in flight still write to shared memory
      for (uint32_t s = 0; s < (uint32_t)n_stages; ++s)
        if (round > 0 || s < stage) mbar_wait(&full[s], (s < stage ? round : round - 1) & 1);
      if (q_round) mbar_wait(&sh.q_full, (q_round - 1) & 1);
    }
  } else if (warp == 9) {
    // ---- tensor cores ----
    uint32_t k_stage = 0, k_round = 0, v_stage = 0, v_round = 0, q_round = 0, p_rounds = 0;  // p_rounds: bit a is place a's parity
    const uint32_t kS = mma_desc<T>(false), kO = mma_desc<T>(true);
    // operand descriptors of the first query row, of the first stages (sixteen-byte units)
    const uint64_t q_desc = smem_desc(smem_u32(q_s), 16, kAtom), k_desc = smem_desc(smem_u32(kv_s), 16, 2 * kAtom);
    const uint64_t v_desc = smem_desc(smem_u32(kv_s + kKStages * kStageBytes), kAtom, 2 * kAtom);
    const auto next_k = [&]() {
      if (++k_stage == kKStages) {
        k_stage = 0;
        ++k_round;
      }
    };
    const auto next_v = [&]() {
      if (++v_stage == kVStages) {
        v_stage = 0;
        ++v_round;
      }
    };
    const auto scores = [&](int a, uint32_t q_at) {  // S = Q K^T with the K of the current stage
      const uint64_t qd = q_desc + (q_at >> 4), kd = k_desc + k_stage * (kStageBytes >> 4);
      if (one_lane()) {
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) {
          const uint32_t q_off = (ks >> 2) * kHalfBytes + (ks & 3) * 32, k_off = (ks >> 2) * kAtom + (ks & 3) * 32;
          mma_ss(tmem + a * 128, qd + (q_off >> 4), kd + (k_off >> 4), kS, ks > 0);
        }
        mma_commit(&sh.s_full[a]);
      }
      __syncwarp();
    };
    const auto commit = [&](uint64_t* bar) {
      if (one_lane()) mma_commit(bar);
      __syncwarp();
    };
    // O += P V in two halves of 64 keys: the first starts while the softmax works on the second
    const auto values = [&](int a, bool add) {
      const uint64_t vd = v_desc + v_stage * (kStageBytes >> 4);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        ok &= mbar_wait(h ? &sh.p_full[a] : &sh.p_half[a], (p_rounds >> a) & 1);
        tc_fence_after();
        if (one_lane()) {
#pragma unroll
          for (int ks = 4 * h; ks < 4 * h + 4; ++ks)
            mma_ts(tmem + 256 + a * 128, tmem + a * 128 + ks * 8, vd + ks * (kPageBytes >> 4), kO, add || ks > 0);
        }
        __syncwarp();
      }
      p_rounds ^= 1u << a;
    };
    const auto wait_k = [&]() { ok &= mbar_wait(&sh.k_full[k_stage], k_round & 1); };
    const auto wait_v = [&]() { ok &= mbar_wait(&sh.v_full[v_stage], v_round & 1); };
    const auto clean_tail = [&](const Item& it) {
      // rows behind the sequence's end may hold anything, and 0 x NaN is not 0
      uint8_t* page = kv_s + (kKStages + v_stage) * kStageBytes + it.tail_page * kPageBytes;
      for (int c = (it.len & (kPage - 1)) * 16 + lane; c < kPage * 16; c += 32) {  // row, half, piece
        const int r = c >> 4;
        *reinterpret_cast<uint4*>(page + (r >> 3) * 2 * kAtom + ((c >> 3) & 1) * kAtom + (r & 7) * 128 + (c & 7) * 16) =
            make_uint4(0, 0, 0, 0);
      }
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
    };
    Item it;
    while (next_item(it)) {
      if (it.n_tiles == 0) continue;
      ok &= mbar_wait(&sh.q_full, q_round & 1);
      ++q_round;
      wait_k();
      if (it.pair) {
        scores(0, 0);
        commit(&sh.k_empty[k_stage]);
        next_k();
        wait_k();
        scores(1, 0);
        commit(&sh.k_empty[k_stage]);
        if (it.n_tiles == 2) commit(&sh.q_free);
        next_k();
        for (int t = 0; t < it.n_tiles; ++t) {
          const int a = t & 1;
          const bool more = t + 2 < it.n_tiles;
          wait_v();
          if (more) wait_k();
          if (t + 1 == it.n_tiles && it.tail_page >= 0) clean_tail(it);
          values(a, t > 1);
          commit(&sh.v_empty[v_stage]);
          next_v();
          if (more) {
            scores(a, 0);
            commit(&sh.k_empty[k_stage]);
            next_k();
            if (t + 3 == it.n_tiles) commit(&sh.q_free);  // the last product with Q has been issued
          } else {
            commit(&sh.o_full[a]);
          }
          ok = all_ok(ok);
          if (!ok) break;
        }
      } else {
        if (it.steps[0] > 0) scores(0, 0);
        if (it.steps[1] > 0) scores(1, kStageBytes);
        commit(&sh.k_empty[k_stage]);
        if (it.n_tiles == 1) commit(&sh.q_free);
        next_k();
        for (int j = 0; j < it.n_tiles; ++j) {
          const bool more = j + 1 < it.n_tiles;
          wait_v();
          if (more) wait_k();
          if (!more && it.tail_page >= 0) clean_tail(it);
          const int last = j < it.steps[1] ? 1 : 0;  // the subtile that uses this V last
#pragma unroll
          for (int a = 0; a < 2; ++a) {
            if (j >= it.steps[a]) continue;
            values(a, j > 0);
            if (a == last) commit(&sh.v_empty[v_stage]);
            if (j + 1 < it.steps[a])
              scores(a, a * kStageBytes);
            else
              commit(&sh.o_full[a]);
          }
          next_v();
          if (more) {
            commit(&sh.k_empty[k_stage]);
            if (j + 2 == it.n_tiles) commit(&sh.q_free);  // the last product with Q has been issued
            next_k();
          }
          ok = all_ok(ok);
          if (!ok) break;
        }
      }
      ok = all_ok(ok);
      if (!ok) break;
    }
    if (!ok) {  // an early end: products in flight still read shared memory and write TMEM
      commit(&sh.drain);
      mbar_wait(&sh.drain, 0);
    }
  } else if (warp < 8) {
    // ---- softmax: thread = row ----
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int a = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // TMEM lane of the warp's first row
    const uint32_t s_t = tmem + lanes + a * 128, o_t = tmem + lanes + 256 + a * 128;
    uint32_t s_round = 0, o_own = 0, o_other = 0, tiles = 0, pairs = 0;
    const int tok_r = r / p.G, head_r = r - tok_r * p.G;
    const float scale = p.scale_log2;
    for (;; ++n_item) {
      // (read in place and given back at the end: a copy would hold registers that a row of scores needs)
      const Item& it = sh.items[n_item & 1];
      ok = all_ok(mbar_wait(&sh.item_full[n_item & 1], (n_item >> 1) & 1));
      if (!ok || it.n_tiles < 0) break;
      const int pair = it.pair;
      const int tok = (pair ? 0 : a * p.tok_tile) + tok_r;  // of the item
      const bool real = tok_r < p.tok_tile && tok < it.ntok;
      const int limit = !real ? -1 : max(-1, p.causal ? it.limit0 + tok : it.limit0);
      float m = -INFINITY, l = 0.f;
      const int steps = a ? it.steps[1] : it.steps[0], steps_other = a ? it.steps[0] : it.steps[1];
      for (int j = 0; j < steps; ++j) {
        ok = mbar_wait(&sh.s_full[a], s_round & 1);
        ++s_round;
        tc_fence_after();
        const int slot = (tiles + (pair ? 2 * j + a : j)) & (kInfoSlots - 1);
        float x[128];
        tmem_ld32(x, s_t);
        tmem_ld32(x + 32, s_t + 32);
        if (!all_ok(ok)) break;
        const bool masked = __any_sync(0xffffffffu, real && sh.hi[slot] > limit);
        tmem_wait_ld32(x);
        tmem_wait_ld32(x + 32);
        tmem_ld32(x + 64, s_t + 64);
        tmem_ld32(x + 96, s_t + 96);
        tmem_wait_ld32(x + 64);
        tmem_wait_ld32(x + 96);
        if (masked) {
#pragma unroll
          for (int pg = 0; pg < 8; ++pg) {
            const int n = limit - sh.pos[slot][pg];  // keys 0..n of the page are seen (at least -2^31: limit is -1 or more)
#pragma unroll
            for (int c = 0; c < kPage; ++c)
              if (c > n) x[16 * pg + c] = -INFINITY;
          }
          __syncwarp();
        }
        const float top = max3(max64(x), max64(x + 64), -INFINITY) * scale;
        // Move the reference, kTop below the maximum, only when that has grown by more than 2^8 (or nothing was seen so far).  (Computing
        // the first weights with the standing reference while the maximum is found was 2 % slower.)
        constexpr float kTop = kTopWeight<T> == 0.f ? 0.f : kTopWeight<T> - 8.f;
        float f = 1.f;
        const bool move = !(top <= m + (kTop + 8.f));  // from -inf: any finite maximum; a NaN moves it too
        if (move) {
          f = tile_ex2(m - (top - kTop));
          m = top - kTop;
          l *= f;
        }
        if (__any_sync(0xffffffffu, move) && j > 0) {
          // S of this step is complete, so the product of the step before is too: O may be changed.  (Not unrolled: this is
          // rare, and its registers would push those of the loop into local memory.)
#pragma unroll 1
          for (int c = 0; c < 4; ++c) {
            float o[32];
            uint32_t w[32];
            tmem_ld32(o, o_t + 32 * c);
            tmem_wait_ld32(o);
#pragma unroll
            for (int e = 0; e < 32; ++e) w[e] = __float_as_uint(o[e] * f);
            tmem_st32(o_t + 32 * c, w);
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t scale2 = f2(scale, scale), ref2 = f2(-ref, -ref);
        uint64_t sum[2] = {0, 0};
        uint32_t w[32];
        weights<T>(x, scale2, ref2, sum, w);
        tmem_st32(s_t, w);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sh.p_half[a]);
        weights<T>(x + 64, scale2, ref2, sum, w);
        tmem_st32(s_t + 32, w);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&sh.p_full[a]);
        float s0, s1;
        f2_split(add2(sum[0], sum[1]), s0, s1);
        l += s0 + s1;
      }
      ok = all_ok(ok);
      if (!ok) break;
      tiles += it.n_tiles;
      // ---- the item's rows: columns c0 .. of O, of both places of a pair ----
      const bool any = steps > 0;
      float f_own = 1.f, f_other = 0.f;
      if (pair) {
        sh.ml[a][r] = make_float2(m, l);
        mbar_arrive(&sh.pair[0]);
        ok = all_ok(mbar_wait(&sh.pair[0], pairs & 1));
        if (!ok) break;
        const float2 v = sh.ml[a ^ 1][r];
        const float mm = fmaxf(m, v.x), ref = mm == -INFINITY ? 0.f : mm;
        f_own = tile_ex2(m - ref);
        f_other = tile_ex2(v.x - ref);
        l = a ? v.y * f_other + l * f_own : l * f_own + v.y * f_other;  // the same sum in both places
        m = mm;
        ok = all_ok(mbar_wait(&sh.o_full[a ^ 1], o_other & 1));
        if (!ok) break;
      }
      if (any) {
        ok = all_ok(mbar_wait(&sh.o_full[a], o_own & 1));
        if (!ok) break;
      }
      o_own += any;
      o_other += steps_other > 0;
      tc_fence_after();
      const int64_t row = (int64_t)it.tok0 + tok, head = it.kvh * p.G + head_r;
      const int64_t part = it.part0 < 0 ? -1 : it.part0 + (int64_t)tok * p.Hq + head;
      const bool write = real && (part < 0 || part < p.part_cap);
      const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll 1
      for (int c = 0; c < 4; ++c) {
        if (pair && (c >> 1) != a) continue;  // each place writes half of the channels
        float o[32];
        __syncwarp();
        if (any) {
          tmem_ld32(o, o_t + 32 * c);
          tmem_wait_ld32(o);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = 0.f;
        }
        if (pair) {
          float z[32];
          tmem_ld32(z, tmem + lanes + 256 + (a ^ 1) * 128 + 32 * c);
          tmem_wait_ld32(z);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = o[e] * f_own + z[e] * f_other;
        }
        if (!write) continue;
        if (part >= 0) {
          if (l != 0.f) {
            float4* to = reinterpret_cast<float4*>(p.part_acc + part * kD + 32 * c);
#pragma unroll
            for (int e = 0; e < 8; ++e) to[e] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        } else {
          uint4* to = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + row * p.o_ts + head * kD + 32 * c);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            uint32_t w[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              w[k] = l != 0.f ? tile_pack2(o[8 * e + 2 * k] * inv, o[8 * e + 2 * k + 1] * inv, T()) : 0u;
            to[e] = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      }
      if (write && !(pair && a)) {
        if (part >= 0)
          p.part_ml[part] = make_float2(m, l);
        else if (p.lse)
          p.lse[row * p.Hq + head] = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
      }
      // a pair's places have read each other's O (and ml): only then may the next item's products replace it
      tc_fence_before();
      if (pair) {
        mbar_arrive(&sh.pair[1]);
        ok = all_ok(mbar_wait(&sh.pair[1], pairs++ & 1));
        if (!ok) break;
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.item_empty[n_item & 1]);
    }
  }
  if (!ok && lane == 0) raise_flag(p.status, TWL_FLAG_WAIT_LIMIT);
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

// ---- host ------------------------------------------------------------------------------------------
using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                              const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                              CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeFn tensor_map_encoder() {
  static const EncodeFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &r) != cudaSuccess ||
        r != cudaDriverEntryPointSuccess)
      f = nullptr;
    return reinterpret_cast<EncodeFn>(f);
  }();
  return fn;
}

int tile_attention_launch(const AttnParams& p, int dtype, cudaStream_t st) {
  const EncodeFn encode = tensor_map_encoder();
  if (!encode) {
    set_last_cuda_error(cudaErrorNotSupported);
    return TWL_ERR_LAUNCH;
  }
  TileParams tp;
  tp.a = p;
  const CUtensorMapDataType type = dtype == TWL_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  const cuuint32_t ones[4] = {1, 1, 1, 1};
  const cuuint64_t kv_dims[4] = {64, 8, 2, (cuuint64_t)p.num_pages_total * p.Hkv * 2};
  const cuuint64_t kv_strides[3] = {kD * 2, 128, 8 * kD * 2};
  const cuuint32_t kv_box[4] = {64, 8, 2, 2};
  const cuuint64_t q_dims[3] = {(cuuint64_t)kD, (cuuint64_t)p.Hq, (cuuint64_t)p.num_tokens};
  const cuuint64_t q_strides[2] = {kD * 2, (cuuint64_t)p.q_ts * 2};
  const cuuint32_t q_box[3] = {64, (cuuint32_t)p.G, (cuuint32_t)p.tok_tile};
  bool ok = true;
  for (int i = 0; i < 2; ++i)
    ok = ok && encode(i ? &tp.tv : &tp.tk, type, 4, const_cast<void*>(i ? p.v_pages : p.k_pages), kv_dims, kv_strides, kv_box,
                      ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  ok = ok && encode(&tp.tq, type, 3, const_cast<void*>(p.q), q_dims, q_strides, q_box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  if (!ok) {
    set_last_cuda_error(cudaErrorInvalidValue);
    return TWL_ERR_LAUNCH;
  }
  static int8_t done[2][kSmemDevices];
  auto* kernel = dtype == TWL_F16 ? prompt_tile_kernel<__half> : prompt_tile_kernel<__nv_bfloat16>;
  TWL_CUDA_TRY(allow_smem(kernel, kTileSmem, done[dtype == TWL_F16]));
  TWL_CUDA_TRY(launch_chain(kernel, dim3((unsigned)num_sms()), dim3(kTileThreads), kTileSmem, st, tp));
  return TWL_OK;
}

}  // namespace twl
