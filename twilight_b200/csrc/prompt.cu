// Attention over the paged cache for more than one token at a time: a prompt's (prompt_attn) and a decode batch's
// over a shared prefix (shared_prefix_attn): plan, row kernel, merge and the C entry points.
//
//   out[row] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * (q.k_j - max)) over the keys the row may see,
// one pass over the keys with a running maximum and sum (32-bit), joined over key chunks as
//   m = max_c m_c,  l = sum_c l_c 2^(m_c - m),  out = sum_c acc_c 2^(m_c - m) / l.
#include "prompt.cuh"

namespace twl {

// ---- plan -------------------------------------------------------------------------------------------
// One block: lengths and work of every segment, the chunk sizes, and the two lists of work items.  A separate
// launch, so that the lengths stay on the device and the other kernels find their work with one load.
constexpr int kPlanThreads = 1024;
constexpr int kRowChunkMin = 16;   // pages: four a warp; shorter chunks cost more in the merge than they balance
constexpr int kTileChunkMin = 32;  // pages: four key tiles, for the same reason

__device__ __forceinline__ Segment load_segment(const AttnParams& p, int i) {
  Segment s;
  const bool second = i >= p.n_first;
  const int j = second ? i - p.n_first : i;
  const int32_t* qo = second ? p.qo2 : p.qo1;
  const int32_t* indptr = second ? p.indptr2 : p.indptr1;
  s.tok0 = qo ? qo[j] : j;
  s.ntok = qo ? qo[j + 1] - s.tok0 : 1;
  s.kvbase = indptr[j];
  s.npages = indptr[j + 1] - s.kvbase;
  const int last = (second ? p.last2 : p.last1)[j];
  s.second = second;
  s.chunks = 1;
  s.chunk_pages = 0;
  s.pbase = -1;
  const bool bad = s.tok0 < 0 || s.ntok < 0 || s.tok0 + s.ntok > p.num_tokens || s.npages < 0 ||
                   (s.npages > 0 && (last < 1 || last > kPage));
  if (bad) {
    raise_flag(p.status, TWL_FLAG_BAD_INDEX);
    s.ntok = 0;
  }
  if (s.npages <= 0 || bad) s.npages = 0;
  s.len = s.npages ? (s.npages - 1) * kPage + last : 0;
  return s;
}

// row tiles of a segment (per KV head); a tile stays within one query block when there are block lists
__device__ __forceinline__ int row_tiles(const AttnParams& p, int ntok) {
  if (p.block_pages == nullptr) return (ntok * p.G + p.row_tile - 1) / p.row_tile;
  const int whole = ntok / p.query_block, rest = ntok - whole * p.query_block;
  return whole * ((p.query_block * p.G + p.row_tile - 1) / p.row_tile) + (rest * p.G + p.row_tile - 1) / p.row_tile;
}
__device__ __forceinline__ int tok_tiles(const AttnParams& p, int ntok) {
  const int t = 2 * p.tok_tile;
  if (p.block_pages == nullptr) return (ntok + t - 1) / t;
  const int whole = ntok / p.query_block, rest = ntok - whole * p.query_block;
  return whole * ((p.query_block + t - 1) / t) + (rest + t - 1) / t;
}

// Sums of N values over the block; every thread gets them.  One barrier before, one after the read.
template <int N>
__device__ __forceinline__ void block_sums(long long (&v)[N], long long (*s)[4]) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  if (lane == 0)
#pragma unroll
    for (int k = 0; k < N; ++k) s[threadIdx.x >> 5][k] = v[k];
  __syncthreads();
#pragma unroll
  for (int k = 0; k < N; ++k) v[k] = lane < warps ? s[lane][k] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], o);
  __syncthreads();
}

// pages of a chunk: enough chunks to give every tile slot about one, but not more than that many items
__device__ __forceinline__ int chunk_size(long long tiles, long long work, int target, int least, int step) {
  if (tiles >= target) return 0x3fffffff;  // every tile has a slot's worth of company
  // a tile of w pages becomes ceil(w/c) items, on average w/c + 1/2
  const long long room = max(1LL, target - tiles / 2);
  const long long c = max((long long)least, (work + room - 1) / room);
  return (int)min((long long)0x3fffffff, (c + step - 1) / step * step);
}

__global__ void __launch_bounds__(kPlanThreads) prompt_plan_kernel(const AttnParams p) {
  __shared__ long long sums[kPlanThreads / 32][4];
  __shared__ int scan[kPlanThreads / 32][3];
  pdl_wait();
  pdl_release();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_thr = blockDim.x, n_warps = n_thr >> 5;
  const int n_seg = p.n_first + p.n_second;
  const auto pages_of = [&](const Segment& s) { return p.block_pages ? min(s.npages, p.max_k) : s.npages; };
  // tiles and tiles x pages of the row kernel and of the tile kernel
  long long v[4] = {0, 0, 0, 0};
  Segment mine;  // this thread's segment of the first round
  mine.ntok = 0;
  for (int i = tid; i < n_seg; i += n_thr) {
    const Segment s = load_segment(p, i);
    if (i == tid) mine = s;
    const bool few = s.ntok * p.G <= p.few_rows;
    const int n = few ? row_tiles(p, s.ntok) : tok_tiles(p, s.ntok);
    v[few ? 0 : 2] += n;
    v[few ? 1 : 3] += (long long)n * pages_of(s);
  }
  block_sums<4>(v, sums);
  const int rc = chunk_size(v[0] * p.Hkv, v[1] * p.Hkv, p.row_target, kRowChunkMin, 1);
  int tc = chunk_size(v[2] * p.Hkv, v[3] * p.Hkv, p.tile_target, kTileChunkMin, 8);  // whole key tiles
  // one wave of tiles should stay one wave: count, and make the chunks longer by what is too much
  if (tc < 0x3fffffff) {
    for (int round = 0; round < 3; ++round) {
      long long items[1] = {0};
      for (int i = tid; i < n_seg; i += n_thr) {
        const Segment s = i == tid ? mine : load_segment(p, i);
        if (s.ntok * p.G > p.few_rows) items[0] += (long long)tok_tiles(p, s.ntok) * max(1, (pages_of(s) + tc - 1) / tc);
      }
      block_sums<1>(items, sums);
      const long long n = items[0] * p.Hkv;
      if (n <= p.tile_target) break;
      tc = (int)(((long long)tc * n / p.tile_target + 8) & ~7LL);
    }
  }

  int row_base = 0, tile_base = 0, part_base = 0, split = 0;
  for (int i0 = 0; i0 < n_seg; i0 += n_thr) {
    const int i = i0 + tid;
    Segment s;
    s.ntok = 0;
    s.chunks = 1;
    int cnt[3] = {0, 0, 0};  // row items, tile items, partial rows
    if (i < n_seg) {
      s = i0 == 0 ? mine : load_segment(p, i);
      const bool few = s.ntok * p.G <= p.few_rows;
      s.chunk_pages = few ? rc : tc;
      s.chunks = max(1, (pages_of(s) + s.chunk_pages - 1) / s.chunk_pages);
      cnt[few ? 0 : 1] = (few ? row_tiles(p, s.ntok) : tok_tiles(p, s.ntok)) * s.chunks;
      if (s.chunks > 1 || p.always_partial) cnt[2] = s.chunks * s.ntok * p.Hq;
      split |= s.chunks > 1;
    }
    // exclusive sums over the segments
    int inc[3] = {cnt[0], cnt[1], cnt[2]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const int x = __shfl_up_sync(0xffffffffu, inc[k], o);
        if (lane >= o) inc[k] += x;
      }
    if (lane == 31)
#pragma unroll
      for (int k = 0; k < 3; ++k) scan[warp][k] = inc[k];
    __syncthreads();
    int at[3], total[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      const int w = lane < n_warps ? scan[lane][k] : 0;
      const int before = __reduce_add_sync(0xffffffffu, lane < warp ? w : 0);
      total[k] = __reduce_add_sync(0xffffffffu, w);
      at[k] = before + inc[k] - cnt[k];
    }
    __syncthreads();
    if (i < n_seg) {
      s.pbase = cnt[2] > 0 ? (int64_t)part_base + at[2] : -1;
      p.segs[i] = s;
    }
    // a few items: their thread writes them; many: the warp does, segment by segment
    constexpr int kSelf = 4;
    const auto row_item = [&](int seg, int ntok, int chunks, int k, int to) {
      const int tile = k / chunks;
      int r0 = tile * p.row_tile, end = ntok * p.G;
      if (p.block_pages) {
        const int per = (p.query_block * p.G + p.row_tile - 1) / p.row_tile, blk = tile / per;
        r0 = blk * p.query_block * p.G + (tile - blk * per) * p.row_tile;
        end = min(end, (blk + 1) * p.query_block * p.G);
      }
      if (to < p.row_cap) p.row_list[to] = make_int4(seg, r0, min(p.row_tile, end - r0), k - tile * chunks);
    };
    const auto tile_item = [&](int seg, int ntok, int chunks, int n, int k, int to) {
      const int tile = n / chunks - 1 - k / chunks;  // the last tiles of a causal segment see most keys: first in the list
      int t0 = tile * 2 * p.tok_tile, end = ntok;
      if (p.block_pages) {
        const int per = (p.query_block + 2 * p.tok_tile - 1) / (2 * p.tok_tile), blk = tile / per;
        t0 = blk * p.query_block + (tile - blk * per) * 2 * p.tok_tile;
        end = min(end, (blk + 1) * p.query_block);
      }
      if (to < p.tile_cap) p.tile_list[to] = make_int4(seg, t0, min(2 * p.tok_tile, end - t0), k % chunks);
    };
    const bool many = cnt[0] + cnt[1] > kSelf;
    if (!many) {
      for (int k = 0; k < cnt[0]; ++k) row_item(i, s.ntok, s.chunks, k, row_base + at[0] + k);
      for (int k = 0; k < cnt[1]; ++k) tile_item(i, s.ntok, s.chunks, cnt[1], k, tile_base + at[1] + k);
    }
    for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
      const int l = __ffs(left) - 1, seg = i0 + warp * 32 + l;
      const int ntok = __shfl_sync(0xffffffffu, s.ntok, l), chunks = __shfl_sync(0xffffffffu, s.chunks, l);
      const int nr = __shfl_sync(0xffffffffu, cnt[0], l), nt = __shfl_sync(0xffffffffu, cnt[1], l);
      const int rb = row_base + __shfl_sync(0xffffffffu, at[0], l), tb = tile_base + __shfl_sync(0xffffffffu, at[1], l);
      for (int k = lane; k < nr; k += 32) row_item(seg, ntok, chunks, k, rb + k);
      for (int k = lane; k < nt; k += 32) tile_item(seg, ntok, chunks, nt, k, tb + k);
    }
    row_base += total[0];
    tile_base += total[1];
    part_base += total[2];
  }
  split = __syncthreads_or(split);
  if (tid == 0) {
    p.hdr->row_items = min(row_base, p.row_cap);
    p.hdr->tile_items = min(tile_base, p.tile_cap);
    p.hdr->split = split;
    p.hdr->next_tile = 0;
  }
}

// ---- row kernel -----------------------------------------------------------------------------------
// Block = one item: up to 8*NT rows of a segment for one KV head, over one chunk of its pages.  Its four warps take
// the pages in turn, each through a ring of its own (three pages of K and V, 16-byte async copies, rows 256 bytes
// with the 16-byte pieces rotated by the row so that ldmatrix is free of bank conflicts), and meet once at the end.
//   S[row][token] = Q K^T   m16n8k16, rows the M side (rows 8-15 are zero for NT = 1), K rows the B operand
//   O^T[channel][row] += V^T P^T: P as the B operand has the layout of the S accumulators.
// Bound by reading K and V.
constexpr int kRowWarps = 4, kRowStages = 3;
constexpr int kRowStageBytes = 2 * kPage * kD * 2;  // K page, V page: 8 KiB
constexpr int kRowSmem = kRowWarps * kRowStages * kRowStageBytes;

__device__ __forceinline__ void cp_async16_or_zero(uint32_t dst, const void* src, bool real) {
  const int n = real ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t a) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typename Elem<T>::T2 v;
  v.x = Elem<T>::from_f(a);
  v.y = Elem<T>::from_f(b);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <typename T, int NT>
__global__ void __launch_bounds__(kRowWarps * 32) prompt_rows_kernel(const AttnParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 ml_s[kRowWarps][8 * NT];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int n_items = p.hdr->row_items * p.Hkv;
  uint8_t* ring = smem + warp * (kRowStages * kRowStageBytes);
  const uint32_t ring_a = (uint32_t)__cvta_generic_to_shared(ring);
  for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
    const int4 it = p.row_list[item / p.Hkv];
    const int kvh = item % p.Hkv;
    const Segment s = p.segs[it.x];
    const int32_t* indices = (s.second ? p.indices2 : p.indices1) + s.kvbase;
    const int tok_first = it.y / p.G, tok_last = (it.y + it.z - 1) / p.G;
    // the pages: a run of the segment's, or of the block's list
    const int32_t* list = nullptr;
    int n_avail = pages_seen(s, tok_last, p.causal);
    if (p.block_pages) {
      const int64_t slot = (int64_t)(s.tok0 / p.query_block + it.x + tok_first / p.query_block) * p.Hkv + kvh;
      list = p.block_pages + slot * p.max_k;
      n_avail = min(max(p.block_npages[slot], 0), p.max_k);
    }
    const int first = it.w * s.chunk_pages;  // chunk_pages can be "all": the product is only used for chunk 0 then
    const int n_pg = max(0, min(n_avail - first, s.chunk_pages));
    // rows g and g + 8 of the tile: query row, and the last position it sees
    uint32_t qa[8][2 * NT];
    int limit[NT];
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      const int r = g + 8 * h;
      const bool ok = r < it.z;
      const int row = it.y + (ok ? r : 0), tok = row / p.G, head = kvh * p.G + row % p.G;
      limit[h] = !ok ? -1 : p.causal ? s.len - s.ntok + tok : s.len - 1;
      const T* src = static_cast<const T*>(p.q) + (int64_t)(s.tok0 + tok) * p.q_ts + head * kD;
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        qa[ks][h] = ok ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 2 * t) : 0u;
        qa[ks][NT + h] = ok ? *reinterpret_cast<const uint32_t*>(src + 16 * ks + 8 + 2 * t) : 0u;
      }
    }
    const int sure = p.causal ? s.len - s.ntok + tok_first : s.len - 1;  // every row sees positions up to here
    float o[8][NT][4], m[NT], l[NT];
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int h = 0; h < NT; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[c][h][e] = 0.f;
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      m[h] = -INFINITY;
      l[h] = 0.f;
    }
    // this warp's pages are first + warp + 4*i; lane j holds number 32*k + j of them: logical page and physical id
    const int mine = (n_pg - warp + kRowWarps - 1) / kRowWarps;
    int my_lp = 0, my_phys = -1;
    auto look_up = [&](int k) {
      const int i = 32 * k + lane;
      my_lp = 0x3fffff;
      my_phys = -1;
      if (i < mine) {
        const int at = first + warp + kRowWarps * i;
        my_lp = list ? list[at] : at;
        if (my_lp >= 0 && my_lp < s.npages) my_phys = indices[my_lp];
        if (my_phys < 0 || my_phys >= p.num_pages_total) {
          raise_flag(p.status, TWL_FLAG_BAD_INDEX);
          my_phys = -1;
          my_lp = 0x3fffff;  // behind every limit
        }
      }
    };
    auto fetch = [&](int i, int lp, int phys) {
      const uint32_t dst = ring_a + (i % kRowStages) * kRowStageBytes;
      const bool ok = phys >= 0;
      const size_t slab = ((size_t)(ok ? phys : 0) * p.Hkv + kvh) * (kPage * kD);
      const T* ksrc = static_cast<const T*>(p.k_pages) + slab;
      const T* vsrc = static_cast<const T*>(p.v_pages) + slab;
      const int valid = ok ? min(kPage, s.len - lp * kPage) : 0;  // rows behind the sequence read as zero
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int piece = 32 * j + lane, row = piece >> 4, c = piece & 15;
        const uint32_t to = dst + row * 256 + ((c ^ (row & 7)) << 4);
        cp_async16_or_zero(to, ksrc + piece * 8, row < valid);
        cp_async16_or_zero(to + kPage * kD * 2, vsrc + piece * 8, row < valid);
      }
    };
    look_up(0);
    int next_lp, next_phys;
#pragma unroll
    for (int i = 0; i < kRowStages - 1; ++i) {
      next_lp = __shfl_sync(0xffffffffu, my_lp, i);
      next_phys = __shfl_sync(0xffffffffu, my_phys, i);
      if (i < mine) fetch(i, next_lp, next_phys);
      cp_async_commit();
    }
    int lp_ring[kRowStages - 1];  // logical pages of the stages in flight
#pragma unroll
    for (int i = 0; i < kRowStages - 1; ++i) lp_ring[i] = __shfl_sync(0xffffffffu, my_lp, i);
    for (int i = 0; i < mine; ++i) {
      const int ahead = i + kRowStages - 1;
      if ((ahead & 31) == 0) look_up(ahead >> 5);
      next_lp = __shfl_sync(0xffffffffu, my_lp, ahead & 31);
      next_phys = __shfl_sync(0xffffffffu, my_phys, ahead & 31);
      if (ahead < mine) fetch(ahead, next_lp, next_phys);
      cp_async_commit();
      cp_async_wait<kRowStages - 1>();
      __syncwarp();
      const int lp = lp_ring[0];
#pragma unroll
      for (int j = 0; j + 1 < kRowStages - 1; ++j) lp_ring[j] = lp_ring[j + 1];
      lp_ring[kRowStages - 2] = next_lp;
      const uint32_t base = ring_a + (i % kRowStages) * kRowStageBytes;
      const int fr = (lane & 7) + ((lane >> 4) << 3), fc = (lane >> 3) & 1;  // ldmatrix row and piece of this lane
      float sc[2][4] = {};
#pragma unroll
      for (int ks = 0; ks < 8; ++ks) {
        uint32_t b[4];
        ldsm4(b, base + fr * 256 + (((2 * ks + fc) ^ (fr & 7)) << 4));
#pragma unroll
        for (int n = 0; n < 2; ++n)
          MmaTile<T>::run(sc[n], qa[ks][0], NT == 2 ? qa[ks][1] : 0u, qa[ks][NT], NT == 2 ? qa[ks][NT + 1] : 0u,
                          b[2 * n], b[2 * n + 1]);
      }
      uint32_t pb[NT][2];
      float f[NT];
      bool moved = false;
      const int pos = lp * kPage + 2 * t;
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        float x[4] = {sc[0][2 * h] * p.scale_log2, sc[0][2 * h + 1] * p.scale_log2, sc[1][2 * h] * p.scale_log2,
                      sc[1][2 * h + 1] * p.scale_log2};
        if (lp * kPage + kPage - 1 > sure) {
          if (pos > limit[h]) x[0] = -INFINITY;
          if (pos + 1 > limit[h]) x[1] = -INFINITY;
          if (pos + 8 > limit[h]) x[2] = -INFINITY;
          if (pos + 9 > limit[h]) x[3] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float mn = fmaxf(m[h], mx);
        const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen so far: every weight is 2^-inf = 0
        f[h] = ex2(m[h] - ref);
        moved |= mn != m[h];
        m[h] = mn;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = ex2(x[e] - ref);
        l[h] = l[h] * f[h] + (x[0] + x[1]) + (x[2] + x[3]);
        // weights go to the tensor cores in the model type (half a step of it each); their sum stays unrounded
        pb[h][0] = pack2<T>(x[0], x[1]);
        pb[h][1] = pack2<T>(x[2], x[3]);
      }
      if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int h = 0; h < NT; ++h) {  // accumulator columns are rows 2t and 2t+1 of the half
          const float f0 = __shfl_sync(0xffffffffu, f[h], 8 * t), f1 = __shfl_sync(0xffffffffu, f[h], 8 * t + 4);
#pragma unroll
          for (int c = 0; c < 8; ++c) {
            o[c][h][0] *= f0;
            o[c][h][1] *= f1;
            o[c][h][2] *= f0;
            o[c][h][3] *= f1;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        uint32_t a[4];
        ldsm4t(a, base + kPage * kD * 2 + fr * 256 + (((2 * c + fc) ^ (fr & 7)) << 4));
#pragma unroll
        for (int h = 0; h < NT; ++h) MmaTile<T>::run(o[c][h], a[0], a[1], a[2], a[3], pb[h][0], pb[h][1]);
      }
      __syncwarp();  // the stage is refilled in the next round
    }
    cp_async_wait<0>();
    // the four warps' results meet in shared memory: [warp][row][channel], a padded row per warp
#pragma unroll
    for (int h = 0; h < NT; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t == 0) ml_s[warp][g + 8 * h] = make_float2(m[h], l[h]);
    }
    __syncthreads();  // every warp is done with its ring
    float* acc_s = reinterpret_cast<float*>(smem);
    constexpr int kRowPitch = kD + 4;
#pragma unroll
    for (int c = 0; c < 8; ++c)
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        float* to = acc_s + (warp * 8 * NT + 8 * h + 2 * t) * kRowPitch + 16 * c + g;
        to[0] = o[c][h][0];
        to[kRowPitch] = o[c][h][1];
        to[8] = o[c][h][2];
        to[kRowPitch + 8] = o[c][h][3];
      }
    __syncthreads();
    for (int r = warp; r < it.z; r += kRowWarps) {
      float mm = -INFINITY;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) mm = fmaxf(mm, ml_s[w][r].x);
      const float ref = mm == -INFINITY ? 0.f : mm;
      float ll = 0.f;
      float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w) {
        const float2 v = ml_s[w][r];
        const float fw = ex2(v.x - ref);
        ll += v.y * fw;
        const float4 x = *reinterpret_cast<const float4*>(acc_s + (w * 8 * NT + r) * kRowPitch + 4 * lane);
        a.x += x.x * fw;
        a.y += x.y * fw;
        a.z += x.z * fw;
        a.w += x.w * fw;
      }
      const int row = it.y + r, tok = row / p.G, head = kvh * p.G + row % p.G;
      if (s.pbase >= 0) {
        const int64_t slot = s.pbase + ((int64_t)it.w * s.ntok + tok) * p.Hq + head;
        if (slot < p.part_cap) {
          if (ll != 0.f) *reinterpret_cast<float4*>(p.part_acc + slot * kD + 4 * lane) = a;
          if (lane == 0) p.part_ml[slot] = make_float2(mm, ll);
        }
      } else {
        const float inv = ll != 0.f ? 1.f / ll : 0.f;
        T* to = static_cast<T*>(p.out) + (int64_t)(s.tok0 + tok) * p.o_ts + head * kD + 4 * lane;
        *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
        if (p.lse && lane == 0)
          p.lse[(int64_t)(s.tok0 + tok) * p.Hq + head] = ll != 0.f ? (mm + log2f(ll)) * 0.69314718055994531f : -INFINITY;
      }
    }
    __syncthreads();  // before the next item's copies
  }
}

// ---- merge -----------------------------------------------------------------------------------------
// Warp = one output row (token, query head): the partial results of its segment's chunks, and of its group's prefix.
template <typename T>
__global__ void __launch_bounds__(256) prompt_merge_kernel(const AttnParams p) {
  pdl_wait();
  if (!p.always_partial && p.hdr->split == 0) return;
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.num_tokens * p.Hq;
  for (int64_t row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); row < rows; row += (int64_t)gridDim.x * 8) {
    const int tok = (int)(row / p.Hq), head = (int)(row - (int64_t)tok * p.Hq);
    float m = -INFINITY, l = 0.f;
    float4 a = make_float4(0.f, 0.f, 0.f, 0.f);
    bool found = false;
    for (int part = 0; part < 2; ++part) {
      const int n = part ? p.n_second : p.n_first;
      const int32_t* qo = part ? p.qo2 : p.qo1;
      if (n == 0) continue;
      int sidx = tok;
      if (qo) {  // last segment that starts at or before the token
        int lo = 0, hi = n;
        while (hi - lo > 1) {
          const int step = (hi - lo + 31) >> 5, c = lo + lane * step;
          const int cnt = __popc(__ballot_sync(0xffffffffu, c < hi && qo[c] <= tok));
          lo += (cnt > 0 ? cnt - 1 : 0) * step;
          hi = min(hi, lo + step);
        }
        sidx = lo;
      }
      if (sidx >= n) continue;
      const Segment s = p.segs[(part ? p.n_first : 0) + sidx];
      if (tok < s.tok0 || tok >= s.tok0 + s.ntok) continue;
      if (s.pbase < 0) continue;
      found = true;
      // a lane takes a chunk's maximum and sum; the accumulators follow, four in flight
      const int64_t slot0 = s.pbase + (int64_t)(tok - s.tok0) * p.Hq + head, step = (int64_t)s.ntok * p.Hq;
      for (int c0 = 0; c0 < s.chunks; c0 += 32) {
        const int n = min(32, s.chunks - c0);
        float2 v = make_float2(-INFINITY, 0.f);
        if (lane < n && slot0 + (c0 + lane) * step < p.part_cap) v = p.part_ml[slot0 + (c0 + lane) * step];
        const float mn = fmaxf(m, warp_max(v.x)), ref = mn == -INFINITY ? 0.f : mn;
        const float f0 = ex2(m - ref);
        const float w = v.y == 0.f ? 0.f : ex2(v.x - ref);  // (a NaN sum goes on)
        l = l * f0 + warp_sum(v.y * w);
        a.x *= f0;
        a.y *= f0;
        a.z *= f0;
        a.w *= f0;
        m = mn;
        const uint32_t has = __ballot_sync(0xffffffffu, v.y != 0.f);  // the others' accumulators were not written
        for (int c = 0; c < n; c += 4) {
          float4 x[4];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if ((has >> (c + k)) & 1) x[k] = *reinterpret_cast<const float4*>(p.part_acc + (slot0 + (c0 + c + k) * step) * kD + 4 * lane);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float f = __shfl_sync(0xffffffffu, w, (c + k) & 31);
            if ((has >> (c + k)) & 1) {
              a.x += x[k].x * f;
              a.y += x[k].y * f;
              a.z += x[k].z * f;
              a.w += x[k].w * f;
            }
          }
        }
      }
    }
    if (!found) continue;
    const float inv = l != 0.f ? 1.f / l : 0.f;
    T* to = static_cast<T*>(p.out) + (int64_t)tok * p.o_ts + head * kD + 4 * lane;
    *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(a.x * inv, a.y * inv), pack2<T>(a.z * inv, a.w * inv));
    if (p.lse && lane == 0) p.lse[row] = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
  }
}

// ---- host ------------------------------------------------------------------------------------------
struct WorkspaceLayout {
  size_t hdr, segs, row_list, tile_list, acc, ml, total;
  int64_t rows;
  int32_t row_cap, tile_cap;
};

static inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

constexpr int kTilesPerSm = 1;
constexpr int kRowBlocksPerSm = 2;

// `tokens` query tokens in n_seg segments; prefix: every row has partial results of both its segments.
static WorkspaceLayout workspace_layout(int64_t tokens, int64_t n_seg, int64_t Hq, int64_t Hkv, int64_t max_pages,
                                        int64_t query_block, bool prefix) {
  WorkspaceLayout w;
  const int64_t G = Hq / Hkv, row_target = (int64_t)num_sms() * kRowBlocksPerSm * 2, tile_target = num_sms() * kTilesPerSm;
  const int64_t tt = kPage * 8 / G;  // tokens of a 128-row tile
  const int64_t blocks = query_block > 0 ? tokens / query_block + n_seg : n_seg;  // runs that are cut into tiles
  // items per KV head without key chunks, and at most two targets more where keys are split
  const int64_t row_u = n_seg * (kFewRows / 8);  // at most 16 rows a segment, in tiles of 8 or 16
  const int64_t tile_u = tokens / (2 * tt) + blocks;
  w.row_cap = (int32_t)(row_u + 2 * row_target + 1);
  w.tile_cap = (int32_t)(tile_u + 2 * tile_target + 1);
  const int64_t chunks = (max_pages + kRowChunkMin - 1) / kRowChunkMin;
  const int64_t most = tokens * Hq * (prefix ? 2 * chunks : chunks);
  const int64_t split = 2 * row_target * 16 + 2 * tile_target * 2 * tt * G + (prefix ? 2 * tokens * Hq : 0);
  w.rows = !prefix && chunks <= 1 ? 0 : most < split ? most : split;
  size_t at = 0;
  w.hdr = at;
  at = up256(at + sizeof(PlanHeader));
  w.segs = at;
  at = up256(at + sizeof(Segment) * n_seg);
  w.row_list = at;
  at = up256(at + sizeof(int4) * w.row_cap);
  w.tile_list = at;
  at = up256(at + sizeof(int4) * w.tile_cap);
  w.ml = at;
  at = up256(at + sizeof(float2) * w.rows);
  w.acc = at;
  at = up256(at + sizeof(float) * kD * w.rows);
  w.total = at;
  return w;
}

static void place_workspace(AttnParams& p, const WorkspaceLayout& w, void* workspace) {
  uint8_t* base = static_cast<uint8_t*>(workspace);
  p.hdr = reinterpret_cast<PlanHeader*>(base + w.hdr);
  p.segs = reinterpret_cast<Segment*>(base + w.segs);
  p.row_list = reinterpret_cast<int4*>(base + w.row_list);
  p.tile_list = reinterpret_cast<int4*>(base + w.tile_list);
  p.part_ml = reinterpret_cast<float2*>(base + w.ml);
  p.part_acc = reinterpret_cast<float*>(base + w.acc);
  p.part_cap = w.rows;
  p.row_cap = w.row_cap;
  p.tile_cap = w.tile_cap;
  p.row_target = num_sms() * kRowBlocksPerSm * 2;
  p.tile_target = num_sms() * kTilesPerSm;
}

template <typename T>
static int run_attention(const AttnParams& p, int dtype, bool need_merge, cudaStream_t st) {
  const int plan_threads = p.n_first + p.n_second <= 256 ? 256 : kPlanThreads;
  TWL_CUDA_TRY(launch_chain(prompt_plan_kernel, dim3(1), dim3(plan_threads), 0, st, p));
  const dim3 rows_grid((unsigned)(num_sms() * kRowBlocksPerSm));
  if (p.row_tile == 8) {
    TWL_CUDA_TRY(cudaFuncSetAttribute(prompt_rows_kernel<T, 1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmem));
    TWL_CUDA_TRY(launch_chain(prompt_rows_kernel<T, 1>, rows_grid, dim3(kRowWarps * 32), kRowSmem, st, p));
  } else {
    TWL_CUDA_TRY(cudaFuncSetAttribute(prompt_rows_kernel<T, 2>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRowSmem));
    TWL_CUDA_TRY(launch_chain(prompt_rows_kernel<T, 2>, rows_grid, dim3(kRowWarps * 32), kRowSmem, st, p));
  }
  if ((int64_t)p.num_tokens * p.G > p.few_rows) {
    const int bad = tile_attention_launch(p, dtype, st);
    if (bad != TWL_OK) return bad;
  }
  if (need_merge) {
    const int64_t blocks = ((int64_t)p.num_tokens * p.Hq + 7) / 8, most = (int64_t)num_sms() * 8;
    TWL_CUDA_TRY(launch_chain(prompt_merge_kernel<T>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, st, p));
  }
  return TWL_OK;
}

}  // namespace twl

static int check_attention(int dtype, int32_t num_tokens, int32_t batch, int32_t num_q_heads, int32_t num_kv_heads,
                           int32_t num_pages_total, int32_t max_pages) {
  if (num_tokens <= 0 || batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages_total <= 0 || max_pages <= 0 ||
      num_q_heads % num_kv_heads != 0)
    return TWL_ERR_BAD_ARG;
  if (dtype != TWL_F16 && dtype != TWL_BF16) return TWL_ERR_UNSUPPORTED;
  if (num_q_heads / num_kv_heads > 128) return TWL_ERR_UNSUPPORTED;
  if ((int64_t)num_pages_total * num_kv_heads * TWL_PAGE_SIZE >= 0x7fffffffLL) return TWL_ERR_TOO_LARGE;
  return TWL_OK;
}

extern "C" size_t twl_prompt_attn_workspace_bytes(int32_t num_tokens, int32_t batch, int32_t num_q_heads,
                                                  int32_t num_kv_heads, int32_t max_pages, int32_t query_block) {
  if (check_attention(TWL_F16, num_tokens, batch, num_q_heads, num_kv_heads, 1, max_pages) != TWL_OK) return 0;
  return twl::workspace_layout(num_tokens, batch, num_q_heads, num_kv_heads, max_pages, query_block, false).total;
}

extern "C" int twl_prompt_attn(const void* q, int dtype, int64_t q_token_stride, const void* k_pages,
                               const void* v_pages, const int32_t* qo_indptr, const int32_t* kv_indptr,
                               const int32_t* kv_indices, const int32_t* kv_last_page_len, int32_t num_tokens,
                               int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t num_pages_total,
                               int32_t max_pages, int32_t causal, const int32_t* block_pages,
                               const int32_t* block_npages, int32_t max_k, int32_t query_block, float sm_scale,
                               void* out, float* lse, void* workspace, size_t workspace_bytes, int32_t* status,
                               void* stream) {
  using namespace twl;
  if (!q || !k_pages || !v_pages || !qo_indptr || !kv_indptr || !kv_indices || !kv_last_page_len || !out)
    return TWL_ERR_BAD_ARG;
  if ((block_pages == nullptr) != (block_npages == nullptr)) return TWL_ERR_BAD_ARG;
  if (block_pages && (max_k <= 0 || query_block <= 0)) return TWL_ERR_BAD_ARG;
  const int bad = check_attention(dtype, num_tokens, batch, num_q_heads, num_kv_heads, num_pages_total, max_pages);
  if (bad != TWL_OK) return bad;
  if (block_pages && query_block % kPage != 0) return TWL_ERR_UNSUPPORTED;
  if (!(sm_scale > 0.f)) return TWL_ERR_BAD_ARG;  // the running maximum is that of the scaled products
  if (!aligned(q, 16) || q_token_stride % 8 != 0 || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16))
    return TWL_ERR_MISALIGNED;
  const WorkspaceLayout w = workspace_layout(num_tokens, batch, num_q_heads, num_kv_heads, max_pages,
                                             block_pages ? query_block : 0, false);
  if (!workspace || workspace_bytes < w.total || !aligned(workspace, 256)) return TWL_ERR_WORKSPACE;
  AttnParams p = {};
  p.q = q; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out; p.lse = lse;
  p.q_ts = q_token_stride; p.o_ts = (int64_t)num_q_heads * kD;
  p.qo1 = qo_indptr; p.indptr1 = kv_indptr; p.indices1 = kv_indices; p.last1 = kv_last_page_len;
  p.n_first = batch; p.causal = causal != 0;
  p.block_pages = block_pages; p.block_npages = block_npages; p.max_k = max_k;
  p.query_block = query_block > 0 ? query_block : 1;
  p.num_tokens = num_tokens; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads;
  p.num_pages_total = num_pages_total; p.tok_tile = 128 / p.G; p.row_tile = 16; p.few_rows = kFewRows;
  p.scale_log2 = sm_scale * 1.44269504088896341f;
  p.status = status;
  place_workspace(p, w, workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == TWL_F16 ? run_attention<__half>(p, dtype, w.rows > 0, st)
                          : run_attention<__nv_bfloat16>(p, dtype, w.rows > 0, st);
}

extern "C" size_t twl_shared_prefix_workspace_bytes(int32_t batch, int32_t num_groups, int32_t num_q_heads,
                                                    int32_t num_kv_heads, int32_t max_pages) {
  if (num_groups <= 0 || check_attention(TWL_F16, batch, batch, num_q_heads, num_kv_heads, 1, max_pages) != TWL_OK)
    return 0;
  return twl::workspace_layout(batch, (int64_t)batch + num_groups, num_q_heads, num_kv_heads, max_pages, 0, true).total;
}

extern "C" int twl_shared_prefix_attn(const void* q, int dtype, int64_t q_token_stride, const void* k_pages,
                                      const void* v_pages, const int32_t* group_indptr, const int32_t* prefix_indptr,
                                      const int32_t* prefix_indices, const int32_t* prefix_last_page_len,
                                      const int32_t* kv_indptr, const int32_t* kv_indices,
                                      const int32_t* kv_last_page_len, int32_t batch, int32_t num_groups,
                                      int32_t num_q_heads, int32_t num_kv_heads, int32_t num_pages_total,
                                      int32_t max_pages, float sm_scale, void* out, float* lse, void* workspace,
                                      size_t workspace_bytes, int32_t* status, void* stream) {
  using namespace twl;
  // (an index list may be null where no sequence, or no group, has pages)
  if (!q || !k_pages || !v_pages || !group_indptr || !prefix_indptr || !prefix_last_page_len || !kv_indptr ||
      !kv_last_page_len || !out || num_groups <= 0)
    return TWL_ERR_BAD_ARG;
  const int bad = check_attention(dtype, batch, batch, num_q_heads, num_kv_heads, num_pages_total, max_pages);
  if (bad != TWL_OK) return bad;
  if (!(sm_scale > 0.f)) return TWL_ERR_BAD_ARG;
  if (!aligned(q, 16) || q_token_stride % 8 != 0 || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16))
    return TWL_ERR_MISALIGNED;
  const WorkspaceLayout w =
      workspace_layout(batch, (int64_t)batch + num_groups, num_q_heads, num_kv_heads, max_pages, 0, true);
  if (!workspace || workspace_bytes < w.total || !aligned(workspace, 256)) return TWL_ERR_WORKSPACE;
  AttnParams p = {};
  p.q = q; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out; p.lse = lse;
  p.q_ts = q_token_stride; p.o_ts = (int64_t)num_q_heads * kD;
  p.indptr1 = kv_indptr; p.indices1 = kv_indices; p.last1 = kv_last_page_len; p.n_first = batch;
  p.qo2 = group_indptr; p.indptr2 = prefix_indptr; p.indices2 = prefix_indices; p.last2 = prefix_last_page_len;
  p.n_second = num_groups; p.always_partial = 1; p.query_block = 1;
  p.num_tokens = batch; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads;
  p.num_pages_total = num_pages_total; p.tok_tile = 128 / p.G; p.row_tile = p.G <= 8 ? 8 : 16; p.few_rows = kFewRows;
  p.scale_log2 = sm_scale * 1.44269504088896341f;
  p.status = status;
  place_workspace(p, w, workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == TWL_F16 ? run_attention<__half>(p, dtype, true, st) : run_attention<__nv_bfloat16>(p, dtype, true, st);
}
