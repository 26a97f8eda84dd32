// Attention over the paged cache for more than one token at a time: a prompt's (prompt_attn) and a decode batch's
// over a shared prefix (shared_prefix_attn): plan, row kernel, merge and the C entry points.
//
//   out[row] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * (q.k_j - max)) over the keys the row may see,
// one pass over the keys with a running maximum and sum (32-bit), joined over key chunks as
//   m = max_c m_c,  l = sum_c l_c 2^(m_c - m),  out = sum_c acc_c 2^(m_c - m) / l.
#include "prompt.cuh"

namespace twl {

// ---- plan -------------------------------------------------------------------------------------------
// One block: lengths and work of every segment, the run of a warp of the row kernel, the key chunks and the list of the
// tile kernel.  A separate launch, so that the lengths stay on the device and the other kernels find their work with one
// load.
constexpr int kPlanThreads = 1024;
constexpr int kRowRunMin = 4;      // pages: shorter runs cost more in the merge than they balance
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
  s.units = 0;
  s.chunks = 1;
  s.chunk_pages = 0x3fffffff;
  s.start = 0;
  s.pbase = -1;
  const bool bad = s.tok0 < 0 || s.ntok < 0 || s.tok0 + s.ntok > p.num_tokens || s.npages < 0 ||
                   (s.npages > 0 && (last < 1 || last > kPage));
  if (bad) {
    raise_flag(p.status, TWL_FLAG_BAD_INDEX);
    s.ntok = 0;
  }
  if (s.npages <= 0 || bad) s.npages = 0;
  s.len = s.npages ? (s.npages - 1) * kPage + last : 0;
  s.few = s.ntok * p.G <= p.row_tile;
  if (s.few && s.ntok > 0) s.units = p.block_pages ? min(s.npages, p.max_k) : s.npages;
  return s;
}

// tiles of the tile kernel (per KV head); a tile stays within one query block when there are block lists
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

__global__ void __launch_bounds__(kPlanThreads) prompt_plan_kernel(const AttnParams p) {
  __shared__ long long sums[kPlanThreads / 32][4];
  __shared__ long long scan[kPlanThreads / 32][3];
  __shared__ int longest;
  pdl_wait();
  pdl_release();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n_thr = blockDim.x, n_warps = n_thr >> 5;
  const int n_seg = p.n_first + p.n_second;
  const auto pages_of = [&](const Segment& s) { return p.block_pages ? min(s.npages, p.max_k) : s.npages; };
  // units of the row kernel; tiles and tiles x pages of the tile kernel
  long long v[3] = {0, 0, 0};
  Segment mine;  // this thread's segment of the first round
  mine.ntok = 0;
  for (int i = tid; i < n_seg; i += n_thr) {
    const Segment s = load_segment(p, i);
    if (i == tid) mine = s;
    if (s.few) {
      v[0] += (long long)p.Hkv * s.units;
    } else {
      const int n = tok_tiles(p, s.ntok) * p.Hkv;
      v[1] += n;
      v[2] += (long long)n * pages_of(s);
    }
  }
  block_sums<3>(v, sums);
  const int per_warp = (int)max((long long)kRowRunMin, (v[0] + p.row_warps - 1) / p.row_warps);
  // Key chunks.  With fewer tiles than blocks: one wave of equal chunks (a tile of w pages gives ceil(w/c) items, on average
  // w/c + 1/2; count, and lengthen by what is too much), unless that leaves more than a fifth of the blocks' time unused.
  // Otherwise chunks of a third of a block's share, so that the counter can balance them.
  const long long share = (v[2] + p.tile_target - 1) / p.tile_target;
  long long tc = 0;
  if (v[1] < p.tile_target) {
    const long long room = p.tile_target - v[1] / 2;
    tc = (max((v[2] + room - 1) / room, (long long)kTileChunkMin) + 7) & ~7LL;  // whole key tiles
    for (int round = 0; round < 3; ++round) {
      long long items[1] = {0};
      int long_chunk = 0;
      for (int i = tid; i < n_seg; i += n_thr) {
        const Segment s = i == tid ? mine : load_segment(p, i);
        if (s.few) continue;
        const int pages = pages_of(s), n = (int)max(1LL, (pages + tc - 1) / tc);
        items[0] += (long long)tok_tiles(p, s.ntok) * p.Hkv * n;
        long_chunk = max(long_chunk, (pages + n - 1) / n);
      }
      if (tid == 0) longest = 0;
      __syncthreads();
      atomicMax(&longest, long_chunk);
      block_sums<1>(items, sums);  // (its barriers order the maximum too)
      if (items[0] <= p.tile_target) break;
      tc = (tc * items[0] / p.tile_target + 8) & ~7LL;
    }
    if (share * 5 < longest * 4LL && share > 24 * 8) tc = 0;
  }
  if (tc == 0) tc = (max((share + 2) / 3, 16 * 8LL) + 7) & ~7LL;

  long long base[3] = {0, 0, 0};  // units, tile items, partial rows so far
  int merge = 0;
  for (int i0 = 0; i0 < n_seg; i0 += n_thr) {
    const int i = i0 + tid;
    Segment s;
    s.ntok = 0;
    s.chunks = 1;
    long long cnt[3] = {0, 0, 0};
    if (i < n_seg) {
      s = i0 == 0 ? mine : load_segment(p, i);
      const int pages = pages_of(s);
      if (s.few) {
        cnt[0] = (long long)p.Hkv * s.units;
        // so many units in a row touch at most so many warps
        cnt[2] = (long long)s.ntok * p.Hq * ((s.units + per_warp - 1) / per_warp + 1);
      } else {
        s.chunks = (int)max(1LL, (pages + tc - 1) / tc);
        s.chunk_pages = s.chunks == 1 ? 0x3fffffff : ((pages + s.chunks - 1) / s.chunks + 7) & ~7;  // equal ones
        cnt[1] = tok_tiles(p, s.ntok) * s.chunks;
        if (s.chunks > 1 || p.always_partial) cnt[2] = (long long)s.chunks * s.ntok * p.Hq;
      }
      merge |= cnt[2] > 0;
    }
    // exclusive sums over the segments
    long long inc[3] = {cnt[0], cnt[1], cnt[2]};
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        const long long x = __shfl_up_sync(0xffffffffu, inc[k], o);
        if (lane >= o) inc[k] += x;
      }
    if (lane == 31)
#pragma unroll
      for (int k = 0; k < 3; ++k) scan[warp][k] = inc[k];
    __syncthreads();
    long long at[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) {  // every warp scans the warps' totals
      long long w = lane < n_warps ? scan[lane][k] : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, w, o);
        if (lane >= o) w += x;
      }
      const long long before = __shfl_sync(0xffffffffu, w, (warp + 31) & 31);
      at[k] = base[k] + (warp ? before : 0) + inc[k] - cnt[k];
      base[k] += __shfl_sync(0xffffffffu, w, 31);
    }
    __syncthreads();
    if (i < n_seg) {
      s.start = at[0];
      if (cnt[2] > 0) s.pbase = at[2];
      p.segs[i] = s;
    }
    // a few items: their thread writes them; many: the warp does, segment by segment
    const auto tile_item = [&](int seg, int ntok, int chunks, int n, int k, long long to) {
      const int tile = n / chunks - 1 - k / chunks;  // the last tiles of a causal segment see most keys: first in the list
      int t0 = tile * 2 * p.tok_tile, end = ntok;
      if (p.block_pages) {
        const int per = (p.query_block + 2 * p.tok_tile - 1) / (2 * p.tok_tile), blk = tile / per;
        t0 = blk * p.query_block + (tile - blk * per) * 2 * p.tok_tile;
        end = min(end, (blk + 1) * p.query_block);
      }
      if (to < p.tile_cap) p.tile_list[to] = make_int4(seg, t0, min(2 * p.tok_tile, end - t0), k % chunks);
    };
    const bool many = cnt[1] > 4;
    if (!many)
      for (int k = 0; k < (int)cnt[1]; ++k) tile_item(i, s.ntok, s.chunks, (int)cnt[1], k, at[1] + k);
    for (uint32_t left = __ballot_sync(0xffffffffu, many); left; left &= left - 1) {
      const int l = __ffs(left) - 1, seg = i0 + warp * 32 + l;
      const int ntok = __shfl_sync(0xffffffffu, s.ntok, l), chunks = __shfl_sync(0xffffffffu, s.chunks, l);
      const int nt = __shfl_sync(0xffffffffu, (int)cnt[1], l);
      const long long tb = __shfl_sync(0xffffffffu, at[1], l);
      for (int k = lane; k < nt; k += 32) tile_item(seg, ntok, chunks, nt, k, tb + k);
    }
  }
  merge = __syncthreads_or(merge);
  if (tid == 0) {
    // (more work than the workspace is sized for: max_pages was smaller than a page count; what does not fit is left out)
    if (base[1] > p.tile_cap || base[2] > p.part_cap) raise_flag(p.status, TWL_FLAG_BAD_INDEX);
    p.hdr->units = base[0];
    p.hdr->per_warp = per_warp;
    p.hdr->tile_items = (int)min(base[1], (long long)p.tile_cap);
    p.hdr->merge = merge;
    p.hdr->next_tile = 0;
  }
}

// ---- row kernel -----------------------------------------------------------------------------------
// A warp works on its own: per_warp consecutive units of the line, a unit being one page for the up to 8*NT rows of a
// segment and one KV head (the order is segment, KV head, page).  Pages come through a ring of the warp's own (three
// pages of K and V, 16-byte async copies, rows of 256 bytes with the 16-byte pieces rotated by the row so that
// ldmatrix is free of bank conflicts), and the copies run two pages ahead across the ends of pieces (a KV head's units), the
// next piece's query rows with its first page: reading does not pause where a piece ends.
//   S[row][token] = Q K^T   m16n8k16, rows the M side (rows 8-15 are zero for NT = 1), K rows the B operand
//   O^T[channel][row] += V^T P^T: P as the B operand has the layout of the S accumulators.
// Each piece leaves a partial result per row; a KV head that several warps share has one from each.
// Bound by reading K and V: 5.4 TB/s over 342 MB of 32 KV heads in a profile, 5.1 over 375 MB of 8 (0.82 and 0.77 of
// the measured copy).
constexpr int kRowStages = 3;
constexpr int kPageKV = 2 * kPage * kD * 2;  // K page, V page: 8 KiB
template <int NT>
struct RowShape {
  static constexpr int kWarps = NT == 1 ? 8 : 7;  // what 227 KiB hold
  static constexpr int kQBytes = 8 * NT * kD * 2;
  static constexpr int kWarpBytes = kRowStages * kPageKV + 2 * kQBytes;
  static constexpr int kSmem = kWarps * kWarpBytes;
};

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

// A position in a warp's run: a piece is the part of one KV head's pages that the run covers.
struct RowCursor {
  int seg, kvh;
  int page, end;  // unit of the KV head, and where the piece ends
  int left;       // units of the run from this one on
  Segment s;

  // the segment that holds unit x of the line
  __device__ __forceinline__ void start(const AttnParams& p, long long x, int n) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = p.n_first + p.n_second;
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) >> 5, c = lo + lane * step;
      const int cnt = __popc(__ballot_sync(0xffffffffu, c < hi && p.segs[c].start <= x));
      lo += (cnt > 0 ? cnt - 1 : 0) * step;
      hi = min(hi, lo + step);
    }
    seg = lo;  // the last that starts at or before x; those after the last unit's start behind it
    s = p.segs[seg];
    const long long in = x - s.start;
    kvh = (int)(in / s.units);
    page = (int)(in - (long long)kvh * s.units);
    left = n;
    end = min(s.units, page + left);
  }
  // to the next unit; true when it is in another piece (or the run is over: left == 0)
  __device__ __forceinline__ bool step(const AttnParams& p) {
    --left;
    if (++page < end) return false;
    if (left > 0) {
      page = 0;
      if (++kvh == p.Hkv) {
        kvh = 0;
        do s = p.segs[++seg];
        while (s.units == 0);
      }
      end = min(s.units, left);
    }
    return true;
  }
};

template <typename T, int NT>
__global__ void __launch_bounds__(RowShape<NT>::kWarps * 32) prompt_rows_kernel(const AttnParams p) {
  using Shape = RowShape<NT>;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_release();  // the tile kernel sets itself up where a block ends, and waits for the others
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int per = p.hdr->per_warp;
  const long long w_id = (long long)blockIdx.x * Shape::kWarps + warp, x0 = w_id * per, units = p.hdr->units;
  if (x0 >= units) return;
  const uint32_t ring_a = (uint32_t)__cvta_generic_to_shared(smem + warp * Shape::kWarpBytes);
  const uint32_t q_a = ring_a + kRowStages * kPageKV;

  RowCursor f, c;  // where the copies are, and the arithmetic
  f.start(p, x0, (int)min((long long)per, units - x0));
  c = f;
  // Of the warps that share the first piece this is number `chunk`; every other piece begins in this run.
  int chunk = (int)(w_id - (c.s.start + (long long)c.kvh * c.s.units) / per);
  const uint32_t inv_g = 65536u / p.G + 1;  // row / G of the at most sixteen rows of a segment
  const auto tok_of = [&](int row) { return (int)((row * inv_g) >> 16); };
  // where this lane's pieces of a page go: rows 2j + lane/16, piece lane%16 rotated by the row; j mod 4 decides the rotation
  uint32_t to_off[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) to_off[j] = (2 * j + (lane >> 4)) * 256 + (((lane & 15) ^ (2 * j + (lane >> 4))) << 4);
  // lane j holds number 32*(page/32) + j of the piece's pages: logical page and physical id (or "none")
  constexpr int kNone = 0x7ffffff;  // a logical page behind every limit: its last position is 2^31 - 1
  int my_lp = kNone, my_phys = -1, window = -1, window_seg = -1;
  const auto look_up = [&]() {
    const int w = f.page >> 5;
    if (w == window && f.seg == window_seg && !p.block_pages) return;  // another KV head of the same pages
    window = w;
    window_seg = f.seg;
    int n = f.s.npages;
    const int32_t* list = nullptr;
    if (p.block_pages) {
      const int64_t slot = (int64_t)(f.s.tok0 / p.query_block + f.seg) * p.Hkv + f.kvh;  // (all in one query block)
      n = min(max(p.block_npages[slot], 0), p.max_k);
      list = p.block_pages + slot * p.max_k;
    }
    const int at = 32 * w + lane;
    my_lp = kNone;
    my_phys = -1;
    if (at < n) {
      my_lp = list ? list[at] : at;
      if (my_lp >= 0 && my_lp < f.s.npages) my_phys = ((f.s.second ? p.indices2 : p.indices1) + f.s.kvbase)[my_lp];
      if (my_phys < 0 || my_phys >= p.num_pages_total) {
        raise_flag(p.status, TWL_FLAG_BAD_INDEX);
        my_phys = -1;
        my_lp = kNone;
      }
    }
  };
  int f_stage = 0, f_piece = 0;  // stage of the next copies, pieces begun
  bool f_first = true;
  // the next page (and, before a piece's first, its query rows) into the ring; returns the logical page
  const auto fetch = [&]() -> int {
    int lp = kNone;
    if (f.left > 0) {
      if (f_first || (f.page & 31) == 0) look_up();
      if (f_first) {
        const uint32_t dst = q_a + (f_piece & 1) * Shape::kQBytes;
        const int n = f.s.ntok * p.G;
        const T* src = static_cast<const T*>(p.q) + (int64_t)f.s.tok0 * p.q_ts + f.kvh * p.G * kD + (lane & 15) * 8;
#pragma unroll
        for (int j = 0; j < 4 * NT; ++j) {
          const int r = 2 * j + (lane >> 4), row = r < n ? r : 0, tok = tok_of(row);
          cp_async16_or_zero(dst + to_off[j & 3] + (j >> 2) * 2048, src + tok * p.q_ts + (row - tok * p.G) * kD, r < n);
        }
        ++f_piece;
      }
      lp = __shfl_sync(0xffffffffu, my_lp, f.page & 31);
      const int phys = __shfl_sync(0xffffffffu, my_phys, f.page & 31);
      const uint32_t dst = ring_a + f_stage * kPageKV;
      const size_t at = ((size_t)max(phys, 0) * p.Hkv + f.kvh) * (kPage * kD) + lane * 8;
      const T* ksrc = static_cast<const T*>(p.k_pages) + at;
      const T* vsrc = static_cast<const T*>(p.v_pages) + at;
      if (phys >= 0 && f.s.len - lp * kPage >= kPage) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t to = dst + to_off[j & 3] + (j >> 2) * 2048;
          cp_async16(to, ksrc + j * 256);
          cp_async16(to + kPage * kD * 2, vsrc + j * 256);
        }
      } else {  // rows behind the sequence (or of a page that is not there) read as zero
        const int valid = phys >= 0 ? f.s.len - lp * kPage : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const uint32_t to = dst + to_off[j & 3] + (j >> 2) * 2048;
          cp_async16_or_zero(to, ksrc + j * 256, 2 * j + (lane >> 4) < valid);
          cp_async16_or_zero(to + kPage * kD * 2, vsrc + j * 256, 2 * j + (lane >> 4) < valid);
        }
      }
      if (++f_stage == kRowStages) f_stage = 0;
      f_first = f.step(p);
    }
    cp_async_commit();
    return lp;
  };

  uint32_t qa[8][2 * NT];
  int limit[NT], sure = 0;
  float o[8][NT][4], m[NT], l[NT];
  bool first = true;
  int stage = 0, piece = 0;
  int lp_ring[kRowStages - 1];  // logical pages of the stages in flight
#pragma unroll
  for (int i = 0; i < kRowStages - 1; ++i) lp_ring[i] = fetch();
  const int fr = (lane & 7) + ((lane >> 4) << 3), fc = (lane >> 3) & 1;  // ldmatrix row and piece of this lane
  while (c.left > 0) {
    cp_async_wait<kRowStages - 2>();
    __syncwarp();
    if (first) {
      const uint32_t src = q_a + (piece & 1) * Shape::kQBytes;
      const int n = c.s.ntok * p.G;
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        const int r = g + 8 * h;
        limit[h] = r >= n ? -1 : p.causal ? c.s.len - c.s.ntok + tok_of(r) : c.s.len - 1;
        m[h] = -INFINITY;
        l[h] = 0.f;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks)
#pragma unroll
          for (int e = 0; e < 2; ++e)
            asm volatile("ld.shared.u32 %0, [%1];"
                         : "=r"(qa[ks][e * NT + h])
                         : "r"(src + r * 256 + (((2 * ks + e) ^ g) << 4) + 4 * t));
#pragma unroll
        for (int k = 0; k < 8; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) o[k][h][e] = 0.f;
      }
      sure = p.causal ? c.s.len - c.s.ntok : c.s.len - 1;  // every row sees positions up to here
      ++piece;
      __syncwarp();  // before the slot is filled again
    }
    const int lp = lp_ring[0];
#pragma unroll
    for (int j = 0; j + 1 < kRowStages - 1; ++j) lp_ring[j] = lp_ring[j + 1];
    lp_ring[kRowStages - 2] = fetch();

    const uint32_t base = ring_a + stage * kPageKV;
    if (++stage == kRowStages) stage = 0;
    float sc[2][4] = {};
#pragma unroll
    for (int ks = 0; ks < 8; ++ks) {
      uint32_t b[4];
      ldsm4(b, base + fr * 256 + (((2 * ks + fc) ^ (fr & 7)) << 4));
#pragma unroll
      for (int n = 0; n < 2; ++n)
        MmaTile<T>::run(sc[n], qa[ks][0], NT == 2 ? qa[ks][1] : 0u, qa[ks][NT], NT == 2 ? qa[ks][NT + 1] : 0u, b[2 * n],
                        b[2 * n + 1]);
    }
    uint32_t pb[NT][2];
    float fac[NT];
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
      const float mn = fmaxf(m[h], mx - kTopWeight<T>);
      const float ref = mn == -INFINITY ? 0.f : mn;  // nothing seen so far: every weight is 2^-inf = 0
      fac[h] = ex2(m[h] - ref);
      moved |= mn != m[h];
      m[h] = mn;
#pragma unroll
      for (int e = 0; e < 4; ++e) x[e] = ex2(x[e] - ref);
      l[h] = l[h] * fac[h] + (x[0] + x[1]) + (x[2] + x[3]);
      // weights go to the tensor cores in the model type (half a step of it each, see kTopWeight); their sum stays unrounded
      pb[h][0] = pack2<T>(x[0], x[1]);
      pb[h][1] = pack2<T>(x[2], x[3]);
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int h = 0; h < NT; ++h) {  // accumulator columns are rows 2t and 2t+1 of the half
        const float f0 = __shfl_sync(0xffffffffu, fac[h], 8 * t), f1 = __shfl_sync(0xffffffffu, fac[h], 8 * t + 4);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          o[k][h][0] *= f0;
          o[k][h][1] *= f1;
          o[k][h][2] *= f0;
          o[k][h][3] *= f1;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t a[4];
      ldsm4t(a, base + kPage * kD * 2 + fr * 256 + (((2 * k + fc) ^ (fr & 7)) << 4));
#pragma unroll
      for (int h = 0; h < NT; ++h) MmaTile<T>::run(o[k][h], a[0], a[1], a[2], a[3], pb[h][0], pb[h][1]);
    }
    if (c.page + 1 == c.end) {  // the piece's results: one for each row
      const int n = c.s.ntok * p.G;
      const int64_t slot0 = c.s.pbase + (int64_t)chunk * c.s.ntok * p.Hq + c.kvh * p.G;
      chunk = 0;
      const auto slot_of = [&](int r) {
        const int tok = tok_of(r);
        return slot0 + tok * p.Hq + (r - tok * p.G);
      };
#pragma unroll
      for (int h = 0; h < NT; ++h) {
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
        l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
        if (t == 0 && g + 8 * h < n) {
          const int64_t slot = slot_of(g + 8 * h);
          if (slot < p.part_cap) p.part_ml[slot] = make_float2(m[h], l[h]);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int r = 8 * h + 2 * t + e;
          if (r >= n) continue;
          const int64_t slot = slot_of(r);
          if (slot >= p.part_cap) continue;
          float* to = p.part_acc + slot * kD + g;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            to[16 * k] = o[k][h][e];
            to[16 * k + 8] = o[k][h][2 + e];
          }
        }
      }
    }
    first = c.step(p);
    __syncwarp();  // the stage is refilled in the next round
  }
  cp_async_wait<0>();
}

// ---- merge -----------------------------------------------------------------------------------------
// L lanes = one output row (token, query head), 128/L channels to a lane: the partial results of its segment's chunks (or of
// the warps that read its keys), and of its group's prefix.  Bound by the latency of three loads in a row (segment, maximum
// and sum, accumulators), so everything that can be asked for at once is.  L = 16 where there are enough rows to fill the
// GPU's warps twice (16K rows of 3 to 4 parts: 12.5 us, with L = 32 17.7), else 32 (2K rows of 18 parts: 7.1 us, 10.8).
template <typename T, int L>
__global__ void __launch_bounds__(256, 3) prompt_merge_kernel(const AttnParams p) {
  pdl_wait();
  if (p.hdr->merge == 0) return;
  const int per = p.hdr->per_warp;
  constexpr int W = kD / L, kFlight = 32 / W;  // channels of a lane, accumulators in flight
  const int lane = threadIdx.x & 31, sub = lane & (L - 1);
  const int64_t rows = (int64_t)p.num_tokens * p.Hq;
  // (all of a warp makes the same number of rounds)
  for (int64_t row0 = ((int64_t)blockIdx.x * 8 + (threadIdx.x >> 5)) * (32 / L); row0 < rows;
       row0 += (int64_t)gridDim.x * (256 / L)) {
    const int64_t row = row0 + lane / L;
    const int tok = row < rows ? (int)(row / p.Hq) : -1, head = (int)(row - (int64_t)tok * p.Hq);
    // the row's partial results: n[0] of its sequence's segment, n[1] of its group's, `step` slots apart
    int n[2] = {0, 0};
    int64_t slot0[2] = {0, 0}, step[2] = {0, 0};
    bool found = false;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      const int segs = part ? p.n_second : p.n_first;
      const int32_t* qo = part ? p.qo2 : p.qo1;
      if (segs == 0 || tok < 0) continue;
      int at = tok;
      if (qo) {  // last segment that starts at or before the token
        int lo = 0, hi = segs;
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (qo[mid] <= tok)
            lo = mid;
          else
            hi = mid;
        }
        at = lo;
      }
      if (at >= segs) continue;
      const Segment& s = p.segs[(part ? p.n_first : 0) + at];
      const int tok0 = s.tok0, ntok = s.ntok;
      const int64_t pbase = s.pbase;
      if (tok < tok0 || tok >= tok0 + ntok || pbase < 0) continue;
      found = true;
      slot0[part] = pbase + (int64_t)(tok - tok0) * p.Hq + head;
      step[part] = (int64_t)ntok * p.Hq;
      n[part] = s.chunks;
      if (s.few) {  // the warps whose runs touch the KV head's units
        const int units = s.units;
        const long long u = s.start + (long long)(head / p.G) * units;
        n[part] = units ? (int)((u + units - 1) / per - u / per) + 1 : 0;
      }
    }
    float m = -INFINITY, l = 0.f, a[W] = {};
    const int total = n[0] + n[1], most = __reduce_max_sync(0xffffffffu, total);
    // a lane takes a partial result's maximum and sum; the accumulators follow, several in flight
    for (int c0 = 0; c0 < most; c0 += L) {
      const int c_mine = c0 + sub;
      int64_t mine = p.part_cap;
      if (c_mine < n[0])
        mine = slot0[0] + c_mine * step[0];
      else if (c_mine < total)
        mine = slot0[1] + (c_mine - n[0]) * step[1];
      float2 v = make_float2(-INFINITY, 0.f);
      if (mine < p.part_cap) v = p.part_ml[mine];
      float mn = v.x;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      mn = fmaxf(m, mn);
      const float ref = mn == -INFINITY ? 0.f : mn;
      const float f0 = ex2(m - ref);
      const float w = v.y == 0.f ? 0.f : ex2(v.x - ref);  // (a NaN sum goes on)
      float sum = v.y * w;
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      l = l * f0 + sum;
#pragma unroll
      for (int e = 0; e < W; ++e) a[e] *= f0;
      m = mn;
      for (int c = 0; c < min(L, most - c0); c += kFlight) {
        float4 x[kFlight][W / 4];
        float f[kFlight];
#pragma unroll
        for (int k = 0; k < kFlight; ++k) {
          f[k] = __shfl_sync(0xffffffffu, w, c + k, L);
          const int64_t slot = __shfl_sync(0xffffffffu, mine, c + k, L);
#pragma unroll
          for (int e = 0; e < W / 4; ++e) {
            x[k][e] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (f[k] != 0.f)  // (no weight: its accumulator may not have been written; a NaN goes on)
              x[k][e] = reinterpret_cast<const float4*>(p.part_acc + slot * kD + W * sub)[e];
          }
        }
#pragma unroll
        for (int k = 0; k < kFlight; ++k)
#pragma unroll
          for (int e = 0; e < W / 4; ++e) {
            a[4 * e] += x[k][e].x * f[k];
            a[4 * e + 1] += x[k][e].y * f[k];
            a[4 * e + 2] += x[k][e].z * f[k];
            a[4 * e + 3] += x[k][e].w * f[k];
          }
      }
    }
    if (found) {
      const float inv = l != 0.f ? 1.f / l : 0.f;
      T* to = static_cast<T*>(p.out) + (int64_t)tok * p.o_ts + head * kD + W * sub;
#pragma unroll
      for (int e = 0; e < W; e += 4)
        *reinterpret_cast<uint2*>(to + e) =
            make_uint2(pack2<T>(a[e] * inv, a[e + 1] * inv), pack2<T>(a[e + 2] * inv, a[e + 3] * inv));
      if (p.lse && sub == 0) p.lse[row] = l != 0.f ? (m + log2f(l)) * 0.69314718055994531f : -INFINITY;
    }
  }
}

// ---- host ------------------------------------------------------------------------------------------
struct WorkspaceLayout {
  size_t hdr, segs, tile_list, acc, ml, total;
  int64_t rows;
  int32_t tile_cap;
};

static inline size_t up256(size_t x) { return (x + 255) / 256 * 256; }

// Query tokens in n_seg segments; prefix: every row has partial results of both its segments.
static WorkspaceLayout workspace_layout(int64_t tokens, int64_t n_seg, int64_t Hq, int64_t Hkv, int64_t max_pages,
                                        int64_t query_block, bool prefix) {
  WorkspaceLayout w;
  const int64_t G = Hq / Hkv, warps = (int64_t)num_sms() * RowShape<1>::kWarps, blocks = num_sms();
  const int64_t tt = 128 / G;  // tokens of a 128-row tile
  const int64_t runs = query_block > 0 ? tokens / query_block + n_seg : n_seg;  // tokens that are cut into tiles together
  const auto least = [](int64_t a, int64_t b) { return a < b ? a : b; };
  // tiles per KV head without key chunks, and at most six times the blocks more where keys are split: those of one wave, or of
  // more work the items longer than a third of a block's share, each cut into fewer pieces than it has thirds plus one
  w.tile_cap = (int32_t)(tokens / (2 * tt) + runs + 6 * blocks + 1);
  // partial rows of the row kernel: at most 16 rows a segment and KV head, one result from each warp that touches them,
  // which are the warps and one or two more for each
  const int64_t few = least(tokens * Hq * (prefix ? 2 : 1), n_seg * kFewRows * Hkv);
  const int64_t row_parts = least(few * ((max_pages + kRowRunMin - 1) / kRowRunMin + 1), few * 2 + warps * kFewRows);
  // and of the tile kernel: a row has those of one segment, or of two where a sequence's own token is more than few rows too
  const int64_t once = tokens * Hq * (prefix && G > kFewRows ? 2 : 1);
  const int64_t whole = once * ((max_pages + kTileChunkMin - 1) / kTileChunkMin);
  const bool no_parts = tokens * G <= 8 || (!prefix && max_pages <= kTileChunkMin);
  const int64_t tile_parts = no_parts ? 0 : least(whole, 6 * blocks * 2 * tt * G + (prefix ? once : 0));
  w.rows = row_parts + tile_parts;
  size_t at = 0;
  w.hdr = at;
  at = up256(at + sizeof(PlanHeader));
  w.segs = at;
  at = up256(at + sizeof(Segment) * n_seg);
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
  p.tile_list = reinterpret_cast<int4*>(base + w.tile_list);
  p.part_ml = reinterpret_cast<float2*>(base + w.ml);
  p.part_acc = reinterpret_cast<float*>(base + w.acc);
  p.part_cap = w.rows;
  p.tile_cap = w.tile_cap;
  p.row_warps = num_sms() * (p.row_tile == 8 ? RowShape<1>::kWarps : RowShape<2>::kWarps);
  p.tile_target = num_sms();
}

template <typename T, int NT>
static int launch_rows(const AttnParams& p, cudaStream_t st) {
  static int8_t done[kSmemDevices];
  TWL_CUDA_TRY(allow_smem(prompt_rows_kernel<T, NT>, RowShape<NT>::kSmem, done));
  TWL_CUDA_TRY(launch_chain(prompt_rows_kernel<T, NT>, dim3((unsigned)num_sms()), dim3(RowShape<NT>::kWarps * 32),
                            RowShape<NT>::kSmem, st, p));
  return TWL_OK;
}

template <typename T>
static int run_attention(const AttnParams& p, int dtype, cudaStream_t st) {
  const int n_seg = p.n_first + p.n_second, plan_threads = n_seg <= 128 ? 128 : n_seg <= 512 ? 512 : kPlanThreads;
  TWL_CUDA_TRY(launch_chain(prompt_plan_kernel, dim3(1), dim3(plan_threads), 0, st, p));
  int bad = p.row_tile == 8 ? launch_rows<T, 1>(p, st) : launch_rows<T, 2>(p, st);
  if (bad == TWL_OK && (int64_t)p.num_tokens * p.G > p.row_tile) bad = tile_attention_launch(p, dtype, st);
  if (bad != TWL_OK) return bad;
  const int64_t rows = (int64_t)p.num_tokens * p.Hq, most = (int64_t)num_sms() * 8;
  const bool halves = rows >= (int64_t)num_sms() * 48;
  const int64_t blocks = halves ? (rows + 15) / 16 : (rows + 7) / 8;
  const dim3 grid((unsigned)(blocks < most ? blocks : most));
  if (halves)
    TWL_CUDA_TRY(launch_chain(prompt_merge_kernel<T, 16>, grid, dim3(256), 0, st, p));
  else
    TWL_CUDA_TRY(launch_chain(prompt_merge_kernel<T, 32>, grid, dim3(256), 0, st, p));
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
  // (the index list may be null where no sequence has pages)
  if (!q || !k_pages || !v_pages || !qo_indptr || !kv_indptr || !kv_last_page_len || !out) return TWL_ERR_BAD_ARG;
  if ((block_pages == nullptr) != (block_npages == nullptr)) return TWL_ERR_BAD_ARG;
  if (block_pages && (max_k <= 0 || query_block <= 0)) return TWL_ERR_BAD_ARG;
  const int bad = check_attention(dtype, num_tokens, batch, num_q_heads, num_kv_heads, num_pages_total, max_pages);
  if (bad != TWL_OK) return bad;
  if (num_tokens == 1) q_token_stride = (int64_t)num_q_heads * kD;  // one token: its stride says nothing
  if (block_pages && query_block % kPage != 0) return TWL_ERR_UNSUPPORTED;
  if (!(sm_scale > 0.f)) return TWL_ERR_BAD_ARG;  // the running maximum is that of the scaled products
  if (!aligned(q, 16) || q_token_stride % 8 != 0 || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16))
    return TWL_ERR_MISALIGNED;
  const WorkspaceLayout w = workspace_layout(num_tokens, batch, num_q_heads, num_kv_heads, max_pages,
                                             block_pages ? query_block : 0, false);
  if (!workspace || workspace_bytes < w.total || !aligned(workspace, 256)) return TWL_ERR_WORKSPACE;
  AttnParams p = {};
  p.q = q; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out; p.lse = lse;
  p.q_ts = q_token_stride;
  p.o_ts = (int64_t)num_q_heads * kD;
  p.qo1 = qo_indptr; p.indptr1 = kv_indptr; p.indices1 = kv_indices; p.last1 = kv_last_page_len;
  p.n_first = batch; p.causal = causal != 0;
  p.block_pages = block_pages; p.block_npages = block_npages; p.max_k = max_k;
  p.query_block = query_block > 0 ? query_block : 1;
  p.num_tokens = num_tokens; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads;
  p.num_pages_total = num_pages_total; p.tok_tile = 128 / p.G; p.row_tile = 16;
  p.scale_log2 = sm_scale * 1.44269504088896341f;
  p.status = status;
  place_workspace(p, w, workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == TWL_F16 ? run_attention<__half>(p, dtype, st) : run_attention<__nv_bfloat16>(p, dtype, st);
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
  if (batch == 1) q_token_stride = (int64_t)num_q_heads * kD;  // one token: its stride says nothing
  if (!(sm_scale > 0.f)) return TWL_ERR_BAD_ARG;
  if (!aligned(q, 16) || q_token_stride % 8 != 0 || !aligned(k_pages, 16) || !aligned(v_pages, 16) || !aligned(out, 16))
    return TWL_ERR_MISALIGNED;
  const WorkspaceLayout w =
      workspace_layout(batch, (int64_t)batch + num_groups, num_q_heads, num_kv_heads, max_pages, 0, true);
  if (!workspace || workspace_bytes < w.total || !aligned(workspace, 256)) return TWL_ERR_WORKSPACE;
  AttnParams p = {};
  p.q = q; p.k_pages = k_pages; p.v_pages = v_pages; p.out = out; p.lse = lse;
  p.q_ts = q_token_stride;
  p.o_ts = (int64_t)num_q_heads * kD;
  p.indptr1 = kv_indptr; p.indices1 = kv_indices; p.last1 = kv_last_page_len; p.n_first = batch;
  p.qo2 = group_indptr; p.indptr2 = prefix_indptr; p.indices2 = prefix_indices; p.last2 = prefix_last_page_len;
  p.n_second = num_groups; p.always_partial = 1; p.query_block = 1;
  p.num_tokens = batch; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.G = num_q_heads / num_kv_heads;
  p.num_pages_total = num_pages_total; p.tok_tile = 128 / p.G;
  // (a batch of up to sixteen rows per KV head is one row tile, its prefixes' too)
  p.row_tile = p.G <= 8 && batch * p.G > kFewRows ? 8 : 16;
  p.scale_log2 = sm_scale * 1.44269504088896341f;
  p.status = status;
  place_workspace(p, w, workspace);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  return dtype == TWL_F16 ? run_attention<__half>(p, dtype, st) : run_attention<__nv_bfloat16>(p, dtype, st);
}
