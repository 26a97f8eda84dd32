// A prompt's (or a decode step's) way into the paged cache in one pass: rotary positions on q and k, K and V
// rows into their pages, INT4 slabs and page (min, max) metadata; and the INT4 slabs read back as values.
//
// Rotation of a head's first R channels at position p, with the angle a_i = p * f_i of pair i < R/2:
//   x'_u = x_u cos a_i - x_v sin a_i,  x'_v = x_v cos a_i + x_u sin a_i,
// (u, v) = (i, i + R/2), or (2i, 2i + 1) when interleaved.  cos and sin carry attention_scale.  Angles are formed
// and reduced to a fraction of a turn in 64 bits (at position 10^5 a 32-bit product is off by 0.004 rad), and so are
// its sine and cosine, once per page and pair; the rotation is 32-bit and rounded once to the model type.
//
// Bound: HBM.  Every row is read once and written once; the INT4 slab and the metadata of a page are made from
// the rows while they are in registers: 20K ragged tokens of 32/8 heads in 109 us, 4.7 TB/s.  The decode form (one token per
// sequence) is bound by the latency of a launch and of three dependent loads (the sequence's entries, its page, the rows): 5 us.
#include "common.cuh"

namespace twl {

struct RopeParams {
  const void *q, *k, *v;
  void* q_out;
  int64_t q_ts, q_hs, k_ts, k_hs, v_ts, v_hs, o_ts, o_hs;  // token and head strides in elements
  const void* positions;                                   // int32 / int64 [T], or null: the cache position
  const double* freqs;                                     // [R/2] radians per position
  void *k_pages, *v_pages, *kmeta;
  uint8_t* k4;
  const int32_t *qo_indptr, *indptr, *indices, *last_len;
  int32_t* status;
  int32_t batch, Hq, Hkv, num_tokens, num_pages_total, rotary, pos64, heads_per_block, wide;
  double attn_scale;
};

constexpr int kRopeWarps = 8;

// Rows of the caller's tensors: 16-byte pieces, or two of 8 bytes where a base or stride asks for it.
template <typename T>
__device__ __forceinline__ uint4 load_row16(const T* p, int wide) {
  if (wide) return ldg_stream_u4(p);
  const uint2 a = ldg_stream_u2(p), b = ldg_stream_u2(p + 4);
  return make_uint4(a.x, a.y, b.x, b.y);
}
// The same of q, which may be written in place: the read-only loads above are undefined for memory that the kernel writes.
template <typename T>
__device__ __forceinline__ uint4 load_q16(const T* p, int wide) {
  uint4 r;
  if (wide)
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w) : "l"(p) : "memory");
  else
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0,%1}, [%4];\n\tld.global.L1::no_allocate.v2.u32 {%2,%3}, [%4+8];"
                 : "=&r"(r.x), "=&r"(r.y), "=&r"(r.z), "=&r"(r.w) : "l"(p) : "memory");
  return r;
}
template <typename T>
__device__ __forceinline__ void store_row16(T* p, const uint4& v, int wide) {
  if (wide) {
    *reinterpret_cast<uint4*>(p) = v;
  } else {
    reinterpret_cast<uint2*>(p)[0] = make_uint2(v.x, v.y);
    reinterpret_cast<uint2*>(p)[1] = make_uint2(v.z, v.w);
  }
}
static_assert(kRopeWarps * 2 == kPage, "a half-warp for every token of a page");

template <typename T>
__device__ __forceinline__ float rope_rnd(float x) {
  return Elem<T>::to_f(Elem<T>::from_f(x));
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, __half) {
  const __half2 v = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_pair(float a, float b, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// minimum and maximum of two pairs of values of the type, a NaN giving way to a number
template <typename T>
__device__ __forceinline__ uint32_t min_pair(uint32_t a, uint32_t b) {
  using T2 = typename Elem<T>::T2;
  const T2 r = __hmin2(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
template <typename T>
__device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  using T2 = typename Elem<T>::T2;
  const T2 r = __hmax2(*reinterpret_cast<T2*>(&a), *reinterpret_cast<T2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}

// The 4-bit codes of a lane's eight values of a group of 32 (four lanes), with the results of quantize_k_pages, which
// rounds every step to the type: code = rint(rnd(rnd(x - min) / scale)).  The quotients are correctly rounded from the
// reciprocal by one correction of the remainder, q + (t - q s) / s (Markstein 1990): both fused steps are exact here, t and
// s having at most 11 bits.
template <typename T>
__device__ __forceinline__ uint32_t codes8(const uint32_t (&u)[4], float* scale_out, float* min_out) {
  uint32_t lo = min_pair<T>(min_pair<T>(u[0], u[1]), min_pair<T>(u[2], u[3]));
  uint32_t hi = max_pair<T>(max_pair<T>(u[0], u[1]), max_pair<T>(u[2], u[3]));
#pragma unroll
  for (int o = 2; o > 0; o >>= 1) {
    lo = min_pair<T>(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = max_pair<T>(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  const float2 l2 = Elem<T>::to_f2(lo), h2 = Elem<T>::to_f2(hi);
  const float mn = fminf(l2.x, l2.y), mx = fmaxf(h2.x, h2.y);
  const float range = fmaxf(rope_rnd<T>(mx - mn), rope_rnd<T>(1e-9f));
  const float scale = rope_rnd<T>(__fdiv_rn(range, 15.f));
  const float inv = scale > 0.f ? __frcp_rn(scale) : 0.f;  // a group without a range: every code is 0
  uint32_t word = 0;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = Elem<T>::to_f2(u[k]);
    const float2 d = Elem<T>::to_f2(pack_pair(x.x - mn, x.y - mn, T()));
    float q0 = d.x * inv, q1 = d.y * inv;
    q0 = fmaf(fmaf(-q0, scale, d.x), inv, q0);
    q1 = fmaf(fmaf(-q1, scale, d.y), inv, q1);
    const float2 r = Elem<T>::to_f2(pack_pair(q0, q1, T()));
    // adding 1.5 * 2^23 rounds to the nearest integer (even on ties), which is then in the low bits
    const uint32_t c0 = __float_as_uint(fminf(fmaxf(r.x, 0.f), 15.f) + 12582912.f) & 15u;
    const uint32_t c1 = __float_as_uint(fminf(fmaxf(r.y, 0.f), 15.f) + 12582912.f) & 15u;
    word |= (c0 | (c1 << 4)) << (8 * k);
  }
  *scale_out = scale;
  *min_out = mn;
  return word;
}
template <typename T>
__device__ __forceinline__ uint4 pack8(const float (&x)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    typename Elem<T>::T2 v;
    v.x = Elem<T>::from_f(x[2 * k]);
    v.y = Elem<T>::from_f(x[2 * k + 1]);
    w[k] = *reinterpret_cast<uint32_t*>(&v);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// cos and sin for the eight channels of a lane (8 * (lane & 15) ..), two channels to a 64-bit register, the sines signed:
// channel j of a half turns with pair j, of interleaved channels 2k and 2k+1 with pair k.
template <bool INTER>
struct Angles {
  uint64_t c[4], s[4];
  __device__ __forceinline__ void read(const float* cos_row, const float* sin_row, int ch, int rotary) {
    if (INTER) {
      const float4 x = *reinterpret_cast<const float4*>(cos_row + (ch >> 1));
      const float4 y = *reinterpret_cast<const float4*>(sin_row + (ch >> 1));
      c[0] = f2(x.x, x.x); c[1] = f2(x.y, x.y); c[2] = f2(x.z, x.z); c[3] = f2(x.w, x.w);
      s[0] = f2(-y.x, y.x); s[1] = f2(-y.y, y.y); s[2] = f2(-y.z, y.z); s[3] = f2(-y.w, y.w);
    } else {
      const int half = rotary >> 1, at = ch >= half ? ch - half : ch;
      const uint32_t sign = ch >= half ? 0u : 0x80000000u;  // the low half takes minus the sine
#pragma unroll
      for (int k = 0; k < 4; k += 2) {
        const float4 x = *reinterpret_cast<const float4*>(cos_row + at + 2 * k);
        const uint4 y = *reinterpret_cast<const uint4*>(sin_row + at + 2 * k);
        c[k] = f2(x.x, x.y);
        c[k + 1] = f2(x.z, x.w);
        s[k] = f2(__uint_as_float(y.x ^ sign), __uint_as_float(y.y ^ sign));
        s[k + 1] = f2(__uint_as_float(y.z ^ sign), __uint_as_float(y.w ^ sign));
      }
    }
  }
};

// Rotates the row that a half-warp holds eight channels to a lane.  Every lane takes part in the exchange of halves;
// lanes behind `rotary` keep their channels.  EXACT (K): both products are rounded, not one fused into the sum, so that the
// stored K and with it the 4-bit codes are those of the formula's 32-bit steps.
template <typename T, bool INTER, bool EXACT>
__device__ __forceinline__ uint4 rotate8(const uint4& u, const Angles<INTER>& g, int ch, int rotary) {
  uint32_t w[4] = {u.x, u.y, u.z, u.w}, v[4] = {u.x, u.y, u.z, u.w};
  if (!INTER) {
    const int half = rotary >> 1, away = half >> 3;  // half is a multiple of 8
    const int lane = threadIdx.x & 31, peer = ch >= rotary ? lane : ch < half ? lane + away : lane - away;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = __shfl_sync(0xffffffffu, w[k], peer);
  }
  if (ch >= rotary) return u;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 x = Elem<T>::to_f2(w[k]), y = Elem<T>::to_f2(v[k]);
    float a, b;
    if (EXACT) {  // (the two-value instructions would be fused)
      float c0, c1, s0, s1;
      f2_split(g.c[k], c0, c1);
      f2_split(g.s[k], s0, s1);
      a = __fadd_rn(__fmul_rn(x.x, c0), __fmul_rn(INTER ? y.y : y.x, s0));
      b = __fadd_rn(__fmul_rn(x.y, c1), __fmul_rn(INTER ? y.x : y.y, s1));
    } else {
      const uint64_t xs = f2(x.x, x.y), ys = INTER ? f2(y.y, y.x) : f2(y.x, y.y);
      f2_split(fma2(xs, g.c[k], mul2(ys, g.s[k])), a, b);
    }
    w[k] = pack_pair(a, b, T());
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

// Block = (a page that gets new tokens, a run of KV heads with their query heads).  The block computes the sines of the
// page's positions once; then K (a warp takes a head, half a warp a token, so that the metadata is folded in
// registers), V (copied) and q (half a warp takes a token and walks the heads with its sines in registers; where the
// page has fewer new tokens, several half-warps share a token).  Rows move in 16-byte pieces, two (K, V) or four (q) of
// them in flight per lane and 32 warps on an SM: with twice as many in flight and three quarters of the warps one token
// for each of 256 sequences (32 KV heads) took 16.3 instead of 14.4 us, 20K tokens of prompts the same 108.
// Pages are found without a scan: sequence b owns the block slots from qo_indptr[b]/16 + 2b on, always as many as
// the pages its new tokens can touch; a slot beyond them has nothing to do.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kRopeWarps * 32, 4) rope_append_kernel(const RopeParams p) {
  __shared__ alignas(16) float cos_s[kPage][kD / 2], sin_s[kPage][kD / 2];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slot = blockIdx.x;
  // largest b with qo_indptr[b]/16 + 2b <= slot, 32 candidates a round; the last round's lanes hold the candidates' entries
  int lo = 0, hi = p.batch, step;  // answer in [lo, hi)
  int row0, n_new, pbase, n_pages, ll;
  do {
    step = (hi - lo + 31) >> 5;
    const int b = min(lo + lane * step, p.batch - 1);
    row0 = __ldg(p.qo_indptr + b);
    if (step == 1) {
      n_new = __ldg(p.qo_indptr + b + 1) - row0;
      pbase = __ldg(p.indptr + b);
      n_pages = __ldg(p.indptr + b + 1) - pbase;
      ll = __ldg(p.last_len + b);
    }
    const bool ok = lo + lane * step < hi && (row0 >> 4) + 2 * b <= slot;
    const int n = __popc(__ballot_sync(0xffffffffu, ok));  // lane 0's candidate always fits
    const int at = n > 0 ? n - 1 : 0;
    if (step == 1) {
      row0 = __shfl_sync(0xffffffffu, row0, at);
      n_new = __shfl_sync(0xffffffffu, n_new, at);
      pbase = __shfl_sync(0xffffffffu, pbase, at);
      n_pages = __shfl_sync(0xffffffffu, n_pages, at);
      ll = __shfl_sync(0xffffffffu, ll, at);
    }
    lo += at * step;
    hi = min(hi, lo + step);
  } while (step > 1);
  const int b = lo;
  if (n_new <= 0) return;
  const int len = (n_pages - 1) * kPage + ll;
  if (n_pages <= 0 || ll < 1 || ll > kPage || n_new > len || row0 < 0 || row0 + n_new > p.num_tokens) {
    if (threadIdx.x == 0) raise_flag(p.status, TWL_FLAG_BAD_INDEX);
    return;
  }
  const int start = len - n_new;  // cache position of the first new token
  // (before the sequence's first slot: rows before the first sequence's, which belong to none, or offsets that go back)
  const int nth = slot - ((row0 >> 4) + 2 * b);
  const int lp = (start >> 4) + nth;
  if (nth < 0 || lp >= n_pages) return;
  const int t0 = max(start, lp * kPage), t1 = min(len, lp * kPage + kPage);
  const int n = t1 - t0;                // new tokens of this page, 1..16
  const int row = row0 + (t0 - start);  // row of the first of them in q, k, v
  const int first_slot = t0 & (kPage - 1);
  const int phys = __ldg(p.indices + pbase + lp);
  const bool page_ok = phys >= 0 && phys < p.num_pages_total;
  if (!page_ok && threadIdx.x == 0) raise_flag(p.status, TWL_FLAG_BAD_INDEX);

  const int half = p.rotary >> 1;
  for (int i = threadIdx.x; i < n * half; i += kRopeWarps * 32) {
    const int tok = i / half, f = i - tok * half;
    double pos;
    if (p.positions == nullptr)
      pos = (double)(t0 + tok);
    else if (p.pos64)
      pos = (double)__ldg(static_cast<const long long*>(p.positions) + row + tok);
    else
      pos = (double)__ldg(static_cast<const int*>(p.positions) + row + tok);
    const double turns = pos * __ldg(p.freqs + f) * 0.15915494309189533577;  // 1 / (2 pi)
    double s, c;
    sincospi(2. * (turns - rint(turns)), &s, &c);
    cos_s[tok][f] = (float)(c * p.attn_scale);
    sin_s[tok][f] = (float)(s * p.attn_scale);
  }
  __syncthreads();

  const int G = p.Hq / p.Hkv;
  const int kv0 = blockIdx.y * p.heads_per_block, kv1 = min(p.Hkv, kv0 + p.heads_per_block);
  const int hw = lane >> 4, ch = 8 * (lane & 15);  // this lane's half of the warp, its channels
  Angles<INTER> ang;

  if (page_ok) {
    for (int task = warp; task < 2 * (kv1 - kv0); task += kRopeWarps) {
      const bool is_k = task < kv1 - kv0;
      const int head = kv0 + (is_k ? task : task - (kv1 - kv0));
      const size_t slab = (size_t)phys * p.Hkv + head;
      const int64_t ts = is_k ? p.k_ts : p.v_ts;
      const T* src = static_cast<const T*>(is_k ? p.k : p.v) + row * ts + head * (is_k ? p.k_hs : p.v_hs) + ch;
      T* dst = static_cast<T*>(is_k ? p.k_pages : p.v_pages) + slab * (kPage * kD) + first_slot * kD + ch;
      uint32_t mn[4], mx[4];
      const bool meta = is_k && p.kmeta != nullptr;
      T* mrow = static_cast<T*>(p.kmeta) + slab * 2 * kD + ch;
      if (meta && first_slot != 0) {  // the page holds older tokens: fold into what it says
        const uint4 a = *reinterpret_cast<const uint4*>(mrow), z = *reinterpret_cast<const uint4*>(mrow + kD);
        mn[0] = a.x; mn[1] = a.y; mn[2] = a.z; mn[3] = a.w;
        mx[0] = z.x; mx[1] = z.y; mx[2] = z.z; mx[3] = z.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mn[j] = pack_pair(INFINITY, INFINITY, T());
          mx[j] = pack_pair(-INFINITY, -INFINITY, T());
        }
      }
      for (int r0 = 0; r0 < n; r0 += 4) {
        uint4 u[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (r0 + 2 * i + hw < n) u[i] = load_row16(src + (r0 + 2 * i + hw) * ts, p.wide);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + 2 * i + hw;
          if (r0 + 2 * i >= n) break;  // (both halves)
          const bool mine = r < n;
          if (is_k) {
            if (p.rotary > 0) {
              ang.read(cos_s[mine ? r : 0], sin_s[mine ? r : 0], ch < p.rotary ? ch : 0, p.rotary);
              u[i] = rotate8<T, INTER, true>(u[i], ang, ch, p.rotary);
            }
            const uint32_t y[4] = {u[i].x, u[i].y, u[i].z, u[i].w};  // as the cache holds them
            if (mine) {
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                mn[j] = min_pair<T>(mn[j], y[j]);
                mx[j] = max_pair<T>(mx[j], y[j]);
              }
            }
            if (p.k4 != nullptr) {
              float scale, gn;
              const uint32_t word = codes8<T>(y, &scale, &gn);
              if (mine) {
                uint8_t* q4 = p.k4 + slab * kSlab;
                const int tok = first_slot + r;
                *reinterpret_cast<uint32_t*>(q4 + tok * 64 + (ch >> 1)) = word;
                if ((lane & 3) == 0)
                  *reinterpret_cast<__half2*>(q4 + kSlabCodes + tok * 16 + (ch >> 5) * 4) =
                      __halves2half2(__float2half_rn(scale), __float2half_rn(gn));
              }
            }
          }
          if (mine) *reinterpret_cast<uint4*>(dst + r * kD) = u[i];
        }
      }
      if (meta) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          mn[j] = min_pair<T>(mn[j], __shfl_xor_sync(0xffffffffu, mn[j], 16));
          mx[j] = max_pair<T>(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 16));
        }
        *reinterpret_cast<uint4*>(mrow + hw * kD) =
            hw ? make_uint4(mx[0], mx[1], mx[2], mx[3]) : make_uint4(mn[0], mn[1], mn[2], mn[3]);
      }
    }
  }

  // q: 16 half-warps over the tokens (rounded up to a power of two), the rest of them over the heads
  const int width = n > 8 ? 16 : n > 4 ? 8 : n > 2 ? 4 : n, unit = 2 * warp + hw;
  const int tok = unit & (width - 1), h_step = kPage / width, h_end = kv1 * G;
  const bool mine = tok < n;
  if (p.rotary > 0) ang.read(cos_s[mine ? tok : 0], sin_s[mine ? tok : 0], ch < p.rotary ? ch : 0, p.rotary);
  const T* src = static_cast<const T*>(p.q) + (int64_t)(row + (mine ? tok : 0)) * p.q_ts + ch;
  T* dst = static_cast<T*>(p.q_out) + (int64_t)(row + (mine ? tok : 0)) * p.o_ts + ch;
  const int h_off = unit / width, rounds = (h_end - kv0 * G + h_step - 1) / h_step;  // rounds: the same for every lane
  for (int i0 = 0; i0 < rounds; i0 += 4) {
    uint4 u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = kv0 * G + h_off + (i0 + i) * h_step;
      if (mine && h < h_end) u[i] = load_q16(src + h * p.q_hs, p.wide);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = kv0 * G + h_off + (i0 + i) * h_step;
      if (i0 + i >= rounds) break;
      if (p.rotary > 0) u[i] = rotate8<T, INTER, false>(u[i], ang, ch, p.rotary);
      if (mine && h < h_end) store_row16(dst + h * p.o_hs, u[i], p.wide);
    }
  }
}

// INT4 slabs as values: thread = eight channels of a token (one code word, one 16-byte store), block = four slabs that
// follow one another in the output (all four in flight; one slab a block: 14.8 instead of 12.7 us on 10.6K slabs, 57 MB).
struct DequantParams {
  const uint8_t* k4;
  const int32_t* page_ids;  // null: every page
  void* out;
  int32_t* status;
  int64_t items;
  int32_t Hkv, num_pages_total;
};
constexpr int kDequantSlabs = 4;
template <typename T>
__global__ void __launch_bounds__(256) dequantize_k_pages_kernel(const DequantParams p) {
  pdl_wait();
  const int64_t item0 = (int64_t)blockIdx.x * kDequantSlabs;
  const int tok = threadIdx.x >> 4, w = threadIdx.x & 15;
  uint32_t code[kDequantSlabs], sz[kDequantSlabs];
#pragma unroll
  for (int k = 0; k < kDequantSlabs; ++k) {
    const int64_t item = item0 + k;
    code[k] = sz[k] = 0;  // a page that is not there: zeros
    if (item >= p.items) continue;
    const int64_t i = item / p.Hkv;
    const int head = (int)(item - i * p.Hkv);
    const int64_t page = p.page_ids ? (int64_t)__ldg(p.page_ids + i) : i;
    if (page >= 0 && page < p.num_pages_total) {
      const uint8_t* slab = p.k4 + ((size_t)page * p.Hkv + head) * kSlab;
      code[k] = ldg_stream_u32(slab + tok * 64 + w * 4);
      sz[k] = ldg_stream_u32(slab + kSlabCodes + tok * 16 + (w >> 2) * 4);
    } else if (threadIdx.x == 0) {
      raise_flag(p.status, TWL_FLAG_BAD_INDEX);
    }
  }
#pragma unroll
  for (int k = 0; k < kDequantSlabs; ++k) {
    if (item0 + k >= p.items) break;
    const float2 f = Elem<__half>::to_f2(sz[k]);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)((code[k] >> (4 * j)) & 15u) * f.x + f.y;
    reinterpret_cast<uint4*>(static_cast<T*>(p.out) + (item0 + k) * (kPage * kD))[threadIdx.x] = pack8<T>(x);
  }
}

static inline bool strides_ok(const void* p, int64_t ts, int64_t hs) {
  return aligned(p, 8) && ts % 4 == 0 && hs % 4 == 0;
}

}  // namespace twl

extern "C" int twl_rope_append_kv(const void* q, const void* k, const void* v, int dtype, int64_t q_token_stride,
                                  int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                                  int64_t v_token_stride, int64_t v_head_stride, void* q_out,
                                  int64_t out_token_stride, int64_t out_head_stride, const void* positions,
                                  int32_t positions_are_64bit, const double* freqs, int32_t rotary_dim,
                                  int32_t interleaved, double attention_scale, void* k_pages, void* v_pages,
                                  uint8_t* k4_pages, void* kmeta, const int32_t* qo_indptr, const int32_t* kv_indptr,
                                  const int32_t* kv_indices, const int32_t* kv_last_page_len, int32_t num_tokens,
                                  int32_t batch, int32_t num_q_heads, int32_t num_kv_heads, int32_t num_pages_total,
                                  int32_t* status, void* stream) {
  using namespace twl;
  if (!q || !k || !v || !q_out || !k_pages || !v_pages || !qo_indptr || !kv_indptr || !kv_indices ||
      !kv_last_page_len)
    return TWL_ERR_BAD_ARG;
  if (num_tokens <= 0 || batch <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || num_pages_total <= 0 ||
      num_q_heads % num_kv_heads != 0)
    return TWL_ERR_BAD_ARG;
  if (rotary_dim < 0 || (rotary_dim > 0 && !freqs)) return TWL_ERR_BAD_ARG;
  if (rotary_dim > kD || rotary_dim % (interleaved ? 8 : 16) != 0) return TWL_ERR_UNSUPPORTED;
  // the strides of one token, and of one head, say nothing
  if (num_tokens == 1) q_token_stride = k_token_stride = v_token_stride = out_token_stride = 0;
  if (num_q_heads == 1) q_head_stride = out_head_stride = 0;
  if (num_kv_heads == 1) k_head_stride = v_head_stride = 0;
  if (!strides_ok(q, q_token_stride, q_head_stride) || !strides_ok(k, k_token_stride, k_head_stride) ||
      !strides_ok(v, v_token_stride, v_head_stride) || !strides_ok(q_out, out_token_stride, out_head_stride) ||
      !aligned(k_pages, 16) || !aligned(v_pages, 16) || (k4_pages && !aligned(k4_pages, 16)) ||
      (kmeta && !aligned(kmeta, 16)) || (freqs && !aligned(freqs, 8)))
    return TWL_ERR_MISALIGNED;
  if (dtype != TWL_F16 && dtype != TWL_BF16) return TWL_ERR_UNSUPPORTED;
  const int64_t slots = (int64_t)num_tokens / kPage + 2 * (int64_t)batch;
  if (slots > 0x7fffffffLL || num_kv_heads > 65535) return TWL_ERR_TOO_LARGE;
  RopeParams p;
  p.q = q; p.k = k; p.v = v; p.q_out = q_out;
  p.q_ts = q_token_stride; p.q_hs = q_head_stride; p.k_ts = k_token_stride; p.k_hs = k_head_stride;
  p.v_ts = v_token_stride; p.v_hs = v_head_stride; p.o_ts = out_token_stride; p.o_hs = out_head_stride;
  p.positions = positions; p.pos64 = positions_are_64bit; p.freqs = freqs; p.rotary = rotary_dim;
  p.attn_scale = attention_scale;
  p.k_pages = k_pages; p.v_pages = v_pages; p.k4 = k4_pages; p.kmeta = kmeta;
  p.qo_indptr = qo_indptr; p.indptr = kv_indptr; p.indices = kv_indices; p.last_len = kv_last_page_len;
  p.status = status; p.batch = batch; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.num_tokens = num_tokens;
  p.num_pages_total = num_pages_total;
  const auto wide = [](const void* x, int64_t ts, int64_t hs) { return aligned(x, 16) && ts % 8 == 0 && hs % 8 == 0; };
  p.wide = wide(q, q_token_stride, q_head_stride) && wide(k, k_token_stride, k_head_stride) &&
           wide(v, v_token_stride, v_head_stride) && wide(q_out, out_token_stride, out_head_stride);
  // One KV head (with its query heads) a block while there are fewer blocks than four per SM (decode: latency), then more,
  // up to eight: a block's look-up of its page and the sines are worth more rows (prompts of 20K tokens, 32/8 heads: 108 us,
  // with three times the blocks 160 us).
  const int64_t room = (int64_t)num_sms() * 4;
  int64_t heads = (slots * num_kv_heads + room - 1) / room;
  heads = heads < 1 ? 1 : heads > kRopeWarps ? kRopeWarps : heads;
  p.heads_per_block = (int32_t)(heads < num_kv_heads ? heads : num_kv_heads);
  const dim3 grid((unsigned)slots, (unsigned)((num_kv_heads + p.heads_per_block - 1) / p.heads_per_block));
  const dim3 block(kRopeWarps * 32);
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  auto* kernel = dtype == TWL_F16 ? (interleaved ? rope_append_kernel<__half, true> : rope_append_kernel<__half, false>)
                                  : (interleaved ? rope_append_kernel<__nv_bfloat16, true>
                                                 : rope_append_kernel<__nv_bfloat16, false>);
  TWL_CUDA_TRY(launch_chain(kernel, grid, block, 0, st, p));
  return TWL_OK;
}

extern "C" int twl_dequantize_k_pages(const uint8_t* k4_pages, const int32_t* page_ids, int64_t n_pages, void* out,
                                      int dtype, int32_t num_kv_heads, int32_t num_pages_total, int32_t* status,
                                      void* stream) {
  using namespace twl;
  if (!k4_pages || !out || n_pages <= 0 || num_kv_heads <= 0 || num_pages_total <= 0) return TWL_ERR_BAD_ARG;
  if (!page_ids && n_pages > num_pages_total) return TWL_ERR_BAD_ARG;
  if (!aligned(k4_pages, 16) || !aligned(out, 16)) return TWL_ERR_MISALIGNED;
  if (dtype != TWL_F16 && dtype != TWL_BF16) return TWL_ERR_UNSUPPORTED;
  const int64_t items = n_pages * num_kv_heads;
  if (items > 0x7fffffffLL) return TWL_ERR_TOO_LARGE;
  DequantParams p;
  p.k4 = k4_pages; p.page_ids = page_ids; p.out = out; p.status = status; p.Hkv = num_kv_heads; p.items = items;
  p.num_pages_total = num_pages_total;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  const dim3 grid((unsigned)((items + kDequantSlabs - 1) / kDequantSlabs));
  if (dtype == TWL_F16)
    TWL_CUDA_TRY(launch_chain(dequantize_k_pages_kernel<__half>, grid, dim3(256), 0, st, p));
  else
    TWL_CUDA_TRY(launch_chain(dequantize_k_pages_kernel<__nv_bfloat16>, grid, dim3(256), 0, st, p));
  return TWL_OK;
}
