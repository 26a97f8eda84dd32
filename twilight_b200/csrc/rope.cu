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
// the rows while they are in registers.  The decode form (one token per sequence) is bound by the latency of a
// launch and of four dependent loads (sequence search, its table entries, the row, the old metadata).
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
template <typename T>
__device__ __forceinline__ void unpack8(const uint4& u, float (&x)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float2 f = Elem<T>::to_f2(w[k]);
    x[2 * k] = f.x;
    x[2 * k + 1] = f.y;
  }
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

// cos and sin for the eight channels of a lane (8 * (lane & 15) ..): channel j of a half turns with pair j, of
// interleaved channels 2k and 2k+1 with pair k.
template <bool INTER>
struct Angles {
  static constexpr int N = INTER ? 4 : 8;
  float c[N], s[N];
  __device__ __forceinline__ void read(const float* cos_row, const float* sin_row, int ch, int rotary) {
    const int at = INTER ? ch >> 1 : ch >= (rotary >> 1) ? ch - (rotary >> 1) : ch;
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const float4 x = *reinterpret_cast<const float4*>(cos_row + at + k);
      const float4 y = *reinterpret_cast<const float4*>(sin_row + at + k);
      c[k] = x.x; c[k + 1] = x.y; c[k + 2] = x.z; c[k + 3] = x.w;
      s[k] = y.x; s[k + 1] = y.y; s[k + 2] = y.z; s[k + 3] = y.w;
    }
  }
};

// Rotates the row that a half-warp holds eight channels to a lane.  Every lane takes part in the exchange of halves;
// lanes behind `rotary` keep their channels.  Both products are rounded (not fused into the sum), so that the stored K
// and with it the 4-bit codes do not depend on which of them a compiler would fuse.
template <typename T, bool INTER>
__device__ __forceinline__ uint4 rotate8(const uint4& u, const Angles<INTER>& g, int ch, int rotary) {
  float x[8];
  unpack8<T>(u, x);
  if (INTER) {
    if (ch >= rotary) return u;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float a = x[2 * k], b = x[2 * k + 1];
      x[2 * k] = __fsub_rn(__fmul_rn(a, g.c[k % Angles<INTER>::N]), __fmul_rn(b, g.s[k % Angles<INTER>::N]));
      x[2 * k + 1] = __fadd_rn(__fmul_rn(b, g.c[k % Angles<INTER>::N]), __fmul_rn(a, g.s[k % Angles<INTER>::N]));
    }
    return pack8<T>(x);
  }
  const int half = rotary >> 1, away = half >> 3;  // half is a multiple of 8
  const bool low = ch < half;
  const int lane = threadIdx.x & 31, peer = ch >= rotary ? lane : low ? lane + away : lane - away;
  uint4 v;
  v.x = __shfl_sync(0xffffffffu, u.x, peer);
  v.y = __shfl_sync(0xffffffffu, u.y, peer);
  v.z = __shfl_sync(0xffffffffu, u.z, peer);
  v.w = __shfl_sync(0xffffffffu, u.w, peer);
  if (ch >= rotary) return u;
  float y[8];
  unpack8<T>(v, y);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float sn = low ? -g.s[k % Angles<INTER>::N] : g.s[k % Angles<INTER>::N];
    x[k] = __fadd_rn(__fmul_rn(x[k], g.c[k % Angles<INTER>::N]), __fmul_rn(y[k], sn));
  }
  return pack8<T>(x);
}

// Block = (a page that gets new tokens, a run of KV heads with their query heads).  The block computes the sines of the
// page's positions once; then K (a warp takes a head, half a warp a token, so that the metadata is folded in
// registers), V (copied) and q (half a warp takes a token and walks the heads with its sines in registers; where the
// page has fewer new tokens, several half-warps share a token).  Rows move in 16-byte pieces, four to eight of
// them in flight per lane.
// Pages are found without a scan: sequence b owns the block slots from qo_indptr[b]/16 + 2b on, always as many as
// the pages its new tokens can touch; a slot beyond them has nothing to do.
template <typename T, bool INTER>
__global__ void __launch_bounds__(kRopeWarps * 32, 3) rope_append_kernel(const RopeParams p) {
  __shared__ alignas(16) float cos_s[kPage][kD / 2], sin_s[kPage][kD / 2];
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slot = blockIdx.x;
  // largest b with qo_indptr[b]/16 + 2b <= slot, 32 candidates a round
  int lo = 0, hi = p.batch;  // answer in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) >> 5;
    const int b = lo + lane * step;
    const bool ok = b < hi && (__ldg(p.qo_indptr + b) >> 4) + 2 * b <= slot;
    const int n = __popc(__ballot_sync(0xffffffffu, ok));  // lane 0's candidate always fits
    const int nlo = lo + (n > 0 ? n - 1 : 0) * step;
    hi = min(hi, nlo + step);
    lo = nlo;
  }
  const int b = lo;
  const int row0 = __ldg(p.qo_indptr + b), n_new = __ldg(p.qo_indptr + b + 1) - row0;
  const int pbase = __ldg(p.indptr + b), n_pages = __ldg(p.indptr + b + 1) - pbase;
  const int ll = __ldg(p.last_len + b);
  if (n_new <= 0) return;
  const int len = (n_pages - 1) * kPage + ll;
  if (n_pages <= 0 || ll < 1 || ll > kPage || n_new > len || row0 < 0 || row0 + n_new > p.num_tokens) {
    if (threadIdx.x == 0) raise_flag(p.status, TWL_FLAG_BAD_INDEX);
    return;
  }
  const int start = len - n_new;  // cache position of the first new token
  const int lp = (start >> 4) + (slot - ((row0 >> 4) + 2 * b));
  if (lp >= n_pages) return;
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
      float mn[8], mx[8];
      const bool meta = is_k && p.kmeta != nullptr;
      T* mrow = static_cast<T*>(p.kmeta) + slab * 2 * kD + ch;
      if (meta && first_slot != 0) {  // the page holds older tokens: fold into what it says
        unpack8<T>(*reinterpret_cast<const uint4*>(mrow), mn);
        unpack8<T>(*reinterpret_cast<const uint4*>(mrow + kD), mx);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          mn[j] = INFINITY;
          mx[j] = -INFINITY;
        }
      }
      for (int r0 = 0; r0 < n; r0 += 8) {
        uint4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (r0 + 2 * i + hw < n) u[i] = load_row16(src + (r0 + 2 * i + hw) * ts, p.wide);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = r0 + 2 * i + hw;
          if (r0 + 2 * i >= n) break;  // (both halves)
          const bool mine = r < n;
          if (is_k) {
            if (p.rotary > 0) {
              ang.read(cos_s[mine ? r : 0], sin_s[mine ? r : 0], ch < p.rotary ? ch : 0, p.rotary);
              u[i] = rotate8<T, INTER>(u[i], ang, ch, p.rotary);
            }
            float y[8];
            unpack8<T>(u[i], y);  // as the cache holds them
            if (mine) {
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                mn[j] = fminf(mn[j], y[j]);
                mx[j] = fmaxf(mx[j], y[j]);
              }
            }
            if (p.k4 != nullptr) {  // groups of 32 channels = four lanes; the arithmetic of quantize_k_pages
              float gx = y[0], gn = y[0];
#pragma unroll
              for (int j = 1; j < 8; ++j) {
                gx = fmaxf(gx, y[j]);
                gn = fminf(gn, y[j]);
              }
#pragma unroll
              for (int o = 2; o > 0; o >>= 1) {
                gx = fmaxf(gx, __shfl_xor_sync(0xffffffffu, gx, o));
                gn = fminf(gn, __shfl_xor_sync(0xffffffffu, gn, o));
              }
              const float range = fmaxf(rope_rnd<T>(gx - gn), rope_rnd<T>(1e-9f));
              const float scale = rope_rnd<T>(__fdiv_rn(range, 15.f));
              uint32_t word = 0;
#pragma unroll
              for (int j = 0; j < 8; ++j) {
                const float t = rope_rnd<T>(y[j] - gn);
                float w = (scale > 0.f) ? rope_rnd<T>(__fdiv_rn(t, scale)) : 0.f;
                w = fminf(fmaxf(rintf(w), 0.f), 15.f);
                word |= (uint32_t)(int)w << (4 * j);
              }
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
        for (int j = 0; j < 8; ++j) {
          mn[j] = fminf(mn[j], __shfl_xor_sync(0xffffffffu, mn[j], 16));
          mx[j] = fmaxf(mx[j], __shfl_xor_sync(0xffffffffu, mx[j], 16));
        }
        *reinterpret_cast<uint4*>(mrow + hw * kD) = pack8<T>(hw ? mx : mn);
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
      if (mine && h < h_end) u[i] = load_row16(src + h * p.q_hs, p.wide);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int h = kv0 * G + h_off + (i0 + i) * h_step;
      if (i0 + i >= rounds) break;
      if (p.rotary > 0) u[i] = rotate8<T, INTER>(u[i], ang, ch, p.rotary);
      if (mine && h < h_end) store_row16(dst + h * p.o_hs, u[i], p.wide);
    }
  }
}

// INT4 slabs as values: thread = eight channels of a token (one code word, one 16-byte store), block = a slab.
struct DequantParams {
  const uint8_t* k4;
  const int32_t* page_ids;  // null: every page
  void* out;
  int32_t* status;
  int32_t Hkv, num_pages_total;
};
template <typename T>
__global__ void __launch_bounds__(256) dequantize_k_pages_kernel(const DequantParams p) {
  pdl_wait();
  const int64_t item = blockIdx.x;
  const int64_t i = item / p.Hkv;
  const int head = (int)(item - i * p.Hkv);
  const int64_t page = p.page_ids ? (int64_t)__ldg(p.page_ids + i) : i;
  const int tok = threadIdx.x >> 4, w = threadIdx.x & 15;
  uint4 r = make_uint4(0, 0, 0, 0);
  if (page >= 0 && page < p.num_pages_total) {
    const uint8_t* slab = p.k4 + ((size_t)page * p.Hkv + head) * kSlab;
    const uint32_t code = ldg_stream_u32(slab + tok * 64 + w * 4);
    const uint32_t sz = ldg_stream_u32(slab + kSlabCodes + tok * 16 + (w >> 2) * 4);
    const float2 f = Elem<__half>::to_f2(sz);
    float x[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = (float)((code >> (4 * j)) & 15u) * f.x + f.y;
    r = pack8<T>(x);
  } else if (threadIdx.x == 0) {
    raise_flag(p.status, TWL_FLAG_BAD_INDEX);
  }
  reinterpret_cast<uint4*>(static_cast<T*>(p.out) + item * (kPage * kD))[threadIdx.x] = r;
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
  // One KV head (with its query heads) a block while there are fewer blocks than eight per SM (decode: latency), then
  // more, up to eight: the sines of a page are computed once per block.
  const int64_t room = (int64_t)num_sms() * 8;
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
  p.k4 = k4_pages; p.page_ids = page_ids; p.out = out; p.status = status; p.Hkv = num_kv_heads;
  p.num_pages_total = num_pages_total;
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TWL_F16)
    TWL_CUDA_TRY(launch_chain(dequantize_k_pages_kernel<__half>, dim3((unsigned)items), dim3(256), 0, st, p));
  else
    TWL_CUDA_TRY(launch_chain(dequantize_k_pages_kernel<__nv_bfloat16>, dim3((unsigned)items), dim3(256), 0, st, p));
  return TWL_OK;
}
