// A prompt's (or a decode step's) way into the paged cache in one pass: rotary positions on q and k, K and V
// rows into their pages, INT4 slabs and page (min, max) metadata; and the INT4 slabs read back as values.
//
// Rotation of a head's first R channels at position p, with the angle a_i = p * f_i of pair i < R/2:
//   x'_u = x_u cos a_i - x_v sin a_i,  x'_v = x_v cos a_i + x_u sin a_i,
// (u, v) = (i, i + R/2), or (2i, 2i + 1) when interleaved.  cos and sin carry attention_scale.  Angles are formed
// and reduced to a fraction of a turn in 64 bits (at position 10^5 a 32-bit product is off by 0.004 rad), the
// sine and cosine of the fraction are 32-bit; the rotation is 32-bit and rounded once to the model type.
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
  int32_t batch, Hq, Hkv, num_tokens, num_pages_total, rotary, interleaved, pos64, tasks_per_block;
  float attn_scale;
};

constexpr int kRopeWarps = 8;

template <typename T>
__device__ __forceinline__ float rope_rnd(float x) {
  return Elem<T>::to_f(Elem<T>::from_f(x));
}

template <typename T>
__device__ __forceinline__ uint2 pack4(const float (&x)[4]) {
  using T2 = typename Elem<T>::T2;
  T2 a, b;
  a.x = Elem<T>::from_f(x[0]);
  a.y = Elem<T>::from_f(x[1]);
  b.x = Elem<T>::from_f(x[2]);
  b.y = Elem<T>::from_f(x[3]);
  return make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}

// Rotates one row held four channels to a lane (channels 4*lane ..).  table: this token's R/2 {cos, sin}.
// Every lane of the warp takes part in the shuffles; lanes past R keep their channels.
__device__ __forceinline__ void rotate_row(float (&x)[4], const float2* table, int rotary, bool inter, int lane) {
  const int c = 4 * lane;
  if (inter) {
    if (c < rotary) {
      const float4 t = reinterpret_cast<const float4*>(table)[lane];  // {cos, sin} of pairs 2*lane, 2*lane+1
      const float a = x[0], b = x[2];
      x[0] = a * t.x - x[1] * t.y;
      x[1] = x[1] * t.x + a * t.y;
      x[2] = b * t.z - x[3] * t.w;
      x[3] = x[3] * t.z + b * t.w;
    }
  } else {
    const int half = rotary >> 1, hl = half >> 2;  // half is a multiple of 4
    const bool lowside = c < half, in = c < rotary;
    const int peer = lowside ? lane + hl : lane - hl;
    float y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = __shfl_sync(0xffffffffu, x[j], in ? peer : lane);
    if (in) {
      const float4* t = reinterpret_cast<const float4*>(table + (lowside ? c : c - half));
      const float4 t0 = t[0], t1 = t[1];
      const float cs[4] = {t0.x, t0.z, t1.x, t1.z};
      const float sn[4] = {t0.y, t0.w, t1.y, t1.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = lowside ? x[j] * cs[j] - y[j] * sn[j] : x[j] * cs[j] + y[j] * sn[j];
    }
  }
}

// Block = (a page that gets new tokens, a run of tasks); a task is one head's rows of that page: K of a KV head
// (rotated, written, quantised, folded into the metadata), V of a KV head (copied), or one query head (rotated).
// A warp takes a task whole, eight rows of 256 bytes in flight, so the metadata needs no exchange between warps;
// the block shares the sines of the page's 16 positions.
// Pages are found without a scan: sequence b owns the block slots from qo_indptr[b]/16 + 2b on, always as many as
// the pages its new tokens can touch; a slot beyond them has nothing to do.
template <typename T>
__global__ void __launch_bounds__(kRopeWarps * 32) rope_append_kernel(const RopeParams p) {
  __shared__ alignas(16) float2 table[kPage][kD / 2];
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
  const int n = t1 - t0;                 // new tokens of this page, 1..16
  const int row = row0 + (t0 - start);   // row of the first of them in q, k, v
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
    float s, c;
    sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
    table[tok][f] = make_float2(c * p.attn_scale, s * p.attn_scale);
  }
  __syncthreads();

  const int tasks = 2 * p.Hkv + p.Hq;
  const int task_end = min(tasks, (int)(blockIdx.y + 1) * p.tasks_per_block);
  for (int task = blockIdx.y * p.tasks_per_block + warp; task < task_end; task += kRopeWarps) {
    const bool is_k = task < p.Hkv, is_v = !is_k && task < 2 * p.Hkv;
    const int head = is_k ? task : is_v ? task - p.Hkv : task - 2 * p.Hkv;
    if ((is_k || is_v) && !page_ok) continue;
    const T* src;
    int64_t ts;
    T* dst;
    int64_t dts;
    const size_t slab = (size_t)max(phys, 0) * p.Hkv + head;
    if (is_k) {
      src = static_cast<const T*>(p.k) + row * p.k_ts + head * p.k_hs;
      ts = p.k_ts;
      dst = static_cast<T*>(p.k_pages) + slab * (kPage * kD) + first_slot * kD;
      dts = kD;
    } else if (is_v) {
      src = static_cast<const T*>(p.v) + row * p.v_ts + head * p.v_hs;
      ts = p.v_ts;
      dst = static_cast<T*>(p.v_pages) + slab * (kPage * kD) + first_slot * kD;
      dts = kD;
    } else {
      src = static_cast<const T*>(p.q) + row * p.q_ts + head * p.q_hs;
      ts = p.q_ts;
      dst = static_cast<T*>(p.q_out) + row * p.o_ts + head * p.o_hs;
      dts = p.o_ts;
    }
    float mn[4] = {INFINITY, INFINITY, INFINITY, INFINITY}, mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
    const bool meta = is_k && p.kmeta != nullptr;
    T* mrow = static_cast<T*>(p.kmeta) + slab * 2 * kD;
    if (meta && first_slot != 0) {  // the page holds older tokens: fold into what it says
      const uint2 a = reinterpret_cast<const uint2*>(mrow)[lane], z = reinterpret_cast<const uint2*>(mrow + kD)[lane];
      const float2 a0 = Elem<T>::to_f2(a.x), a1 = Elem<T>::to_f2(a.y);
      const float2 z0 = Elem<T>::to_f2(z.x), z1 = Elem<T>::to_f2(z.y);
      mn[0] = a0.x; mn[1] = a0.y; mn[2] = a1.x; mn[3] = a1.y;
      mx[0] = z0.x; mx[1] = z0.y; mx[2] = z1.x; mx[3] = z1.y;
    }
    for (int r0 = 0; r0 < n; r0 += 8) {
      uint2 u[8];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (r0 + i < n) u[i] = ldg_stream_u2(src + (r0 + i) * ts + 4 * lane);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = r0 + i;
        if (r >= n) break;
        if (!is_v) {
          const float2 a = Elem<T>::to_f2(u[i].x), c = Elem<T>::to_f2(u[i].y);
          float x[4] = {a.x, a.y, c.x, c.y};
          if (p.rotary > 0) rotate_row(x, table[r], p.rotary, p.interleaved != 0, lane);
          u[i] = pack4<T>(x);
          if (is_k) {
            const float2 y0 = Elem<T>::to_f2(u[i].x), y1 = Elem<T>::to_f2(u[i].y);  // as the cache holds them
            const float y[4] = {y0.x, y0.y, y1.x, y1.y};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              mn[j] = fminf(mn[j], y[j]);
              mx[j] = fmaxf(mx[j], y[j]);
            }
            if (p.k4 != nullptr) {  // groups of 32 channels = eight lanes; the arithmetic of quantize_k_pages
              float gx = fmaxf(fmaxf(y[0], y[1]), fmaxf(y[2], y[3]));
              float gn = fminf(fminf(y[0], y[1]), fminf(y[2], y[3]));
#pragma unroll
              for (int o = 4; o > 0; o >>= 1) {
                gx = fmaxf(gx, __shfl_xor_sync(0xffffffffu, gx, o));
                gn = fminf(gn, __shfl_xor_sync(0xffffffffu, gn, o));
              }
              const float range = fmaxf(rope_rnd<T>(gx - gn), rope_rnd<T>(1e-9f));
              const float scale = rope_rnd<T>(__fdiv_rn(range, 15.f));
              uint32_t word = 0;
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                const float t = rope_rnd<T>(y[j] - gn);
                float w = (scale > 0.f) ? rope_rnd<T>(__fdiv_rn(t, scale)) : 0.f;
                w = fminf(fmaxf(rintf(w), 0.f), 15.f);
                word |= (uint32_t)(int)w << (4 * j);
              }
              uint8_t* q4 = p.k4 + slab * kSlab;
              const int tok = first_slot + r;
              *reinterpret_cast<uint16_t*>(q4 + tok * 64 + 2 * lane) = (uint16_t)word;
              if ((lane & 7) == 0)
                *reinterpret_cast<__half2*>(q4 + kSlabCodes + tok * 16 + (lane >> 3) * 4) =
                    __halves2half2(__float2half_rn(scale), __float2half_rn(gn));
            }
          }
        }
        *reinterpret_cast<uint2*>(dst + r * dts + 4 * lane) = u[i];
      }
    }
    if (meta) {
      reinterpret_cast<uint2*>(mrow)[lane] = pack4<T>(mn);
      reinterpret_cast<uint2*>(mrow + kD)[lane] = pack4<T>(mx);
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
    float a[4], b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = (float)((code >> (4 * j)) & 15u) * f.x + f.y;
      b[j] = (float)((code >> (4 * j + 16)) & 15u) * f.x + f.y;
    }
    const uint2 x = pack4<T>(a), y = pack4<T>(b);
    r = make_uint4(x.x, x.y, y.x, y.y);
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
                                  int32_t interleaved, float attention_scale, void* k_pages, void* v_pages,
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
  if (rotary_dim > kD || rotary_dim % 8 != 0) return TWL_ERR_UNSUPPORTED;
  if (!strides_ok(q, q_token_stride, q_head_stride) || !strides_ok(k, k_token_stride, k_head_stride) ||
      !strides_ok(v, v_token_stride, v_head_stride) || !strides_ok(q_out, out_token_stride, out_head_stride) ||
      !aligned(k_pages, 16) || !aligned(v_pages, 16) || (k4_pages && !aligned(k4_pages, 16)) ||
      (kmeta && !aligned(kmeta, 16)) || (freqs && !aligned(freqs, 8)))
    return TWL_ERR_MISALIGNED;
  if (dtype != TWL_F16 && dtype != TWL_BF16) return TWL_ERR_UNSUPPORTED;
  const int64_t slots = (int64_t)num_tokens / kPage + 2 * (int64_t)batch;
  const int64_t tasks = 2 * (int64_t)num_kv_heads + num_q_heads;
  if (slots > 0x7fffffffLL || tasks > 65535LL * kRopeWarps) return TWL_ERR_TOO_LARGE;
  RopeParams p;
  p.q = q; p.k = k; p.v = v; p.q_out = q_out;
  p.q_ts = q_token_stride; p.q_hs = q_head_stride; p.k_ts = k_token_stride; p.k_hs = k_head_stride;
  p.v_ts = v_token_stride; p.v_hs = v_head_stride; p.o_ts = out_token_stride; p.o_hs = out_head_stride;
  p.positions = positions; p.pos64 = positions_are_64bit; p.freqs = freqs; p.rotary = rotary_dim;
  p.interleaved = interleaved; p.attn_scale = attention_scale;
  p.k_pages = k_pages; p.v_pages = v_pages; p.k4 = k4_pages; p.kmeta = kmeta;
  p.qo_indptr = qo_indptr; p.indptr = kv_indptr; p.indices = kv_indices; p.last_len = kv_last_page_len;
  p.status = status; p.batch = batch; p.Hq = num_q_heads; p.Hkv = num_kv_heads; p.num_tokens = num_tokens;
  p.num_pages_total = num_pages_total;
  // One task per warp while that leaves every block resident at once (decode: latency), two where there is
  // work for several waves (the sines of a page are then computed half as often).
  const int64_t fine = (tasks + kRopeWarps - 1) / kRopeWarps;
  p.tasks_per_block = slots * fine <= (int64_t)num_sms() * 6 ? kRopeWarps : 2 * kRopeWarps;
  const dim3 grid((unsigned)slots, (unsigned)((tasks + p.tasks_per_block - 1) / p.tasks_per_block));
  cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == TWL_F16)
    TWL_CUDA_TRY(launch_chain(rope_append_kernel<__half>, grid, dim3(kRopeWarps * 32), 0, st, p));
  else
    TWL_CUDA_TRY(launch_chain(rope_append_kernel<__nv_bfloat16>, grid, dim3(kRopeWarps * 32), 0, st, p));
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
