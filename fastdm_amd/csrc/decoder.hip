// Row kernels of a decoder layer: residual addition + RMS norm with a bf16 or 8-bit output, and rotary positions at given places.
// HBM-bound like the rows kernels of elementwise.hip: 16-byte vectors per lane, every byte read and written once.
#include "common.h"
#include "launch.h"

namespace fdm {

// 16 bytes of bf16 at any (element) alignment: one global_load/store_dwordx4 either way, the hardware splits what straddles lines
typedef i32x4 i32x4_u __attribute__((aligned(2)));
typedef i32x2 i32x2_u __attribute__((aligned(1)));

// =============================================================================================== add_rms_norm
//   h = bf16(x + res)                 (the residual stream is kept in bf16; without res: h = x)
//   y = h * w * rsqrt(mean(h^2) + eps)            in fp32, ONE rounding at the output:
//   bf16(y)  |  e4m3(y / s), s = max|y| / 448  |  int8: rint(y / s) + z, s = (max y - min y) / 255, z = -128 - rint(min y / s)
// One block per row, the row in registers (from 32769 columns on six of the twelve forms spill 20 .. 172 bytes a thread): the block's one reduction carries the sum of squares and the extremes of h * w together (the
// extremes of y are theirs times the row's rsqrt: a product with one positive factor keeps the order, roundings included).
// Bound: HBM, 7 bytes per element (8 with a bf16 output).  16384 x 5120 to e4m3: 100 us = 5.8 TB/s (a copy of 300 MB: 5.4), to int8 the same; 4099 x 3584 to
// bf16: 18 us; one row of 4096: 2.6 us, the launch; 1023 x 1536 to int8: 5.0 - 6 us, one round of blocks that wait for memory (67 % of their waves' cycles).
// 2048 x 65536 to e4m3: 190 us = 4.9 TB/s, to int8 206 us; without a residual, where most of the spills are, 156 and 190 us for 3 bytes per element (bf16, 4 bytes: 108 us).
// Threads per row (fdm_add_rms_norm): 64 / 128 / 256 / 512 / 1024 threads take, 16384 rows to e4m3, for 512 columns 11.8 / 14.5 / 21 / 37 / 75 us, for 4096
// 87 / 85 / 83 / 83 / 117 us, for 5120 - / 105 / 103 / 105 / 131 us; 8192 rows of 8192 - / 88.4 / 86.2 / 84.6 / 86.4 us.  Up to 512 columns take 64 threads, the
// others 256 and more.  There is no form of 128: 520 to 1024 columns pay for idle lanes (16384 rows of 520 / 768 / 1024: 22 / 23 / 24 us, 2.7 / 3.9 / 4.9 TB/s).
struct NormArgs {
  bf16_t* out;
  uint8_t* q;
  float* scale;
  int32_t* azp;
  bf16_t* h;            // may be x or res
  const bf16_t* x;
  const bf16_t* res;
  const bf16_t* w;
  int64_t x_stride, res_stride, h_stride;
  int64_t row0;         // of this launch
  int width;
  float eps;
};

// the IEEE 754-2019 maximum and minimum, which keep a NaN (v_maximum3_f32, v_minimum3_f32), where fmaxf and fminf drop it
struct OpMaximum { __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_elementwise_maximum(a, b); } };
struct OpMinimum { __device__ __forceinline__ float operator()(float a, float b) const { return __builtin_elementwise_minimum(a, b); } };

// MODE 0: bf16, 1: e4m3, 2: int8.  EDGE: the width is no multiple of 8 or a row is not 16-byte aligned; the last vector may be short.
template <int THREADS, int NIT, int MODE, bool RES, bool EDGE>
__global__ void __launch_bounds__(THREADS) add_rms_norm_kernel(const NormArgs p) {
  constexpr int NW = THREADS / 64;
  __shared__ float red[3][NW];
  const int64_t row = p.row0 + blockIdx.x;
  const int tid = threadIdx.x;
  const int nvec = (p.width + 7) >> 3;
  const bf16_t* xr = p.x + row * p.x_stride;
  const bf16_t* rr = RES ? p.res + row * p.res_stride : nullptr;

  auto load = [&](const bf16_t* base, int v) -> i32x4 {
    if constexpr (!EDGE) return *reinterpret_cast<const i32x4*>(base + (size_t)v * 8);
    const int n = p.width - v * 8;
    if (n >= 8) return *reinterpret_cast<const i32x4_u*>(base + (size_t)v * 8);
    uint32_t e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = base[(size_t)v * 8 + (j < n ? j : 0)];      // past the end: the vector's first element again
    return i32x4{(int)(e[0] | e[1] << 16), (int)(e[2] | e[3] << 16), (int)(e[4] | e[5] << 16), (int)(e[6] | e[7] << 16)};
  };

  i32x4 xv[NIT], rv[NIT], wv[NIT];
#pragma unroll
  for (int i = 0; i < NIT; ++i) {       // all of a thread's loads go out together; past the row they read its last vector again
    const int v = min(tid + i * THREADS, nvec - 1);
    xv[i] = load(xr, v);
    if constexpr (RES) rv[i] = load(rr, v);
  }
#pragma unroll
  for (int i = 0; i < NIT; ++i) wv[i] = load(p.w, min(tid + i * THREADS, nvec - 1));

  float ss = 0.f, hi = MODE == 1 ? 0.f : -INFINITY, lo = INFINITY;
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const int v = tid + i * THREADS;
    if (v < nvec) {
      Vec8 a = unpack8(xv[i]);
      if constexpr (RES) {
        const Vec8 b = unpack8(rv[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) xv[i][j] = (int)pack2bf(a.v[2 * j] + b.v[2 * j], a.v[2 * j + 1] + b.v[2 * j + 1]);
        a = unpack8(xv[i]);
        bf16_t* hp = p.h + row * p.h_stride + (size_t)v * 8;
        if (!EDGE) *reinterpret_cast<i32x4*>(hp) = xv[i];
        else if (p.width - v * 8 >= 8) *reinterpret_cast<i32x4_u*>(hp) = xv[i];
        else
          for (int j = 0; j < p.width - v * 8; ++j) hp[j] = f2bf(a.v[j]);
      }
      const Vec8 g = unpack8(wv[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (!EDGE || v * 8 + j < p.width) ss = __builtin_fmaf(a.v[j], a.v[j], ss);
        if constexpr (MODE != 0) {
          const float t = a.v[j] * g.v[j];
          if constexpr (MODE == 1) hi = __builtin_elementwise_maximum(hi, fabsf(t));
          else {
            hi = __builtin_elementwise_maximum(hi, t);
            lo = __builtin_elementwise_minimum(lo, t);
          }
        }
      }
    }
  }
  ss = wave_reduce(ss, OpSum());
  if constexpr (MODE != 0) hi = wave_reduce(hi, OpMaximum());
  if constexpr (MODE == 2) lo = wave_reduce(lo, OpMinimum());
  if constexpr (NW > 1) {
    if ((tid & 63) == 0) {
      red[0][tid >> 6] = ss;
      if constexpr (MODE != 0) red[1][tid >> 6] = hi;
      if constexpr (MODE == 2) red[2][tid >> 6] = lo;
    }
    __syncthreads();
    ss = red[0][0];
#pragma unroll
    for (int k = 1; k < NW; ++k) ss += red[0][k];
    if constexpr (MODE != 0) {
      hi = red[1][0];
#pragma unroll
      for (int k = 1; k < NW; ++k) hi = __builtin_elementwise_maximum(hi, red[1][k]);
    }
    if constexpr (MODE == 2) {
      lo = red[2][0];
#pragma unroll
      for (int k = 1; k < NW; ++k) lo = __builtin_elementwise_minimum(lo, red[2][k]);
    }
  }
  const float rs = 1.0f / sqrtf(ss / (float)p.width + p.eps);

  // 8-bit forms: y / s as y * (1 / s).  A row of zeros gets the scale of max|y| = 1e-12 (the row quantisers' floor); int8 rows whose values
  // lie closer together than 1/16 of their size get the scale of that spread, so that z stays small (a step is then 2^-12 of the values).
  // A NaN in the row makes ss NaN, and with it rs; a NaN product (an infinity times a weight of 0, a NaN weight) makes the extremes NaN; an infinite
  // product makes them inf * 0.  Each way the scale, and so the row's e4m3 bytes, are NaN (comparisons with NaN leave it in place).
  float inv = 1.f, zero = 0.f;
  if constexpr (MODE == 1) {
    float amax = hi * rs;
    amax = amax < 1e-12f ? 1e-12f : amax;
    const float s = amax / 448.0f;
    inv = 1.0f / s;
    if (tid == 0) p.scale[row] = s;
  } else if constexpr (MODE == 2) {
    const float top = hi * rs, low = lo * rs;
    float range = top - low;
    const float least = fmaxf(fmaxf(fabsf(top), fabsf(low)) * 0.0625f, 1e-12f);
    range = range < least ? least : range;
    const float s = range / 255.0f;
    inv = 1.0f / s;
    zero = -128.0f - __builtin_rintf(low * inv);
    if (tid == 0) {
      p.scale[row] = s;
      p.azp[row] = (int32_t)zero;
    }
  }
#pragma unroll
  for (int i = 0; i < NIT; ++i) {
    const int v = tid + i * THREADS;
    if (v >= nvec) continue;
    const Vec8 a = unpack8(xv[i]), g = unpack8(wv[i]);
    Vec8 y;
#pragma unroll
    for (int j = 0; j < 8; ++j) y.v[j] = a.v[j] * g.v[j] * rs;
    const int n = p.width - v * 8;
    if constexpr (MODE == 0) {
      bf16_t* op = p.out + row * (int64_t)p.width + (size_t)v * 8;
      i32x4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (int)pack2bf(y.v[2 * j], y.v[2 * j + 1]);
      if (!EDGE) *reinterpret_cast<i32x4*>(op) = o;
      else if (n >= 8) *reinterpret_cast<i32x4_u*>(op) = o;
      else
        for (int j = 0; j < n; ++j) op[j] = f2bf(y.v[j]);
    } else {
      uint32_t b[2] = {0, 0};
#pragma unroll
      for (int j = 0; j < 8; j += 2) {
        uint32_t two;
        if constexpr (MODE == 1) {
          two = cvt2_e4m3<false>(y.v[j] * inv, y.v[j + 1] * inv);      // <= 448 (1 + 2^-22): rounds to 448
        } else {
          const int ia = (int)fmaxf(-128.f, fminf(__builtin_rintf(y.v[j] * inv + zero), 127.f));
          const int ib = (int)fmaxf(-128.f, fminf(__builtin_rintf(y.v[j + 1] * inv + zero), 127.f));
          two = ((uint32_t)ia & 0xffu) | (((uint32_t)ib & 0xffu) << 8);
        }
        b[j >> 2] |= two << (8 * (j & 3));
      }
      uint8_t* qp = p.q + row * (int64_t)p.width + (size_t)v * 8;
      if (!EDGE) *reinterpret_cast<i32x2*>(qp) = i32x2{(int)b[0], (int)b[1]};
      else if (n >= 8) *reinterpret_cast<i32x2_u*>(qp) = i32x2{(int)b[0], (int)b[1]};
      else
        for (int j = 0; j < n; ++j) qp[j] = (uint8_t)(b[j >> 2] >> (8 * (j & 3)));
    }
  }
}

template <int THREADS, int NIT>
static int launch_norm(NormArgs a, int64_t rows, int mode, bool edge, hipStream_t s) {
#define FDM_NORM(M, R, E) add_rms_norm_kernel<THREADS, NIT, M, R, E><<<dim3(count), dim3(THREADS), 0, s>>>(a)
#define FDM_NORM_M(M)                                                   \
  if (a.res) { if (edge) FDM_NORM(M, true, true); else FDM_NORM(M, true, false); } \
  else { if (edge) FDM_NORM(M, false, true); else FDM_NORM(M, false, false); }
  return launch_pieces(rows, THREADS, [&](int64_t first, unsigned count) -> int {
    a.row0 = first;
    switch (mode) {
      case 0: FDM_NORM_M(0); break;
      case 1: FDM_NORM_M(1); break;
      default: FDM_NORM_M(2); break;
    }
    FDM_CHECK_LAUNCH();
    return FDM_OK;
  });
#undef FDM_NORM_M
#undef FDM_NORM
}

// =============================================================================================== rotary positions
// Pair i of a head turns by p * theta_i at place p.  turns[i] = theta_i / (2 pi) in 64 bits: the angle's fraction of a full turn is taken in
// 64 bits (an angle of 10^6 rad has no fraction bits left in fp32's 24), then sine and cosine of that fraction in fp32.
// A block takes a few tokens: their sines and cosines once into LDS (a 64-bit product and about 40 fp32 instructions each, shared by all heads), then
// every head of q and k from there.
// Bound: HBM, 4 bytes per element.  16384 tokens, 40 heads x 128: 64 us = 5.25 TB/s (a copy: 5.4); 3 x 1371 tokens, 48 heads x 64, half of each head
// rotated: 10.1 us (13.6 with one item at a time and divisions by the items per token and head); 32 single tokens: 4.8 us, two memory latencies in a
// row (the places, then q and k behind the sines and cosines).
struct RopeAtArgs {
  const bf16_t* q;
  const bf16_t* k;
  bf16_t* qo;             // may be q / k (in place)
  bf16_t* ko;
  const double* turns;
  const void* pos;        // nullptr: 0 .. seq - 1
  int64_t pos_bs, pos_ts; // strides in elements
  int64_t q_bs, q_ts, k_bs, k_ts, qo_bs, qo_ts, ko_bs, ko_ts;
  int64_t tokens;
  int64_t block0;         // of this launch
  int seq, q_heads, k_heads, head, rot;
  int pos_bytes;          // 4 or 8
  int items;              // work items per token
  int per_head;           // ... per head
  int n_turn;             // ... of these: rotated ones (the others are copied)
  int tok_per_block;
  uint32_t items_magic, head_magic;      // ceil(2^32 / items), ceil(2^32 / per_head); 0 for 1
  float amplitude;
};

constexpr int ROPE_MAX_HALF = 128, ROPE_MAX_TOK = 16;

// V: elements per vector.  An item is, rotated: V low and V high elements (half layout) or V elements (interleaved: V / 2 pairs; V == 1: one pair, element by
// element); behind the rotated part: V elements copied as they are.
template <int V, bool NEOX>
struct RopeItem {
  static constexpr int W = !NEOX && V == 1 ? 2 : V;
  typedef uint16_t vec_t __attribute__((ext_vector_type(V == 1 ? 2 : V)));
  uint16_t a[W], b[W];

  static __device__ __forceinline__ void get(uint16_t (&x)[W], const bf16_t* p, int n) {
    if constexpr (V == 1) {
      x[0] = p[0];
      if (W == 2 && n == 2) x[W - 1] = p[1];
    } else {
      const vec_t v = *reinterpret_cast<const vec_t*>(p);
#pragma unroll
      for (int j = 0; j < W; ++j) x[j] = v[j];
    }
  }
  static __device__ __forceinline__ void put(bf16_t* p, const uint16_t (&x)[W], int n) {
    if constexpr (V == 1) {
      p[0] = x[0];
      if (W == 2 && n == 2) p[1] = x[W - 1];
    } else {
      vec_t v;
#pragma unroll
      for (int j = 0; j < W; ++j) v[j] = x[j];
      *reinterpret_cast<vec_t*>(p) = v;
    }
  }
};

template <int V, bool NEOX>
__global__ void __launch_bounds__(256) rope_at_kernel(const RopeAtArgs p) {
  typedef RopeItem<V, NEOX> Item;
  constexpr int U = 4;                           // items per thread and turn: their loads go out together
  extern __shared__ float2 turn_cs[];            // [tok_per_block][rot / 2]
  __shared__ int64_t at_q[ROPE_MAX_TOK], at_k[ROPE_MAX_TOK], at_qo[ROPE_MAX_TOK], at_ko[ROPE_MAX_TOK];
  const int half = p.rot >> 1;
  const int64_t tok0 = (p.block0 + blockIdx.x) * p.tok_per_block;
  const int ntok = (int)min((int64_t)p.tok_per_block, p.tokens - tok0);

  if (threadIdx.x < ntok) {
    const int64_t tok = tok0 + threadIdx.x, b = tok / p.seq, s = tok - b * p.seq;
    at_q[threadIdx.x] = b * p.q_bs + s * p.q_ts;
    at_k[threadIdx.x] = b * p.k_bs + s * p.k_ts;
    at_qo[threadIdx.x] = b * p.qo_bs + s * p.qo_ts;
    at_ko[threadIdx.x] = b * p.ko_bs + s * p.ko_ts;
  }
  for (int i = threadIdx.x; i < ntok * half; i += 256) {
    const int t = i / half, f = i - t * half;
    const int64_t tok = tok0 + t;
    const int64_t b = tok / p.seq, s = tok - b * p.seq;
    double place = (double)s;
    if (p.pos != nullptr) {
      const int64_t at = b * p.pos_bs + s * p.pos_ts;
      place = p.pos_bytes == 8 ? (double)static_cast<const int64_t*>(p.pos)[at] : (double)static_cast<const int32_t*>(p.pos)[at];
    }
    const double turn = place * p.turns[f];
    const float frac = (float)(turn - rint(turn));
    float sn, cs;
    sincospif(2.0f * frac, &sn, &cs);
    turn_cs[i] = make_float2(cs * p.amplitude, sn * p.amplitude);
  }
  __syncthreads();

  auto by = [](int i, uint32_t magic) { return magic ? (int)__umulhi((uint32_t)i, magic) : i; };
  const int total = ntok * p.items;
  for (int i0 = threadIdx.x; i0 < total; i0 += 256 * U) {
    Item x[U];
    const float2* cs[U];
    bf16_t* dst[U];
    int it[U];                                   // of the head: < n_turn rotated, else copied
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = min(i0 + u * 256, total - 1);
      const int t = p.tok_per_block == 1 ? 0 : by(i, p.items_magic);
      const int in_tok = i - t * p.items;
      int hd = by(in_tok, p.head_magic);
      it[u] = in_tok - hd * p.per_head;
      const bool is_k = hd >= p.q_heads;
      hd -= is_k ? p.q_heads : 0;
      const int at = it[u] < p.n_turn ? it[u] * Item::W : p.rot + (it[u] - p.n_turn) * V;
      const bf16_t* src = (is_k ? p.k + at_k[t] : p.q + at_q[t]) + (int64_t)hd * p.head + at;
      dst[u] = (is_k ? p.ko + at_ko[t] : p.qo + at_qo[t]) + (int64_t)hd * p.head + at;
      cs[u] = turn_cs + t * half + (NEOX ? at : at >> 1);
      const bool turned = it[u] < p.n_turn;
      Item::get(x[u].a, src, turned ? 2 : 1);
      if (NEOX) Item::get(x[u].b, src + (turned ? half : 0), 1);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (i0 + u * 256 >= total) break;
      if (it[u] < p.n_turn) {
        if constexpr (NEOX) {
#pragma unroll
          for (int j = 0; j < V; ++j) {
            const float a = bf2f(x[u].a[j]), c = bf2f(x[u].b[j]);
            const float2 r = cs[u][j];
            x[u].a[j] = f2bf(a * r.x - c * r.y);
            x[u].b[j] = f2bf(c * r.x + a * r.y);
          }
          Item::put(dst[u] + half, x[u].b, 1);
        } else {
#pragma unroll
          for (int j = 0; j < Item::W / 2; ++j) {
            const float a = bf2f(x[u].a[2 * j]), c = bf2f(x[u].a[2 * j + 1]);
            const float2 r = cs[u][j];
            x[u].a[2 * j] = f2bf(a * r.x - c * r.y);
            x[u].a[2 * j + 1] = f2bf(c * r.x + a * r.y);
          }
        }
        Item::put(dst[u], x[u].a, 2);
      } else {
        Item::put(dst[u], x[u].a, 1);
      }
    }
  }
}

}  // namespace fdm

using namespace fdm;

extern "C" {

int fdm_add_rms_norm(void* out_bf16, void* out_q, float* out_scale, int32_t* out_azp, int quant_mode, const void* x, const void* res,
                     const void* weight, void* h_out, int64_t rows, int64_t width, int64_t x_row_stride, int64_t res_row_stride,
                     int64_t h_row_stride, float eps, fdm_stream_t stream) {
  (void)hipGetLastError();  // drop any stale error of an earlier, unrelated runtime call: FDM_CHECK_LAUNCH must see only ours
  if (rows < 0 || width <= 0 || quant_mode < 0 || quant_mode > 2) return FDM_ERR_INVALID;
  if (rows == 0) return FDM_OK;
  if (!x || !weight || x_row_stride < width || (quant_mode == 0 && !out_bf16) || (quant_mode != 0 && (!out_q || !out_scale)) ||
      (quant_mode == 2 && !out_azp))
    return FDM_ERR_INVALID;
  if ((res == nullptr) != (h_out == nullptr)) return FDM_ERR_INVALID;
  if (res && (res_row_stride < width || h_row_stride < width)) return FDM_ERR_INVALID;
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(res) | reinterpret_cast<uintptr_t>(weight) |
                       reinterpret_cast<uintptr_t>(h_out) | reinterpret_cast<uintptr_t>(out_bf16);
  if (at & 1) return FDM_ERR_INVALID;
  if (width > 65536 || rows > 0x7fffffff) return FDM_ERR_UNSUPPORTED;
  const bool edge = (width & 7) || (at & 15) || (reinterpret_cast<uintptr_t>(out_q) & 7) || (x_row_stride & 7) ||
                    (res && ((res_row_stride & 7) || (h_row_stride & 7)));
  const NormArgs a{(bf16_t*)out_bf16, (uint8_t*)out_q, out_scale, out_azp, (bf16_t*)h_out, (const bf16_t*)x, (const bf16_t*)res,
                   (const bf16_t*)weight, x_row_stride, res_row_stride, h_row_stride, 0, (int)width, eps};
  hipStream_t s = to_stream(stream);
  const int nvec = (int)((width + 7) >> 3);
  if (nvec <= 64) return launch_norm<64, 1>(a, rows, quant_mode, edge, s);
  if (nvec <= 256) return launch_norm<256, 1>(a, rows, quant_mode, edge, s);
  if (nvec <= 512) return launch_norm<256, 2>(a, rows, quant_mode, edge, s);
  if (nvec <= 768) return launch_norm<256, 3>(a, rows, quant_mode, edge, s);
  if (nvec <= 1024) return launch_norm<512, 2>(a, rows, quant_mode, edge, s);
  if (nvec <= 2048) return launch_norm<512, 4>(a, rows, quant_mode, edge, s);
  if (nvec <= 4096) return launch_norm<1024, 4>(a, rows, quant_mode, edge, s);
  return launch_norm<1024, 8>(a, rows, quant_mode, edge, s);
}

int fdm_rope_positions(void* q_out, void* k_out, const void* q, const void* k, const void* turns, const void* positions, int position_bytes,
                       int64_t pos_batch_stride, int64_t pos_tok_stride, int64_t batch, int64_t seq, int q_heads, int k_heads, int head_size,
                       int rot_dim, int64_t q_batch_stride, int64_t q_tok_stride, int64_t k_batch_stride, int64_t k_tok_stride,
                       int64_t qo_batch_stride, int64_t qo_tok_stride, int64_t ko_batch_stride, int64_t ko_tok_stride, float amplitude,
                       int is_neox, fdm_stream_t stream) {
  (void)hipGetLastError();  // drop any stale error of an earlier, unrelated runtime call: FDM_CHECK_LAUNCH must see only ours
  if (batch < 0 || seq < 0 || q_heads < 0 || k_heads < 0 || head_size <= 0 || rot_dim <= 0 || (rot_dim & 1) || rot_dim > head_size)
    return FDM_ERR_INVALID;
  if (batch == 0 || seq == 0 || (q_heads == 0 && k_heads == 0)) return FDM_OK;
  if (!turns || (reinterpret_cast<uintptr_t>(turns) & 7) || (q_heads && (!q || !q_out)) || (k_heads && (!k || !k_out))) return FDM_ERR_INVALID;
  if (positions && position_bytes != 4 && position_bytes != 8) return FDM_ERR_INVALID;
  if (positions && (reinterpret_cast<uintptr_t>(positions) & (position_bytes - 1))) return FDM_ERR_INVALID;
  if (rot_dim > 2 * ROPE_MAX_HALF || seq > 0x7fffffff || batch > 0x7fffffff || head_size > 1024 ||
      ((int64_t)q_heads + k_heads) * head_size > (1 << 22))
    return FDM_ERR_UNSUPPORTED;
  uintptr_t at = 0;
  int64_t strides = 0;
  if (q_heads) {
    at |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out);
    strides |= q_batch_stride | q_tok_stride | qo_batch_stride | qo_tok_stride;
  }
  if (k_heads) {
    at |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out);
    strides |= k_batch_stride | k_tok_stride | ko_batch_stride | ko_tok_stride;
  }
  if (at & 1) return FDM_ERR_INVALID;
  const int half = rot_dim >> 1;
  // the widest vector that every address and every part of a head is a multiple of
  auto fits = [&](int v) {
    return (at & (2 * v - 1)) == 0 && (strides & (v - 1)) == 0 && head_size % v == 0 && (is_neox ? half : rot_dim) % v == 0 &&
           (head_size - rot_dim) % v == 0;
  };
  const int v = fits(8) ? 8 : fits(4) ? 4 : fits(2) ? 2 : 1;
  const bool same = (!q_heads || q == q_out) && (!k_heads || k == k_out);       // in place: nothing to copy
  RopeAtArgs a{};
  a.q = (const bf16_t*)q; a.k = (const bf16_t*)k; a.qo = (bf16_t*)q_out; a.ko = (bf16_t*)k_out;
  a.turns = (const double*)turns; a.pos = positions; a.pos_bs = pos_batch_stride; a.pos_ts = pos_tok_stride;
  a.q_bs = q_batch_stride; a.q_ts = q_tok_stride; a.k_bs = k_batch_stride; a.k_ts = k_tok_stride;
  a.qo_bs = qo_batch_stride; a.qo_ts = qo_tok_stride; a.ko_bs = ko_batch_stride; a.ko_ts = ko_tok_stride;
  a.tokens = batch * seq; a.seq = (int)seq; a.q_heads = q_heads; a.k_heads = k_heads; a.head = head_size; a.rot = rot_dim;
  a.pos_bytes = position_bytes; a.amplitude = amplitude;
  a.n_turn = is_neox ? half / v : rot_dim / (v == 1 ? 2 : v);
  a.per_head = a.n_turn + (same ? 0 : (head_size - rot_dim) / v);
  a.items = (q_heads + k_heads) * a.per_head;
  int tok = 1024 / a.items;
  tok = tok < 1 ? 1 : tok > ROPE_MAX_TOK ? ROPE_MAX_TOK : tok;
  a.tok_per_block = tok;
  // i / d as the high word of i * ceil(2^32 / d), exact while i * d < 2^32: with several tokens i < 1024; within a token i < 2^22 and d <= 1024
  a.items_magic = a.items == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + a.items - 1) / a.items);
  a.head_magic = a.per_head == 1 ? 0 : (uint32_t)((((uint64_t)1 << 32) + a.per_head - 1) / a.per_head);
  const int64_t grid = (a.tokens + tok - 1) / tok;
  if (grid > 0x7fffffff) return FDM_ERR_UNSUPPORTED;
  const size_t lds = (size_t)tok * half * sizeof(float2);
  hipStream_t s = to_stream(stream);
#define FDM_ROPE_AT(V)                                                                              \
  if (is_neox) rope_at_kernel<V, true><<<dim3(count), dim3(256), lds, s>>>(a);                      \
  else rope_at_kernel<V, false><<<dim3(count), dim3(256), lds, s>>>(a)
  return launch_pieces(grid, 256, [&](int64_t first, unsigned count) -> int {
    a.block0 = first;
    switch (v) {
      case 8: FDM_ROPE_AT(8); break;
      case 4: FDM_ROPE_AT(4); break;
      case 2: FDM_ROPE_AT(2); break;
      default: FDM_ROPE_AT(1); break;
    }
    FDM_CHECK_LAUNCH();
    return FDM_OK;
  });
#undef FDM_ROPE_AT
}

}  // extern "C"
