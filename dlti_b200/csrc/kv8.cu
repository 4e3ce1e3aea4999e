// A paged cache of keys and values in 8 bits: rows written (dlti_rope_cache8, dlti_acc_rope_cache8), attention of single tokens over it
// (dlti_paged_decode8), cached rows laid out in 16 bits (dlti_gather_rows8).
//
// Pages are [num_blocks, KV_heads, block_size, 128] e4m3: the tokens of one page and head are contiguous, so that attention reads whole
// lines and a page's scale belongs to one piece of memory. Scales are [num_blocks, KV_heads] fp32, powers of two: e4m3 is a floating type, a
// finer scale would not make its numbers more exact, and with a power of two a number leaves and enters without a second rounding.
#include "common.cuh"

#include <cstdio>
#include <initializer_list>
#include <type_traits>

namespace {

constexpr int HD = 128;
constexpr int E_LOW = -120, E_HIGH = 120;      // exponents of a page's scale: its reciprocal and 448 of it are normal fp32 numbers

__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127

// Smallest power of two s with largest <= 448 s, 448 = 1.75 * 2^8.
__device__ __forceinline__ float scale_for(float largest) {
  const uint32_t u = __float_as_uint(largest);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u);
  return pow2i(max(E_LOW, min(E_HIGH, e)));
}
// low byte of the result: a
__device__ __forceinline__ uint32_t e4m3x2(float a, float b) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(b), "f"(a));
  return r;
}
__device__ __forceinline__ uint32_t half2_of_e4m3x2(uint32_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)v));
  return r;
}
__device__ __forceinline__ float2 float2_of_e4m3x2(uint32_t v) {
  const uint32_t h = half2_of_e4m3x2(v);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}
template <typename T>
__device__ __forceinline__ void unpack8(const int4& v, float (&f)[8]) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float2 t = Cvt<T>::unpack2(u[i]);
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}
template <typename T>
__device__ __forceinline__ int4 pack8(const float (&f)[8]) {
  int4 v;
  uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) u[i] = Cvt<T>::pack2(f[2 * i], f[2 * i + 1]);
  return v;
}

// ---------------------------------------------------------------------------------------------
// Rows of a step. Sixteen lanes hold one head of one row, 8 elements each; the element that a rotation pairs with is 8 lanes away, and a warp
// has two rows at a time. A CTA takes a block of rows, whose angles it keeps in shared memory in the rows' type, and a share of the heads. Of
// keys and values a warp takes all rows of one page (consecutive rows with slots in it) for one head, so nobody else touches that head's piece of
// the page or its scale; a page that goes on behind the block is done by the CTA in whose block it begins. Up to 16 rows are in flight and stay in
// registers between finding the scale and rounding to it. Bound by a warp's loads and arithmetic taking turns: 6,506 rows of 48 heads 40 us, a call
// among others (182 MB, 4.5 TB/s; in place the same; the first form, a warp of rows at a time with angles from global memory, 64); a CTA more an SM, or
// one less, 47 and 50.
// ---------------------------------------------------------------------------------------------
struct Rows8 {
  const void* x;                 // [tokens, x_ld] in the rows' type, or the fp32 accumulator [tokens, (H + 2 KV) * 128], left zero
  void* out;                     // [tokens, out_ld]; may be x
  long long x_ld, out_ld;
  const int* pos;
  const float *cos_t, *sin_t;
  const long long* slots;
  uint8_t *k8, *v8;
  float *ks, *vs;
  int tokens, H, KV, bs, shift;  // shift: bs = 1 << shift, or -1
};

template <typename T, bool ACC>
__device__ __forceinline__ int4 take(const Rows8& p, long long t, int h, int l16) {
  if constexpr (ACC) {
    float4* a = reinterpret_cast<float4*>(const_cast<float*>(reinterpret_cast<const float*>(p.x)) + t * p.x_ld + h * HD + l16 * 8);
    const float4 a0 = a[0], a1 = a[1];
    a[0] = make_float4(0.f, 0.f, 0.f, 0.f);
    a[1] = make_float4(0.f, 0.f, 0.f, 0.f);
    const float r[8] = {a0.x, a0.y, a0.z, a0.w, a1.x, a1.y, a1.z, a1.w};
    return pack8<T>(r);
  } else {
    return *reinterpret_cast<const int4*>(reinterpret_cast<const T*>(p.x) + t * p.x_ld + h * HD + l16 * 8);
  }
}
// ROWS of a block, KEEP pairs of rows that a warp has in flight and keeps in registers. Decode steps: 1 and 1, a row is a page of its own.
template <int ROWS_, int KEEP_, int CTAS_>
struct RowsCfg {
  static constexpr int ROWS = ROWS_, KEEP = KEEP_, CTAS = CTAS_;
};
using DecodeRows = RowsCfg<1, 1, 4>;
using PromptRows = RowsCfg<16, 8, 3>;

// cosines and sines of a row, rounded to the rows' type as the 16-bit cache's ops round them
struct Angles {
  float c[8], s[8];
};
template <typename T>
__device__ __forceinline__ float4 rounded4(const float* f) {
  const float4 a = *reinterpret_cast<const float4*>(f);
  return make_float4(Cvt<T>::to_f(Cvt<T>::from_f(a.x)), Cvt<T>::to_f(Cvt<T>::from_f(a.y)), Cvt<T>::to_f(Cvt<T>::from_f(a.z)), Cvt<T>::to_f(Cvt<T>::from_f(a.w)));
}
// the larger of a pair and the magnitudes of eight elements; NaN is passed over
template <typename T>
__device__ __forceinline__ uint32_t larger(uint32_t top, const int4& v);
template <>
__device__ __forceinline__ uint32_t larger<__nv_bfloat16>(uint32_t top, const int4& v) {
  const uint32_t u[4] = {(uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = u[i] & 0x7fff7fffu;
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&top), *reinterpret_cast<const __nv_bfloat162*>(&a));
    top = *reinterpret_cast<const uint32_t*>(&m);
  }
  return top;
}
template <>
__device__ __forceinline__ uint32_t larger<__half>(uint32_t top, const int4& v) {
  const uint32_t u[4] = {(uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t a = u[i] & 0x7fff7fffu;
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&top), *reinterpret_cast<const __half2*>(&a));
    top = *reinterpret_cast<const uint32_t*>(&m);
  }
  return top;
}
// The lane's 8 elements rotated (all lanes of the warp call). Products of two 16-bit numbers are exact in fp32, so one rounding is left.
template <typename T>
__device__ __forceinline__ int4 turn(const int4& v, const Angles& an, bool low) {
  int4 w;
  w.x = __shfl_xor_sync(0xffffffffu, v.x, 8);
  w.y = __shfl_xor_sync(0xffffffffu, v.y, 8);
  w.z = __shfl_xor_sync(0xffffffffu, v.z, 8);
  w.w = __shfl_xor_sync(0xffffffffu, v.w, 8);
  if (low) w = make_int4(w.x ^ 0x80008000, w.y ^ 0x80008000, w.z ^ 0x80008000, w.w ^ 0x80008000);
  float a[8], b[8];
  unpack8<T>(v, a);
  unpack8<T>(w, b);
#pragma unroll
  for (int j = 0; j < 8; ++j) a[j] = a[j] * an.c[j] + b[j] * an.s[j];
  return pack8<T>(a);
}

template <typename T, bool ACC, typename C>
__global__ void __launch_bounds__(256, C::CTAS) rows8_kernel(const Rows8 p) {
  constexpr int block = C::ROWS, KEEP = C::KEEP, STAGED = block == 1 ? 1 : 2 * block;
  griddep_pass(p.tokens);
  __shared__ float4 s_angle[STAGED][32];                    // of a row: 16 pieces of cosines, 16 of sines
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, l16 = lane & 15, half = lane >> 4;
  const int first = blockIdx.x * block, last = min(p.tokens, first + block);
  const int staged = min(p.tokens - first, STAGED);
  const bool copy = ACC || p.out != p.x, low = l16 < 8;
  T* out = reinterpret_cast<T*>(p.out);
  const int heads = p.H + 2 * p.KV;
  int4 held[KEEP];
  // rows t, t + 1, ... of a run of n
  auto request = [&](int t, int n, int col) {
#pragma unroll
    for (int i = 0; i < KEEP; ++i) {
      held[i] = make_int4(0, 0, 0, 0);
      if (2 * i + half < n) held[i] = take<T, ACC>(p, t + 2 * i + half, col, l16);
    }
  };
  for (int i = threadIdx.x; i < staged * 32; i += 256) {
    const long long at = (long long)p.pos[first + (i >> 5)] * (HD / 2) + (i & 15) * 4;
    s_angle[i >> 5][i & 31] = rounded4<T>((i & 16 ? p.sin_t : p.cos_t) + at);
  }
  __syncthreads();
  auto staged_angles = [&](int t) {
    const float4* a = s_angle[t - first] + (l16 & 7) * 2;
    const float4 c0 = a[0], c1 = a[1], s0 = a[16], s1 = a[17];
    return Angles{{c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w}};
  };
  auto angles = [&](int t) {
    if (t - first < staged) return staged_angles(t);
    const long long at = (long long)p.pos[t] * (HD / 2) + (l16 & 7) * 8;
    const float4 c0 = rounded4<T>(p.cos_t + at), c1 = rounded4<T>(p.cos_t + at + 4), s0 = rounded4<T>(p.sin_t + at), s1 = rounded4<T>(p.sin_t + at + 4);
    return Angles{{c0.x, c0.y, c0.z, c0.w, c1.x, c1.y, c1.z, c1.w}, {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w}};
  };
  auto put_out = [&](int t, int col, const int4& v) { *reinterpret_cast<int4*>(out + t * p.out_ld + col * HD + l16 * 8) = v; };
  const int stride = gridDim.y * 8;
  int col = blockIdx.y * 8 + warp;
  // query heads: the angles of two rows serve two of them (reading them for every head took 29 us of 107 MB of queries, 22 without)
  constexpr int QH = KEEP >= 4 ? 2 : 1, QP = KEEP / QH;
  for (; col < p.H; col += QH * stride) {
    for (int at = first; at < last; at += 2 * QP) {
#pragma unroll
      for (int i = 0; i < QP; ++i)
#pragma unroll
        for (int j = 0; j < QH; ++j) {
          const int t = at + 2 * i + half;
          held[i * QH + j] = make_int4(0, 0, 0, 0);
          if (t < last && col + j * stride < p.H) held[i * QH + j] = take<T, ACC>(p, t, col + j * stride, l16);
        }
#pragma unroll
      for (int i = 0; i < QP; ++i) {
        if (at + 2 * i >= last) break;
        const int t = at + 2 * i + half;
        const Angles an = staged_angles(min(t, last - 1));
#pragma unroll
        for (int j = 0; j < QH; ++j)
          if (col + j * stride < p.H) {
            const int4 v = turn<T>(held[i * QH + j], an, low);
            if (t < last) put_out(t, col + j * stride, v);
          }
      }
    }
  }
  for (col = p.H + (blockIdx.y * 8 + warp + stride * heads - p.H) % stride; col < heads; col += stride) {
    const int hh = col - p.H;                               // key heads, then value heads
    const bool key = hh < p.KV;
    const int head = key ? hh : hh - p.KV;
    uint8_t* cache = key ? p.k8 : p.v8;
    float* scales = key ? p.ks : p.vs;
    const uint32_t bs = p.bs;
    auto page_in = [&](long long s) { return p.shift >= 0 ? (int)((uint32_t)s >> p.shift) : (int)((uint32_t)s / bs); };
    auto page_of = [&](int t) { const long long s = p.slots[t]; return s < 0 ? -1 : page_in(s); };
    for (int t = first; t < last;) {
      const int page = page_of(t);
      if (page >= 0 && t == first && t > 0 && page_of(t - 1) == page) {   // these rows belong to the block before
        while (t < last && page_of(t) == page) ++t;
        continue;
      }
      // the run [t, t + n) of rows of this page; a row without a slot is by itself. Lane i < 32 looks at row t + i
      int n = 1;
      bool fresh = false;
      uint32_t off = 0;                                     // place of row t + lane
      if (page >= 0) {
        for (int k = 0;; k += 32) {
          const int r = t + k + lane;
          const long long s = r < p.tokens ? p.slots[r] : -1;
          const bool in = s >= 0 && page_in(s) == page;
          const uint32_t place = (uint32_t)s - (uint32_t)page * bs;
          if (k == 0) off = place;
          const uint32_t out_of = ~__ballot_sync(0xffffffffu, in);
          const int more = out_of ? __ffs(out_of) - 1 : 32;
          fresh |= __any_sync(0xffffffffu, in && lane < more && place == 0);
          n = k + more;
          if (more < 32) break;
        }
      }
      const long long sc = (long long)page * p.KV + head;
      float old = pow2i(E_LOW);
      if (page >= 0 && !fresh) old = scales[sc];
      float largest = 0.f;
      uint32_t top = 0;
      for (int k = 0; k < n; k += 2 * KEEP) {
        request(t + k, n - k, col);
#pragma unroll
        for (int i = 0; i < KEEP; ++i) {
          if (k + 2 * i >= n) break;
          const int r = k + 2 * i + half;
          if (key) held[i] = turn<T>(held[i], angles(t + min(r, n - 1)), low);
          if (r < n && (key || copy)) put_out(t + r, col, held[i]);
          top = larger<T>(top, held[i]);                    // rows that are not there are 0
        }
      }
      if (page >= 0) {
        auto of_warp = [&]() {
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, o));
        };
        const float2 pair = Cvt<T>::unpack2(top);
        largest = fmaxf(pair.x, pair.y);
        of_warp();
        if (largest == INFINITY) {                          // infinities do not set the scale (nor does NaN): once more without them
          largest = 0.f;
          auto finite = [&](const int4& v) {
            float f[8];
            unpack8<T>(v, f);
#pragma unroll
            for (int j = 0; j < 8; ++j) largest = fmaxf(largest, fabsf(f[j]) < INFINITY ? fabsf(f[j]) : 0.f);
          };
          if (n <= 2 * KEEP) {
#pragma unroll
            for (int i = 0; i < KEEP; ++i)
              if (2 * i + half < n) finite(held[i]);
          } else {
            for (int r = half; r < n; r += 2) finite(*reinterpret_cast<const int4*>(out + (long long)(t + r) * p.out_ld + col * HD + l16 * 8));
          }
          of_warp();
        }
        uint8_t* piece = cache + sc * bs * HD;
        const float now = fmaxf(old, scale_for(largest));
        if (!fresh && now > old) {                          // what the page holds is rounded to the new scale
          const float ratio = old / now;
          for (int i = lane; i < (int)bs * (HD / 16); i += 32) {
            int4 v = reinterpret_cast<const int4*>(piece)[i];
            uint32_t* u = reinterpret_cast<uint32_t*>(&v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 a = float2_of_e4m3x2(u[j] & 0xffffu), b = float2_of_e4m3x2(u[j] >> 16);
              u[j] = e4m3x2(a.x * ratio, a.y * ratio) | e4m3x2(b.x * ratio, b.y * ratio) << 16;
            }
            reinterpret_cast<int4*>(piece)[i] = v;
          }
        }
        __syncwarp();
        if (lane == 0) scales[sc] = now;
        const float inv = 1.f / now;
        auto put = [&](uint32_t place, const int4& v) {
          float f[8];
          unpack8<T>(v, f);
          uint2 o;
          o.x = e4m3x2(f[0] * inv, f[1] * inv) | e4m3x2(f[2] * inv, f[3] * inv) << 16;
          o.y = e4m3x2(f[4] * inv, f[5] * inv) | e4m3x2(f[6] * inv, f[7] * inv) << 16;
          *reinterpret_cast<uint2*>(piece + place * HD + l16 * 8) = o;
        };
        if (n <= 2 * KEEP) {
#pragma unroll
          for (int i = 0; i < KEEP; ++i) {
            const uint32_t place = __shfl_sync(0xffffffffu, off, 2 * i + half);
            if (2 * i + half < n) put(place, held[i]);
          }
        } else {                                            // longer pages: this lane wrote (or, without a copy, read) these pieces itself
          for (int r = half; r < n; r += 2)
            put((uint32_t)p.slots[t + r] - (uint32_t)page * bs, *reinterpret_cast<const int4*>(out + (long long)(t + r) * p.out_ld + col * HD + l16 * 8));
        }
      }
      t += n;
    }
  }
}

template <typename T, bool ACC>
int rows8_t(const Rows8& p, cudaStream_t st) {
  const int heads = p.H + 2 * p.KV, eights = (heads + 7) / 8;
  // A row a block up to the size of most decode steps, whose rows have a page each: sixteen of them would take turns. us of a call alone (cold L2, 6 of
  // them the launch's, read to 2), a row a block / sixteen rows, 32 query and 8 key heads: decode rows 1 8/10, 8 10/27, 64 10/45, 256 14/45, 512 20/47;
  // rows of one prompt 8 12/10, 16 16/12, 128 16/12, 256 20/14, 512 23/14. Their number does not tell them apart: a prompt of up to 256 rows alone
  // takes 4 to 6 us more than it could, a step of more than 256 decode rows 27.
  if (p.tokens <= DLTI_PDL_MAX_ROWS) {
    DLTI_CUDA_CHECK(dlti_launch_pdl(p.tokens, rows8_kernel<T, ACC, DecodeRows>, dim3((unsigned)p.tokens, (unsigned)eights), dim3(256), 0, st, p));
  } else {
    const int blocks = (p.tokens + PromptRows::ROWS - 1) / PromptRows::ROWS;
    const long long ctas = (long long)blocks * eights;
    // Heads of a warp: few blocks need every SM, many serve their angles to more heads. us as above for 1 / 2 / 4 heads, 32 query and 32 key heads: 495
    // rows (372 CTAs) 20/29/41, 993 (756) 25/29/37, 1,989 (1,500) 39/41/42, 3,979 64/65/63, 7,959 117/111/106; 64 and 8 heads: 495 (310) 20/24/25, 993
    // (630) 25/22/25, 1,989 (1,250) 33/30/29, 3,979 (2,490) 51/47/45, 7,959 90/78/76.
    const int share = ctas <= 3 * 148 ? 1 : ctas <= 10 * 148 ? 2 : 4;
    DLTI_CUDA_CHECK(dlti_launch_pdl(p.tokens, rows8_kernel<T, ACC, PromptRows>, dim3((unsigned)blocks, (unsigned)((eights + share - 1) / share)), dim3(256),
                                    0, st, p));
  }
  dlti_count_launch();
  return 0;
}

// ---------------------------------------------------------------------------------------------
// Attention of single tokens. A CTA takes one split of one sequence's context for up to 8 query heads of one key/value head; its warps take
// tiles of 16 tokens in turn and never wait for one another before the end.
//
// Each warp has a ring of tiles of its own in shared memory, filled by cp.async (16 bytes a lane; the 16-byte pieces of a row change places with
// the row, so that neither the writes nor the two kinds of reads meet in a bank).
// Both products are m16n8k16 in fp16 with fp32 sums: e4m3 numbers are fp16 numbers. The order of the contraction is free as long as both
// operands agree, so a lane takes 32 consecutive numbers of a key (dimensions 32 t ...) as its share of the eight k-steps, and 16 consecutive
// numbers of four values (tokens 2t, 2t+1, 2t+8, 2t+9, dimensions 16 g ...) as the columns g of 16 n-tiles: bytes of neighbouring tokens are
// paired by a permute.
//   queries: scaled by a power of two per head so that their 16 bits are fp16 numbers exactly (down to 2^-39 of the head's largest);
//   weights p s_v: p <= 1 times the page's value scale over the largest seen so far, as fp16 hi + lo, rows g and g + 8 of the same product:
//   22 bits, absolutely 2^-40 of the largest.
// Bound by HBM: 128 rows of up to 2,048 tokens with 32 key heads 293 us in a loop over fresh inputs (1.62 GB, 5.5 TB/s; through registers instead of the
// ring 503), 4 rows of up to 30,011 with 8 key heads 49 us. Three CTAs an SM at 168 registers: four spill (the first case over one set of inputs, which
// stays warm in part: 370 instead of 257).
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ void mma_f16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t word(const int4& v, int i) { return (uint32_t)(i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w); }

constexpr int NW = 4;            // warps of a CTA
constexpr int RING = 3;          // tiles of a warp in flight or in use
constexpr float P_UNIT = 32768.f;
constexpr int MAX_PARTS = 16;

struct __align__(128) Stage {
  uint8_t k[16][128], v[16][128];
};
constexpr int PITCH = HD + 4;
union AttendSmem {
  Stage ring[NW][RING];
  float o[NW][8][PITCH];         // joining the warps
};

// both halves of a word as fp16 pairs
__device__ __forceinline__ void half4_of_e4m3x4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{.reg .b16 a, b; mov.b32 {a, b}, %2; cvt.rn.f16x2.e4m3x2 %0, a; cvt.rn.f16x2.e4m3x2 %1, b;}" : "=r"(lo), "=r"(hi) : "r"(w));
}
__device__ __forceinline__ int4 lds128(uint32_t a) {
  int4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ void cp16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}

struct Attend8 {
  const void* q;
  long long q_ld;
  const uint8_t *k8, *v8;
  const float *ks, *vs;
  const int *tables, *ctx;
  int max_blocks, bs, shift, G, KV, splits, parts;      // shift: bs = 1 << shift, or -1; parts: clusters of a context
  float scale_log2;
  float *part_o, *part_ml;       // [batch, heads, parts, 128], [..., 2]
  void* out;
  long long out_ld;
};

__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t remote(uint32_t a, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  return r;
}
__device__ __forceinline__ float remote_f(uint32_t a, int rank) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(remote(a, rank)) : "memory");
  return v;
}
__device__ __forceinline__ float2 remote_f2(uint32_t a, int rank) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(remote(a, rank)) : "memory");
  return v;
}
// factor of a part with maximum m and sum l among parts of maximum top; a part without tokens has m = -inf and l = 0
__device__ __forceinline__ float share(float m, float l, float top) { return m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2f(m - top); }
template <typename T>
__device__ __forceinline__ void finish(const Attend8& p, T* out, int b, int head, int d, float acc, float sum, float top, int part) {
  if (p.parts == 1) {
    out[b * p.out_ld + (long long)head * HD + d] = Cvt<T>::from_f(sum == 0.f ? 0.f : acc / sum);
  } else {
    const long long at = ((long long)b * (p.G * p.KV) + head) * p.parts + part;
    p.part_o[at * HD + d] = acc;
    if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(top, sum);
  }
}

// WHOLE: a tile lies in one page (block_size a multiple of 16). CLUSTER: the context is cut into splits
template <typename T, bool WHOLE, bool CLUSTER>
__global__ void __launch_bounds__(32 * NW, 3) attend8_kernel(const Attend8 p) {
  extern __shared__ __align__(128) unsigned char raw[];
  AttendSmem& sm = *reinterpret_cast<AttendSmem*>(raw);
  __shared__ float s_m[NW][8], s_l[NW][8];
  __shared__ float2 s_cml[8];
  __shared__ __align__(16) float s_scale[NW][RING][4];      // of a tile's halves: keys, values
  griddep_pass(gridDim.z);
  const int split = blockIdx.x, b = blockIdx.z;
  const int groups = (p.G + 7) / 8;
  const int kvh = blockIdx.y / groups, h0 = kvh * p.G + (blockIdx.y % groups) * 8;
  const int nh = min(8, (kvh + 1) * p.G - h0);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int ctx = min(p.ctx[b], p.max_blocks * p.bs);
  const int tiles = (ctx + 15) / 16;
  const int per = (tiles + p.splits - 1) / p.splits;
  const int end = min(tiles, (split + 1) * per);
  int tile = split * per + warp;

  // ---- the ring
  const int* table = p.tables + (long long)b * p.max_blocks;
  const uint32_t ring = smem_u32(&sm.ring[warp][0]), scales = smem_u32(&s_scale[warp][0][0]);
  // a lane copies 16 bytes of rows r8, r8 + 4 of both halves
  const int r8 = lane >> 3, c16 = (lane & 7) * 16;
  const uint8_t* kl = p.k8 + r8 * HD + c16;
  const uint8_t* vl = p.v8 + r8 * HD + c16;
  const uint32_t to0 = ring + r8 * 128 + (c16 ^ (r8 << 4)), to1 = ring + (r8 + 4) * 128 + (c16 ^ (r8 + 4) << 4);
  const bool sv = lane & 1;                                 // lanes 0 .. 3 bring the scales: keys, values of the halves
  const float* sl = sv ? p.vs : p.ks;
  const uint32_t sto = scales + (2 * sv + (lane >> 1)) * 4;
  auto page_at = [&](int tb) { return p.shift >= 0 ? tb >> p.shift : (int)((uint32_t)tb / (uint32_t)p.bs); };
  // pages of a tile's halves. A half that begins behind the end takes the first half's rows: it has no weight
  auto pages = [&](int at, int (&pg)[2]) {
    if (at < end) {
      pg[0] = table[page_at(at * 16)];
      if (!WHOLE) pg[1] = at * 16 + 8 < ctx ? table[page_at(at * 16 + 8)] : -1;
    }
  };
  auto fill = [&](int at, const int (&pg)[2], int slot) {
    if (at < end) {
      const uint32_t s = slot * (uint32_t)sizeof(Stage);
      uint32_t head[2], row[2];                             // page and head; row of the cache
      const int tb = at * 16;
      head[0] = (uint32_t)pg[0] * p.KV + kvh;
      row[0] = head[0] * p.bs + (tb - page_at(tb) * p.bs);
      head[1] = head[0];
      row[1] = row[0] + 8;
      if (!WHOLE) {
        if (pg[1] >= 0) {
          head[1] = (uint32_t)pg[1] * p.KV + kvh;
          row[1] = head[1] * p.bs + (tb + 8 - page_at(tb + 8) * p.bs);
        } else {
          row[1] = row[0];
        }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const unsigned long long at_row = (unsigned long long)row[h] * HD;
        cp16(to0 + s + h * 1024, kl + at_row);
        cp16(to1 + s + h * 1024, kl + at_row + 4 * HD);
        cp16(to0 + s + h * 1024 + 2048, vl + at_row);
        cp16(to1 + s + h * 1024 + 2048, vl + at_row + 4 * HD);
      }
      if (lane < 4) cp4(sto + slot * 16, sl + head[lane >> 1]);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  int pg[2];
#pragma unroll
  for (int i = 0; i < RING - 1; ++i) {
    pages(tile + i * NW, pg);
    fill(tile + i * NW, pg, i);
  }
  pages(tile + (RING - 1) * NW, pg);

  // ---- the queries
  uint32_t aq[8][2];
  float fq = 0.f;
  {
    float f[32], top = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float a[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (g < nh) unpack8<T>(*reinterpret_cast<const int4*>(reinterpret_cast<const T*>(p.q) + b * p.q_ld + (long long)(h0 + g) * HD + 32 * t + 8 * i), a);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[8 * i + j] = a[j];
        top = fmaxf(top, fabsf(a[j]));
      }
    }
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
    const int e = max(-100, min(127, (int)(__float_as_uint(top) >> 23) - 127));
    const float up = pow2i(14 - e);
    fq = p.scale_log2 * pow2i(e - 14);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      aq[s][0] = Cvt<__half>::pack2(f[4 * s] * up, f[4 * s + 1] * up);
      aq[s][1] = Cvt<__half>::pack2(f[4 * s + 2] * up, f[4 * s + 3] * up);
    }
  }

  float m = -INFINITY, l = 0.f, vref = pow2i(E_LOW), vinv = pow2i(-E_LOW);
  float o[16][4];
#pragma unroll
  for (int j = 0; j < 16; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;

  int slot = 0;
  auto step = [&](auto last) {
    constexpr bool edge = decltype(last)::value;            // some tokens of the tile are behind the end
    asm volatile("cp.async.wait_group %0;" ::"n"(RING - 2) : "memory");
    __syncwarp();                                           // this tile is there for every lane, and every lane has read the one before it
    const uint32_t kv = ring + slot * (uint32_t)sizeof(Stage);
    const float4 sc = *reinterpret_cast<const float4*>(&s_scale[warp][slot][0]);
    {
      const int ahead = slot == 0 ? RING - 1 : slot - 1;
      fill(tile + (RING - 1) * NW, pg, ahead);
      pages(tile + RING * NW, pg);
    }
    slot = slot == RING - 1 ? 0 : slot + 1;
    const float ksc[2] = {sc.x, sc.y}, vsc[2] = {sc.z, sc.w};
    float z[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};      // two chains of four products are shorter than one of eight
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int4 k = lds128(kv + (8 * h + g) * 128 + ((2 * t + i) ^ g) * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          uint32_t b0, b1;
          half4_of_e4m3x4(word(k, w), b0, b1);
          mma_f16(c[i], aq[4 * i + w][0], 0u, aq[4 * i + w][1], 0u, b0, b1);
        }
      }
      const float f = fq * ksc[h];
      z[h][0] = (c[0][0] + c[1][0]) * f;
      z[h][1] = (c[0][1] + c[1][1]) * f;
    }
    const int left = ctx - tile * 16 - 2 * t;               // tokens 2t + 8h + i are there while 8h + i < left
    if constexpr (edge) {                                   // tokens behind the end have no weight
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (8 * h + i >= left) z[h][i] = -INFINITY;
    }
    float mx = fmaxf(fmaxf(z[0][0], z[0][1]), fmaxf(z[1][0], z[1][1]));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
    const float vnew = fmaxf(vref, fmaxf(vsc[0], vsc[1]));
    if (__any_sync(0xffffffffu, mx > m) || vnew > vref) {
      const float mn = fmaxf(m, mx);
      const float a = m == -INFINITY ? (l == 0.f ? 0.f : 1.f) : ex2f(m - mn);
      l *= a;
      vinv = 1.f / vnew;
      const float ao = a * (vref * vinv);
      m = mn;
      vref = vnew;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        o[j][0] *= ao;
        o[j][1] *= ao;
        o[j][2] *= ao;
        o[j][3] *= ao;
      }
    }
    uint32_t hi[2], lo[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float p0 = ex2f(z[h][0] - m), p1 = ex2f(z[h][1] - m);
      if constexpr (edge) {                                 // m may be -inf itself
        if (8 * h >= left) p0 = 0.f;
        if (8 * h + 1 >= left) p1 = 0.f;
      }
      l += p0 + p1;
      const float f = vsc[h] * vinv * P_UNIT;               // powers of two
      p0 *= f;
      p1 *= f;
      const __half2 a = __floats2half2_rn(p0, p1);
      const float2 r = __half22float2(a);
      const __half2 c = __floats2half2_rn(p0 - r.x, p1 - r.y);
      hi[h] = *reinterpret_cast<const uint32_t*>(&a);
      lo[h] = *reinterpret_cast<const uint32_t*>(&c);
    }
    int4 v[2][2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        v[h][i] = lds128(kv + 16 * 128 + (8 * h + 2 * t + i) * 128 + (g ^ (2 * t + i)) * 16);
        if constexpr (edge)                                 // whatever a page holds behind the end is no value
          if (8 * h + i >= left) v[h][i] = make_int4(0, 0, 0, 0);
      }
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      uint32_t b[2][4];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        half4_of_e4m3x4(__byte_perm(word(v[h][0], w), word(v[h][1], w), 0x5140), b[h][0], b[h][1]);
        half4_of_e4m3x4(__byte_perm(word(v[h][0], w), word(v[h][1], w), 0x7362), b[h][2], b[h][3]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) mma_f16(o[4 * w + i], hi[0], lo[0], hi[1], lo[1], b[0][i], b[1][i]);
    }
    tile += NW;
  };
  const int whole = min(end, ctx / 16);
  while (tile < whole) step(std::false_type{});
  if (tile < end) step(std::true_type{});
  asm volatile("cp.async.wait_all;" ::: "memory");

  // join the warps: lane (g, t) holds dimensions 32 t .. 32 t + 31 of head g
  __syncthreads();                                          // the rings are done with
  auto& s_o = sm.o;
  l += __shfl_xor_sync(0xffffffffu, l, 1);
  l += __shfl_xor_sync(0xffffffffu, l, 2);
  {
    const float f = vref / P_UNIT;
    float* d = &s_o[warp][g][32 * t];
#pragma unroll
    for (int j = 0; j < 16; j += 4) {
      *reinterpret_cast<float4*>(d + j) = make_float4((o[j][0] + o[j][2]) * f, (o[j + 1][0] + o[j + 1][2]) * f, (o[j + 2][0] + o[j + 2][2]) * f,
                                                      (o[j + 3][0] + o[j + 3][2]) * f);
      *reinterpret_cast<float4*>(d + 16 + j) = make_float4((o[j][1] + o[j][3]) * f, (o[j + 1][1] + o[j + 1][3]) * f,
                                                           (o[j + 2][1] + o[j + 2][3]) * f, (o[j + 3][1] + o[j + 3][3]) * f);
    }
    if (t == 0) {
      s_m[warp][g] = m;
      s_l[warp][g] = l;
    }
  }
  __syncthreads();
  // Splits of one context are a cluster of up to 8 CTAs that join through distributed shared memory; with more, each cluster's sum goes to the
  // workspace.
  const uint32_t crank = CLUSTER ? cluster_rank() : 0, csize = CLUSTER ? cluster_size() : 1;
  const int d = threadIdx.x;
  for (int h = 0; h < nh; ++h) {
    float gm = s_m[0][h], gl = 0.f, acc = 0.f;
#pragma unroll
    for (int w = 1; w < NW; ++w) gm = fmaxf(gm, s_m[w][h]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float a = share(s_m[w][h], s_l[w][h], gm);
      gl += s_l[w][h] * a;
      acc += s_o[w][h][d] * a;
    }
    if (!CLUSTER) {
      finish(p, reinterpret_cast<T*>(p.out), b, h0 + h, d, acc, gl, gm, split);
    } else {
      s_o[0][h][d] = acc;                                   // nobody else reads column d
      if (d == 0) s_cml[h] = make_float2(gm, gl);
    }
  }
  if (!CLUSTER) return;
  cluster_barrier();
  for (int h = crank; h < nh; h += csize) {
    const uint32_t ml = smem_u32(&s_cml[h]), at = smem_u32(&s_o[0][h][d]);
    float2 x[8];
    float v[8], gm = -INFINITY, gl = 0.f, acc = 0.f;
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < (int)csize) {
        x[c] = remote_f2(ml, c);
        v[c] = remote_f(at, c);
      }
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < (int)csize) gm = fmaxf(gm, x[c].x);
#pragma unroll
    for (int c = 0; c < 8; ++c)
      if (c < (int)csize) {
        const float a = share(x[c].x, x[c].y, gm);
        gl += x[c].y * a;
        acc += v[c] * a;
      }
    finish(p, reinterpret_cast<T*>(p.out), b, h0 + h, d, acc, gl, gm, split / (int)csize);
  }
  cluster_barrier();                                        // shared memory stays until everyone has read it
}

template <typename T>
__global__ void __launch_bounds__(HD) join8_kernel(const float* __restrict__ part_o, const float* __restrict__ part_ml, int parts,
                                                   T* __restrict__ out, long long out_ld) {
  griddep_pass(gridDim.y);
  const int h = blockIdx.x, b = blockIdx.y, d = threadIdx.x;
  const long long at = ((long long)b * gridDim.x + h) * parts;
  float gm = -INFINITY, acc = 0.f, gl = 0.f;
  float v[MAX_PARTS];
  float2 x[MAX_PARTS];
#pragma unroll
  for (int s = 0; s < MAX_PARTS; ++s)
    if (s < parts) {
      x[s] = *reinterpret_cast<const float2*>(part_ml + (at + s) * 2);
      v[s] = part_o[(at + s) * HD + d];
      gm = fmaxf(gm, x[s].x);
    }
#pragma unroll
  for (int s = 0; s < MAX_PARTS; ++s)
    if (s < parts) {
      const float a = share(x[s].x, x[s].y, gm);
      gl += x[s].y * a;
      acc += v[s] * a;
    }
  out[b * out_ld + (long long)h * HD + d] = Cvt<T>::from_f(gl == 0.f ? 0.f : acc / gl);
}

template <typename T>
int attend8_t(const Attend8& p, int batch, cudaStream_t st) {
  const int H = p.G * p.KV;
  const bool whole = p.bs % 16 == 0;
  static bool set[64] = {};                       // the attribute is per device
  int dev = 0;
  DLTI_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev & 63]) {
    for (auto k : {attend8_kernel<T, true, true>, attend8_kernel<T, false, true>, attend8_kernel<T, true, false>, attend8_kernel<T, false, false>})
      DLTI_CUDA_CHECK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(AttendSmem)));
    set[dev & 63] = true;
  }
  const auto kernel = p.splits > 1 ? (whole ? attend8_kernel<T, true, true> : attend8_kernel<T, false, true>)
                                   : (whole ? attend8_kernel<T, true, false> : attend8_kernel<T, false, false>);
  DLTI_CUDA_CHECK(dlti_launch_pdl_cluster(batch, p.splits / p.parts, kernel, dim3(p.splits, p.KV * ((p.G + 7) / 8), batch),
                                          dim3(32 * NW), sizeof(AttendSmem), st, p));
  if (p.parts > 1)
    DLTI_CUDA_CHECK(dlti_launch_pdl(batch, join8_kernel<T>, dim3(H, batch), dim3(HD), 0, st, (const float*)p.part_o, (const float*)p.part_ml,
                                    p.parts, (T*)p.out, p.out_ld));
  dlti_count_launch(p.parts > 1 ? 2 : 1);
  return 0;
}

// ---------------------------------------------------------------------------------------------
// Cached rows in 16 bits: row rows[i] of ext gets the keys and values of slot slots[i] at its key and value columns. A warp takes 16 heads of one
// row, 8 numbers a lane and load, all eight loads before the first store. 326 MB in 56 us, 90 % of HBM's copy rate (a thread a piece with its own
// divisions: 81).
// ---------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(256) gather8_kernel(T* __restrict__ ext, long long ext_ld, const long long* __restrict__ rows,
                                                      const long long* __restrict__ slots, const uint8_t* __restrict__ k8,
                                                      const uint8_t* __restrict__ v8, const float* __restrict__ ks, const float* __restrict__ vs,
                                                      int n, int H, int KV, int bs) {
  const int lane = threadIdx.x & 31, c = (lane & 15) * 8;
  const int r = blockIdx.x * 8 + (threadIdx.x >> 5), h0 = blockIdx.y * 16 + (lane >> 4);
  if (r >= n) return;
  const uint32_t slot = (uint32_t)slots[r], page = slot / (uint32_t)bs, off = slot - page * bs;
  T* dst = ext + rows[r] * ext_ld + (long long)H * HD + c;
  uint2 v[8];
  float s[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int hh = h0 + 2 * i;
    if (hh < 2 * KV) {
      const bool key = hh < KV;
      const uint32_t sc = page * KV + (key ? hh : hh - KV);
      v[i] = *reinterpret_cast<const uint2*>((key ? k8 : v8) + ((unsigned long long)sc * bs + off) * HD + c);
      s[i] = (key ? ks : vs)[sc];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int hh = h0 + 2 * i;
    if (hh < 2 * KV) {
      const float2 a = float2_of_e4m3x2(v[i].x & 0xffffu), b = float2_of_e4m3x2(v[i].x >> 16), d = float2_of_e4m3x2(v[i].y & 0xffffu),
                   e = float2_of_e4m3x2(v[i].y >> 16);
      const float f[8] = {a.x * s[i], a.y * s[i], b.x * s[i], b.y * s[i], d.x * s[i], d.y * s[i], e.x * s[i], e.y * s[i]};
      *reinterpret_cast<int4*>(dst + hh * HD) = pack8<T>(f);
    }
  }
}

bool sizes_ok(const char* what, int H, int KV, int hd, int bs) {
  if (hd == HD && KV > 0 && H > 0 && H % KV == 0 && bs >= 8 && bs % 8 == 0) return true;
  char msg[200];
  std::snprintf(msg, sizeof msg, "%s: heads of 128, query heads a multiple of key/value heads, pages of a multiple of 8 tokens (got %d, %d / %d, %d)",
                what, hd, H, KV, bs);
  dlti_set_error(msg);
  return false;
}
// What the kernels read and write in pieces of `unit` bytes: addresses, and the pitch of rows in elements of two bytes.
bool begins_ok(const char* what, std::initializer_list<const void*> at, long long pitch, int unit = 16) {
  bool ok = pitch % 8 == 0;
  for (const void* p : at) ok &= reinterpret_cast<uintptr_t>(p) % unit == 0;
  if (ok) return true;
  char msg[160];
  std::snprintf(msg, sizeof msg, "%s: rows, pages, rotation tables and accumulators begin at multiples of %d bytes", what, unit);
  dlti_set_error(msg);
  return false;
}
// Rows that are written (b) are the rows they are made from (a), or share no memory with them: blocks of rows have no order among them. Pitches and
// widths in bytes.
bool apart_ok(const char* what, const void* a_, long long la, long long wa, const void* b_, long long lb, long long wb, long long rows) {
  const long long a = (long long)reinterpret_cast<uintptr_t>(a_), b = (long long)reinterpret_cast<uintptr_t>(b_);
  if (rows == 1) la = lb = 0;
  if ((a == b && la == lb) || b >= a + (rows - 1) * la + wa || a >= b + (rows - 1) * lb + wb) return true;
  if (la == lb && la > 0) {                       // columns side by side
    const long long d = ((b - a) % la + la) % la;
    if (d >= wa && d <= la - wb) return true;
  }
  char msg[120];
  std::snprintf(msg, sizeof msg, "%s: rows that are written overlap other rows that are read", what);
  dlti_set_error(msg);
  return false;
}

}  // namespace

// Rows x [tokens, x_ld] -> out [tokens, out_ld] (may be x): queries and keys rotated, values as they are; keys and values of the rows with
// slots[t] >= 0 also go to the 8-bit pages. Rows of one page are consecutive.
DLTI_API int dlti_rope_cache8(const void* x, long long x_ld, void* out, long long out_ld, const int* pos, const float* cos_t, const float* sin_t,
                              const long long* slots, void* k8, void* v8, float* ks, float* vs, long long tokens, int H, int KV, int hd, int bs,
                              int dtype, cudaStream_t st) {
  if (!sizes_ok("rope_cache8", H, KV, hd, bs)) return DLTI_ERR_UNSUPPORTED;
  if (tokens <= 0) return 0;
  if (tokens > 1 << 24) return DLTI_ERR_TOO_LARGE;
  const long long width = 2LL * (H + 2 * KV) * HD;
  if (!begins_ok("rope_cache8", {x, out, cos_t, sin_t, k8, v8}, x_ld | out_ld) ||
      !apart_ok("rope_cache8", x, 2 * x_ld, width, out, 2 * out_ld, width, tokens))
    return DLTI_ERR_BAD_ARG;
  const Rows8 p{x, out, x_ld, out_ld, pos, cos_t, sin_t, slots, (uint8_t*)k8, (uint8_t*)v8, ks, vs, (int)tokens, H, KV, bs, (bs & (bs - 1)) ? -1 : __builtin_ctz(bs)};
  if (dtype == DLTI_BF16) return rows8_t<__nv_bfloat16, false>(p, st);
  if (dtype == DLTI_FP16) return rows8_t<__half, false>(p, st);
  return DLTI_ERR_UNSUPPORTED;
}

// The same from the fp32 accumulator [tokens, (H + 2 KV) * 128] of the decode GEMM, which is left zero.
DLTI_API int dlti_acc_rope_cache8(float* acc, void* out, long long out_ld, const int* pos, const float* cos_t, const float* sin_t,
                                  const long long* slots, void* k8, void* v8, float* ks, float* vs, long long tokens, int H, int KV, int hd,
                                  int bs, int dtype, cudaStream_t st) {
  if (!sizes_ok("acc_rope_cache8", H, KV, hd, bs)) return DLTI_ERR_UNSUPPORTED;
  if (tokens <= 0) return 0;
  if (tokens > 1 << 24) return DLTI_ERR_TOO_LARGE;
  if (!begins_ok("acc_rope_cache8", {acc, out, cos_t, sin_t, k8, v8}, out_ld)) return DLTI_ERR_BAD_ARG;
  const Rows8 p{acc, out, (long long)(H + 2 * KV) * HD, out_ld, pos, cos_t, sin_t, slots, (uint8_t*)k8, (uint8_t*)v8, ks, vs, (int)tokens, H, KV, bs, (bs & (bs - 1)) ? -1 : __builtin_ctz(bs)};
  if (dtype == DLTI_BF16) return rows8_t<__nv_bfloat16, true>(p, st);
  if (dtype == DLTI_FP16) return rows8_t<__half, true>(p, st);
  return DLTI_ERR_UNSUPPORTED;
}

// floats of workspace that dlti_paged_decode8 needs: none for up to 8 splits, which are one cluster
DLTI_API long long dlti_paged_decode8_floats(int batch, int H, int splits) { return splits > 8 ? (long long)batch * H * ((splits + 7) / 8) * (HD + 2) : 0; }

// q [batch, q_ld] (head h at column h * 128) -> out [batch, out_ld]; contexts of 0 give zeros. splits: 1 .. 128, the same number in each of
// ceil(splits / 8) clusters.
DLTI_API int dlti_paged_decode8(const void* q, long long q_ld, const void* k8, const void* v8, const float* ks, const float* vs,
                                const int* tables, int max_blocks, const int* ctx, int batch, int bs, int H, int KV, int hd, float scale,
                                int splits, float* workspace, void* out, long long out_ld, int dtype, cudaStream_t st) {
  if (!sizes_ok("paged_decode8", H, KV, hd, bs)) return DLTI_ERR_UNSUPPORTED;
  if (batch <= 0) return 0;
  const int parts = (splits + 7) / 8;
  if (batch > 65535 || splits < 1 || parts > MAX_PARTS || splits % parts || (parts > 1 && !workspace)) return DLTI_ERR_BAD_ARG;
  if (!begins_ok("paged_decode8", {q, k8, v8}, q_ld) || !apart_ok("paged_decode8", q, 2 * q_ld, 2LL * H * HD, out, 2 * out_ld, 2LL * H * HD, batch))
    return DLTI_ERR_BAD_ARG;
  const Attend8 p{q, q_ld, (const uint8_t*)k8, (const uint8_t*)v8, ks, vs, tables, ctx, max_blocks, bs, (bs & (bs - 1)) ? -1 : __builtin_ctz(bs),
                  H / KV, KV, splits, parts, scale * 1.4426950408889634f, workspace, workspace + (long long)batch * H * parts * HD, out, out_ld};
  if (dtype == DLTI_BF16) return attend8_t<__nv_bfloat16>(p, batch, st);
  if (dtype == DLTI_FP16) return attend8_t<__half>(p, batch, st);
  return DLTI_ERR_UNSUPPORTED;
}

// ext [*, ext_ld]: columns H * 128 .. (H + 2 KV) * 128 of the rows rows[0 .. n) from the pages' slots slots[0 .. n).
DLTI_API int dlti_gather_rows8(void* ext, long long ext_ld, const long long* rows, const long long* slots, const void* k8, const void* v8,
                               const float* ks, const float* vs, long long n, int H, int KV, int hd, int bs, int dtype, cudaStream_t st) {
  if (!sizes_ok("gather_rows8", H, KV, hd, bs)) return DLTI_ERR_UNSUPPORTED;
  if (n <= 0) return 0;
  if (n > 1 << 30) return DLTI_ERR_TOO_LARGE;
  if (!begins_ok("gather_rows8", {ext}, ext_ld) || !begins_ok("gather_rows8", {k8, v8}, 0, 8)) return DLTI_ERR_BAD_ARG;
  const dim3 grid((unsigned)((n + 7) / 8), (unsigned)((2 * KV + 15) / 16));
  if (dtype == DLTI_BF16)
    gather8_kernel<__nv_bfloat16><<<grid, 256, 0, st>>>((__nv_bfloat16*)ext, ext_ld, rows, slots, (const uint8_t*)k8, (const uint8_t*)v8, ks, vs, (int)n, H, KV, bs);
  else if (dtype == DLTI_FP16)
    gather8_kernel<__half><<<grid, 256, 0, st>>>((__half*)ext, ext_ld, rows, slots, (const uint8_t*)k8, (const uint8_t*)v8, ks, vs, (int)n, H, KV, bs);
  else
    return DLTI_ERR_UNSUPPORTED;
  dlti_count_launch();
  return (int)cudaGetLastError();
}
