// Tokens from given random numbers (dlti_sample_given): temperature, top-k, top-p, min-p over rows of any length up to 2^18.
//
// A token has to be the one that exact arithmetic gives, also where a cut or the drawn number falls close to a border: with n kept tokens a
// relative error of d in the running sums moves about one draw in 1 / (2 n d), which for sums in 32 bits is one in a hundred over a whole
// vocabulary. So weights exp((x - max) / T) are taken in double precision and held as whole numbers of 2^-45: their sums are exact, do not depend
// on the order of atomics, and with up to 2^18 of them stay below 2^63.
//
// The kept tokens are a prefix of the order (logit descending, index ascending); each cut is found as the last token that it keeps, a 64-bit
// number of the logit's order-preserving bits and the index. A CTA takes a row and reads it several times, after the first time from L2:
//   1. the largest logit and the sum for the log-probability,
//   2. counts over 2048 bins of the logit's distance from the largest: the bin in which top-k ends, and bounds for the bin in which top-p ends,
//   3. the exact sums: of everything, above those bins, and of each of them; then the few tokens of the one bin are ranked by themselves,
//   4. the kept weights of every 256 tokens; of these the group, the lane and the token that the given number falls on.
// A bin of too many tokens (equal logits, or logits in a narrow range) is divided further by 11 bits of the logit at a time.
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int TH = 1024, PER = 8;                 // threads, and consecutive tokens of a thread in a chunk
constexpr int CHUNK = TH * PER;
constexpr int NB = 2 * TH, LIST = 1024;
constexpr int V_MAX = 1 << 18;
constexpr double UNIT = 35184372088832.0;         // 2^45
constexpr float RANGE = 32.f;                     // bins reach this far below the largest logit, in units of T: e^-32 < 2^-46

struct Work {
  uint32_t cnt[NB];
  u64 mass[NB];
  u64 lc[LIST], lw[LIST];
  u64 cw[V_MAX / (32 * PER)];
  u64 red[32];
  float fred[32];
  u64 u0, u1;
  int i0, i1;
  uint32_t n;
};

template <typename T>
struct Row {
  const T* p;
  int V;
  bool vec;
  // tokens base .. base + 7; those behind the end and NaN as -inf
  __device__ __forceinline__ void get(int base, float (&x)[PER]) const {
    if (vec && base + PER <= V) {
      if constexpr (sizeof(T) == 2) {
        const int4 v = *reinterpret_cast<const int4*>(p + base);
        const uint32_t u[4] = {(uint32_t)v.x, (uint32_t)v.y, (uint32_t)v.z, (uint32_t)v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Cvt<T>::unpack2(u[i]);
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        }
      } else {
        const float4 a = *reinterpret_cast<const float4*>(p + base), b = *reinterpret_cast<const float4*>(p + base + 4);
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = base + j < V ? Cvt<T>::to_f(p[base + j]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = x[j] != x[j] ? -INFINITY : x[j] + 0.f;      // -0 is 0
  }
};

__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ u64 place(float x, int i) { return (u64)key_of(x) << 32 | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ float below(float top, float x) { return x == top ? 0.f : top - x; }
__device__ __forceinline__ int bin_of(float d, float per_bin) { return (int)fminf(d * per_bin, (float)(NB - 1)); }
__device__ __forceinline__ u64 weight(float top, float x, double inv_t) {
  if (x == top) return (u64)UNIT;
  return x == -INFINITY || top == INFINITY ? 0 : __double2ull_rn(exp(((double)x - (double)top) * inv_t) * UNIT);
}

template <typename S>
__device__ __forceinline__ S warp_scan(S v) {                            // inclusive
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const S a = __shfl_up_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) >= o) v += a;
  }
  return v;
}
// Inclusive sum over the threads of the CTA; total: that of all.
template <typename S>
__device__ __forceinline__ S cta_scan(S v, S* red, S& total) {
  const int w = threadIdx.x >> 5;
  v = warp_scan(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 31) red[w] = v;
  __syncthreads();
  const S mine = warp_scan(red[threadIdx.x & 31]);
  const S before = __shfl_sync(0xffffffffu, mine, w ? w - 1 : 0);
  total = __shfl_sync(0xffffffffu, mine, 31);
  return v + (w ? before : S(0));
}
__device__ __forceinline__ u64 cta_sum(u64 v, u64* red) {
  u64 total;
  cta_scan<u64>(v, red, total);
  return total;
}

// The last token kept of a bin's tokens at or above `floor`: the r-th in order (MASS false), or the first at which the weights reach `want`.
template <bool MASS, typename T>
__device__ u64 last_kept(const Row<T>& row, Work& s, float top, float per_bin, double inv_t, int bin, u64 floor, uint32_t n, uint32_t r, double want) {
  const int tid = threadIdx.x;
  const int chunks = (row.V + CHUNK - 1) / CHUNK;
  int shift = 32;
  uint32_t prefix = 0;
  auto each = [&](auto&& body) {
    for (int c = 0; c < chunks; ++c) {
      const int base = c * CHUNK + tid * PER;
      float x[PER];
      row.get(base, x);
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const bool in = base + j < row.V && bin_of(below(top, x[j]), per_bin) == bin && place(x[j], base + j) >= floor &&
                        (shift == 32 || key_of(x[j]) >> shift == prefix);
        body(c, base + j, x[j], in);
      }
    }
  };
  while (n > LIST && shift > 0) {
    const int wide = min(11, shift), low = shift - wide;
    const uint32_t mask = (1u << wide) - 1;
    for (int i = tid; i < NB; i += TH) {
      s.cnt[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    each([&](int, int, float x, bool in) {
      if (in) {
        const uint32_t d = mask - (key_of(x) >> low & mask);
        atomicAdd(&s.cnt[d], 1u);
        if (MASS) atomicAdd(&s.mass[d], weight(top, x, inv_t));
      }
    });
    if (tid == 0) s.i0 = -1;
    __syncthreads();
    // the digit in which the cut lies: the last one that is there, if sums fall short of it
    const uint32_t c0 = s.cnt[2 * tid], c1 = s.cnt[2 * tid + 1];
    const u64 v0 = MASS ? s.mass[2 * tid] : c0, v1 = MASS ? s.mass[2 * tid + 1] : c1;
    u64 all;
    const u64 after = cta_scan<u64>(v0 + v1, s.red, all);
    const u64 b0 = after - v0 - v1, b1 = after - v1;
    const double goal = MASS ? want : (double)r;
    const double capped = fmin(goal, (double)all);
    if (c0 && (double)b0 < capped && capped <= (double)b1) { s.i0 = 2 * tid; s.u0 = b0; }
    if (c1 && (double)b1 < capped && capped <= (double)after) { s.i0 = 2 * tid + 1; s.u0 = b1; }
    __syncthreads();
    const bool none = s.i0 < 0;
    __syncthreads();
    if (none) {                                                        // no weight at all: everything is kept up to the last token there is
      if (c0) atomicMax(&s.i0, 2 * tid);
      if (c1) atomicMax(&s.i0, 2 * tid + 1);
      if (tid == 0) s.u0 = all;
      __syncthreads();
    }
    const int at = s.i0;
    n = s.cnt[at];
    if (MASS) want -= (double)s.u0;
    else r -= (uint32_t)s.u0;
    prefix = prefix << wide | (mask - (uint32_t)at);
    shift = low;
    __syncthreads();
  }
  if (n <= LIST) {
    if (tid == 0) {
      s.n = 0;
      s.u0 = ~0ull;
      s.u1 = ~0ull;
    }
    __syncthreads();
    each([&](int, int i, float x, bool in) {
      if (in) {
        const uint32_t k = atomicAdd(&s.n, 1u);
        if (k < LIST) {
          s.lc[k] = place(x, i);
          s.lw[k] = MASS ? weight(top, x, inv_t) : 1;
        }
      }
    });
    __syncthreads();
    for (uint32_t i = tid; i < n; i += TH) {
      const u64 mine = s.lc[i];
      u64 before = 0;
      uint32_t rank = 0;
      for (uint32_t j = 0; j < n; ++j)
        if (s.lc[j] > mine) {
          before += s.lw[j];
          ++rank;
        }
      if (MASS ? (double)before < want && want <= (double)(before + s.lw[i]) : rank == r - 1) s.u0 = mine;
      if (rank == n - 1) s.u1 = mine;                                  // sums that fall short of `want` keep all
    }
    __syncthreads();
    const u64 got = s.u0 != ~0ull ? s.u0 : s.u1;
    __syncthreads();
    return got;
  }
  // many tokens with one logit: the r-th by index
  if (MASS) {
    const uint32_t key = prefix;
    const float x = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
    const double w = (double)weight(top, x, inv_t);
    r = w > 0 ? (uint32_t)fmin(fmax(ceil(want / w), 1.0), (double)n) : n;
  }
  r = min(max(r, 1u), n);
  const int groups = chunks * 32;
  for (int c = 0; c < chunks; ++c) {
    const int base = c * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
    uint32_t k = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      k += base + j < row.V && key_of(x[j]) == prefix && place(x[j], base + j) >= floor;
    k = __reduce_add_sync(0xffffffffu, k);
    if ((tid & 31) == 0) s.cw[c * 32 + (tid >> 5)] = k;
  }
  __syncthreads();
  const u64 mine = tid < groups ? s.cw[tid] : 0;
  u64 all;
  const u64 upto = cta_scan<u64>(mine, s.red, all);
  if (upto - mine < r && r <= upto) {
    s.i0 = tid;
    s.u0 = upto - mine;
  }
  __syncthreads();
  const int g = s.i0;
  if ((tid >> 5) == (g & 31)) {
    const int base = (g >> 5) * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
    uint32_t k = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) k += base + j < row.V && key_of(x[j]) == prefix && place(x[j], base + j) >= floor;
    uint32_t at = (uint32_t)s.u0 + warp_scan(k) - k;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (base + j < row.V && key_of(x[j]) == prefix && place(x[j], base + j) >= floor)
        if (++at == r) s.u1 = place(x[j], base + j);
  }
  __syncthreads();
  const u64 got = s.u1;
  __syncthreads();
  return got;
}

template <typename T>
__global__ void __launch_bounds__(TH, 1) sample_given_kernel(const T* __restrict__ logits, long long ld, int V, const double* __restrict__ u,
                                                             const float* __restrict__ temperature, const int* __restrict__ top_k,
                                                             const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                             long long* __restrict__ out, float* __restrict__ out_logprob) {
  extern __shared__ __align__(16) unsigned char raw[];
  Work& s = *reinterpret_cast<Work*>(raw);
  const int b = blockIdx.x, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* p = logits + (long long)b * ld;
  const Row<T> row{p, V, (reinterpret_cast<uintptr_t>(p) & 15) == 0};
  const int chunks = (V + CHUNK - 1) / CHUNK;

  // the largest logit, at its lowest index
  u64 best = 0;
  for (int c = 0; c < chunks; ++c) {
    const int base = c * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (base + j < V) best = max(best, place(x[j], base + j));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.red[warp] = best;
  __syncthreads();
  best = s.red[lane];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  const int arg = (int)(0xffffffffu - (uint32_t)best);
  const uint32_t bk = (uint32_t)(best >> 32);
  const float top = __uint_as_float(bk & 0x80000000u ? bk & 0x7fffffffu : ~bk);
  __syncthreads();
  if (top == -INFINITY) {                                              // nothing is left: no token is more likely than another
    if (tid == 0) {
      out[b] = 0;
      if (out_logprob) out_logprob[b] = -INFINITY;
    }
    return;
  }
  const float t = temperature ? temperature[b] : 0.f;
  const bool drawn = t > 0.f;
  const int k = drawn && top_k ? top_k[b] : 0;
  const bool k_on = k > 0 && k < V;
  const float tp = drawn && top_p ? top_p[b] : 1.f;
  const bool p_on = tp < 1.f;
  const float tt = fmaxf(t, 1e-30f);                                   // the distances of a row in units of T stay finite
  const double inv_t = drawn ? 1.0 / (double)tt : 1.0;
  const float per_bin = (float)NB / (RANGE * tt);

  if (drawn && (k_on || p_on)) {
    for (int i = tid; i < NB; i += TH) {
      s.cnt[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
  }
  float sum1 = 0.f;
  if (out_logprob || (drawn && (k_on || p_on)))
    for (int c = 0; c < chunks; ++c) {
      const int base = c * CHUNK + tid * PER;
      float x[PER];
      row.get(base, x);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (base + j < V) {
          const float d = below(top, x[j]);
          if (out_logprob) sum1 += expf(-d);
          if (k_on || p_on) atomicAdd(&s.cnt[bin_of(d, per_bin)], 1u);
        }
    }
  float log_sum = 0.f;
  if (out_logprob) {
    double v = (double)sum1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) s.red[warp] = __double_as_longlong(v);
    __syncthreads();
    v = __longlong_as_double(s.red[lane]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    log_sum = (float)log(v);
  }
  if (!drawn) {
    if (tid == 0) {
      out[b] = arg;
      if (out_logprob) out_logprob[b] = -log_sum;
    }
    return;
  }
  __syncthreads();

  u64 floor = 0;
  if (k_on) {
    const uint32_t c0 = s.cnt[2 * tid], c1 = s.cnt[2 * tid + 1];
    u64 all;
    const u64 after = cta_scan<u64>((u64)c0 + c1, s.red, all);
    const u64 b0 = after - c0 - c1, b1 = after - c1;
    if (b0 < (u64)k && (u64)k <= b1) { s.i0 = 2 * tid; s.u0 = b0; }
    if (b1 < (u64)k && (u64)k <= after) { s.i0 = 2 * tid + 1; s.u0 = b1; }
    __syncthreads();
    const int bin = s.i0;
    const uint32_t before = (uint32_t)s.u0, n = s.cnt[bin];
    __syncthreads();
    floor = last_kept<false>(row, s, top, per_bin, inv_t, bin, 0ull, n, (uint32_t)k - before, 0.0);
    if (p_on) {
      // the counts of what is left for top-p (dividing a bin may have used the bins)
      for (int i = tid; i < NB; i += TH) {
        s.cnt[i] = 0;
        s.mass[i] = 0;
      }
      __syncthreads();
      for (int c = 0; c < chunks; ++c) {
        const int base = c * CHUNK + tid * PER;
        float x[PER];
        row.get(base, x);
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (base + j < V && place(x[j], base + j) >= floor) atomicAdd(&s.cnt[bin_of(below(top, x[j]), per_bin)], 1u);
      }
      __syncthreads();
    }
  }
  if (p_on) {
    // a bin's weight lies between its count times its least and its largest weight; so do the running sums, and with them the bins in which the
    // sum can reach top_p of the whole
    const uint32_t c0 = s.cnt[2 * tid], c1 = s.cnt[2 * tid + 1];
    const float step = RANGE / NB, w0 = __expf(-step * (2 * tid)), fall = __expf(-step);
    const float h0 = (float)c0 * w0 * 1.0001f, h1 = (float)c1 * w0 * fall * 1.0001f;
    // the last bin has no least weight
    const float l0 = (float)c0 * w0 * fall * 0.9999f, l1 = tid == TH - 1 ? 0.f : (float)c1 * w0 * fall * fall * 0.9999f;
    float most, least;
    const float ah = cta_scan<float>(h0 + h1, s.fred, most);
    const float al = cta_scan<float>(l0 + l1, s.fred, least);
    const float pp = fmaxf(tp, 0.f);
    const float lo_goal = pp * least * 0.9999f, hi_goal = pp * most * 1.0001f;
    if (tid == 0) {
      s.i0 = NB - 1;
      s.i1 = NB - 1;
    }
    __syncthreads();
    if (ah - h1 >= lo_goal) atomicMin(&s.i0, 2 * tid);
    else if (ah >= lo_goal) atomicMin(&s.i0, 2 * tid + 1);
    if (al - l1 >= hi_goal) atomicMin(&s.i1, 2 * tid);
    else if (al >= hi_goal) atomicMin(&s.i1, 2 * tid + 1);
    __syncthreads();
    const int from = s.i0, to = max(s.i1, from);
    u64 whole = 0, above = 0;
    for (int c = 0; c < chunks; ++c) {
      const int base = c * CHUNK + tid * PER;
      float x[PER];
      row.get(base, x);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (base + j < V && place(x[j], base + j) >= floor) {
          const u64 w = weight(top, x[j], inv_t);
          const int bin = bin_of(below(top, x[j]), per_bin);
          whole += w;
          if (bin < from) above += w;
          else if (bin <= to) atomicAdd(&s.mass[bin], w);
        }
    }
    whole = cta_sum(whole, s.red);
    above = cta_sum(above, s.red);
    const double goal = fmax((double)tp * (double)whole, 0.5) - (double)above;
    const u64 m0 = s.mass[2 * tid], m1 = s.mass[2 * tid + 1];
    u64 all;
    const u64 after = cta_scan<u64>(m0 + m1, s.red, all);
    const u64 b0 = after - m0 - m1, b1 = after - m1;
    if (tid == 0) s.i0 = -1;
    __syncthreads();
    if (m0 && (double)b0 < goal && goal <= (double)b1) { s.i0 = 2 * tid; s.u0 = b0; }
    if (m1 && (double)b1 < goal && goal <= (double)after) { s.i0 = 2 * tid + 1; s.u0 = b1; }
    __syncthreads();
    const int bin = s.i0;
    if (bin >= 0) {                                                    // else nothing is cut
      const double want = goal - (double)s.u0;
      const uint32_t n = s.cnt[bin];
      __syncthreads();
      floor = last_kept<true>(row, s, top, per_bin, inv_t, bin, floor, n, 0u, want);
    }
  }

  // the draw
  const double least_w = min_p ? fmin((double)min_p[b], 1.0) * UNIT : 0.0;
  auto kept = [&](float x, int i) -> u64 {
    if (i >= V || place(x, i) < floor) return 0;
    const u64 w = weight(top, x, inv_t);
    return (double)w >= least_w ? w : 0;
  };
  for (int c = 0; c < chunks; ++c) {
    const int base = c * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
    u64 w = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) w += kept(x[j], base + j);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    if (lane == 0) s.cw[c * 32 + warp] = w;
  }
  __syncthreads();
  const u64 mine = tid < chunks * 32 ? s.cw[tid] : 0;
  u64 all;
  const u64 upto = cta_scan<u64>(mine, s.red, all);
  // a number that rounding takes to the whole sum falls on the last token
  const double goal = fmin(fmax(u[b], 0.0) * (double)all, (double)all * (1.0 - 2.3e-16));
  if (tid == 0) s.i0 = 0;
  __syncthreads();
  if (mine && (double)(upto - mine) <= goal && goal < (double)upto) {
    s.i0 = tid;
    s.u0 = upto - mine;
  }
  __syncthreads();
  const int g = s.i0;
  if (warp == (g & 31)) {
    const int base = (g >> 5) * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
    u64 w[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      w[j] = kept(x[j], base + j);
      sum += w[j];
    }
    u64 at = s.u0 + warp_scan(sum) - sum;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      if (w[j] && (double)at <= goal && goal < (double)(at + w[j])) {
        out[b] = base + j;
        if (out_logprob) out_logprob[b] = -below(top, x[j]) - log_sum;
      }
      at += w[j];
    }
  }
}

template <typename T>
int launch(const void* logits, long long ld, int batch, int V, const double* u, const float* t, const int* k, const float* p, const float* mp,
           long long* out, float* lp, cudaStream_t st) {
  static bool set[64] = {};                       // the attribute is per device
  int dev = 0;
  DLTI_CUDA_CHECK(cudaGetDevice(&dev));
  if (!set[dev & 63]) {
    DLTI_CUDA_CHECK(cudaFuncSetAttribute(sample_given_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Work)));
    set[dev & 63] = true;
  }
  sample_given_kernel<T><<<batch, TH, sizeof(Work), st>>>((const T*)logits, ld, V, u, t, k, p, mp, out, lp);
  dlti_count_launch();
  return (int)cudaGetLastError();
}

}  // namespace

// logits [batch, V], row pitch ld (elements); u in [0, 1) and the settings of each row (NULL: greedy, off); out int64 [batch], out_logprob
// (optional): log p(token) at temperature 1.
DLTI_API int dlti_sample_given(const void* logits, long long ld, int batch, int V, const double* u, const float* temperature, const int* top_k,
                               const float* top_p, const float* min_p, long long* out, float* out_logprob, int dtype, cudaStream_t st) {
  if (batch <= 0) return 0;
  if (V < 1 || !u) return DLTI_ERR_BAD_ARG;
  if (V > V_MAX) {
    dlti_set_error("sample_given: at most 262144 logits a row");
    return DLTI_ERR_TOO_LARGE;
  }
  if (dtype == DLTI_BF16) return launch<__nv_bfloat16>(logits, ld, batch, V, u, temperature, top_k, top_p, min_p, out, out_logprob, st);
  if (dtype == DLTI_FP16) return launch<__half>(logits, ld, batch, V, u, temperature, top_k, top_p, min_p, out, out_logprob, st);
  if (dtype == DLTI_FP32) return launch<float>(logits, ld, batch, V, u, temperature, top_k, top_p, min_p, out, out_logprob, st);
  return DLTI_ERR_UNSUPPORTED;
}
