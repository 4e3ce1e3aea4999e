// Tokens from given random numbers (dlti_sample_given): temperature, top-k, top-p, min-p over rows of any length up to 2^18.
//
// A token has to be the one that exact arithmetic gives, also where a cut or the drawn number falls close to a border: with n kept tokens a
// relative error of d in the running sums moves about one draw in 1 / (2 n d), which for sums in 32 bits is one in a hundred over a whole
// vocabulary. So weights exp((x - max) / T) are taken in double precision and held as whole numbers of 2^-45: their sums are exact, do not depend
// on the order of atomics, and with up to 2^18 of them are at most 2^63, in 64 bits without a sign.
//
// The kept tokens are a prefix of the order (logit descending, index ascending); each cut is found as the last token that it keeps, a 64-bit
// number of the logit's order-preserving bits and the index. A CTA takes a row and reads it three times, after the first time from L2:
//   1. the largest logit,
//   2. the sum for the log-probability, and counts over 8192 bins of the distance from the largest: the bin in which top-k ends, and bounds for
//      the bins in which top-p can end,
//   3. the weights: tokens before these bins are kept whatever comes and go into sums of 256 tokens each; the tokens of these bins, some
//      thousand of a whole vocabulary, go to a list with their weights.
// The list then says where the cuts lie and is added to the sums; of these the group, the lane and the token follow that the number falls on.
// Where the list does not hold those bins' tokens (equal logits, or logits in a narrow range) a bin is divided further by 11 bits of the logit at a
// time, and the row read once more for each division, once for the ranks and once for the sums.
//
// Up to 64 long rows have a cluster of CTAs each. Every CTA reads its share of the row's chunks; largest, sums and bins are added up in each other's
// shared memory, the list and the sums of 256 tokens go to the first CTA's, which finds the cuts and the token by itself.
//
// Bound by arithmetic: 256 rows of 128,000 16-bit logits with top-p 188 us a call among others (weights by the library's exp, taken again for each cut
// and for the draw: 396). One row an SM, 148 of them, a call alone with a cold L2: 104 us, of which 6 are the launch's, 18 go to the largest logit (25 us
// is what greedy tokens take), 12 to the log-probability's sum, 16 to counts and bounds, 41 to the weights, 10 to the cut and the draw (by leaving out
// what follows each); the second 108 rows take as long again, 197 in all.
#include "common.cuh"

namespace {

typedef unsigned long long u64;

constexpr int TH = 512, WARPS = TH / 32, PER = 8; // threads, and consecutive tokens of a thread in a chunk
constexpr int CHUNK = TH * PER;
constexpr int NB = 8192, ND = 2048;               // bins of the distance from the largest; digits of 11 bits
constexpr int LIST = 512, WINDOW = 7168;
// Half of the range that is looked at first, relative to top-p's sum. The mean of a bin's bounds is off by at most 2^-9 of a token's weight, evenly
// to either side: by 3e-5 of the sum of a thousand tokens of one weight.
constexpr float NEAR = 3e-4f;
constexpr int MOST_CTAS = 8;                      // of a row
constexpr int V_MAX = 1 << 18, GROUPS = V_MAX / (32 * PER);
constexpr double UNIT = 35184372088832.0;         // 2^45
constexpr float RANGE = 32.f;                     // bins reach this far below the largest logit, in units of T: e^-32 < 2^-46

struct Work {
  uint32_t bins[NB];                              // tokens of each bin
  uint32_t cnt[ND];
  u64 mass[ND];
  union {
    struct {
      u64 lc[LIST], lw[LIST];                     // tokens of one bin, and their weights
    };
    struct {
      u64 wc[WINDOW], ww[WINDOW];                 // tokens of all bins in which a cut may lie
    };
  };
  u64 cw[GROUPS];                                 // kept weight of 256 tokens each
  u64 red[32];
  float fred[32];
  u64 u0, u1;
  int i0, i1, g0, g1;
  uint32_t n;
  u64 best, part[2];                              // of this CTA's share of a row, for the others of its cluster
  double sum1;
};

// ---- a row's CTAs: a cluster that reads each its share of the chunks. The first one keeps the list and the sums and does what follows alone.
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void cluster_barrier() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_u32(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ uint4 remote_u32x4(const uint32_t* p, int rank) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
__device__ __forceinline__ u64 remote_u64(const void* p, int rank) {
  u64 v;
  asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(at_rank(p, rank)) : "memory");
  return v;
}
// in the first CTA's memory
template <bool SHARED>
__device__ __forceinline__ uint32_t take_place(uint32_t* n) {
  if constexpr (!SHARED) return atomicAdd(n, 1u);
  uint32_t v;
  asm volatile("atom.shared::cluster.add.u32 %0, [%1], 1;" : "=r"(v) : "r"(at_rank(n, 0)) : "memory");
  return v;
}
template <bool SHARED>
__device__ __forceinline__ void store_first(u64* p, u64 v) {
  if constexpr (!SHARED) *p = v;
  else asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at_rank(p, 0)), "l"(v) : "memory");
}

template <typename T>
struct Row {
  const T* p;
  int V;
  bool vec;
  int rank, ctas;                                 // this CTA's share: chunks rank, rank + ctas, ...
  struct Raw {
    int4 v[sizeof(T) / 2];
  };
  __device__ __forceinline__ Raw fetch(int base) const {
    Raw r;
    if (vec && base + PER <= V) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.v[i] = reinterpret_cast<const int4*>(p + base)[i];
    }
    return r;
  }
  // tokens base .. base + 7; those behind the end and NaN as -inf
  __device__ __forceinline__ void open(const Raw& r, int base, float (&x)[PER]) const {
    if (vec && base + PER <= V) {
      if constexpr (sizeof(T) == 2) {
        const uint32_t u[4] = {(uint32_t)r.v[0].x, (uint32_t)r.v[0].y, (uint32_t)r.v[0].z, (uint32_t)r.v[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = Cvt<T>::unpack2(u[i]);
          x[2 * i] = f.x;
          x[2 * i + 1] = f.y;
        }
      } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          x[4 * i] = __int_as_float(r.v[i].x);
          x[4 * i + 1] = __int_as_float(r.v[i].y);
          x[4 * i + 2] = __int_as_float(r.v[i].z);
          x[4 * i + 3] = __int_as_float(r.v[i].w);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < PER; ++j) x[j] = base + j < V ? Cvt<T>::to_f(p[base + j]) : -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < PER; ++j) x[j] = fmaxf(x[j], -INFINITY);                     // NaN is -inf
  }
  __device__ __forceinline__ void get(int base, float (&x)[PER]) const { open(fetch(base), base, x); }
  // body(chunk, base, tokens) for the thread's tokens of the CTA's share; two chunks are on their way meanwhile
  template <typename F>
  __device__ __forceinline__ void each_chunk(F&& body) const {
    const int chunks = (V + CHUNK - 1) / CHUNK, stride = CHUNK * ctas;
    int base = (rank * TH + threadIdx.x) * PER;
    Raw a = fetch(base), n = fetch(base + stride);
    for (int c = rank; c < chunks; c += ctas, base += stride) {
      const Raw m = fetch(base + 2 * stride);
      float x[PER];
      open(a, base, x);
      body(c, base, x);
      a = n;
      n = m;
    }
  }
};

__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x + 0.f);                         // -0 is 0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ u64 place(float x, int i) { return (u64)key_of(x) << 32 | (0xffffffffu - (uint32_t)i); }
__device__ __forceinline__ float below(float top, float x) { return fmaxf(top - x, 0.f); }      // inf - inf is nothing
__device__ __forceinline__ float logit_of(u64 c) {
  const uint32_t k = (uint32_t)(c >> 32);
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ int bin_of(float d, float per_bin) { return (int)fminf(d * per_bin, (float)(NB - 1)); }
// A token's weight 2^(-(top - x) c), c = log2(e) / T, in units of 2^-45. 2^r on [-1/2, 1/2] is the polynomial of degree 9 through its values at the
// Chebyshev nodes: relatively 2^-45.6 off at most, and 2^45 of the largest logit's own. 15 operations in double precision, at half the rate of
// those in single, which is why a row's weights are taken once.
__constant__ double POLY[12] = {0x1.000000000003dp+0, 0x1.62e42fefa39f7p-1, 0x1.ebfbdff8149f2p-3, 0x1.c6b08d7044119p-5, 0x1.3b2ab72b175eep-7,
                                0x1.5d87fe908f88ap-10, 0x1.43088e257f341p-13, 0x1.ffcb76789860fp-17, 0x1.63ef969a64d3cp-20,
                                0x1.b6571de2f2351p-24, 6755399441055744.0, 4503599627370496.0};
constexpr float NOTHING = 47.f * NB / (RANGE * 1.4426950408889634f);   // in bins: weights below 2^-47
struct Weigh {
  float top, per_bin;
  double top64, c;
  __device__ __forceinline__ Weigh(float top_, float t)
      : top(top_), per_bin(fmaxf((float)NB / RANGE / t, 1e-44f)) /* of an infinite T: any but -inf is near */, top64(wide(top_)), c(1.4426950408889634074 / (double)t) {}
  // x in double by its bits (a conversion runs at a quarter of the rate): numbers below 2^-126 become others of that size, infinity 2^128
  static __device__ __forceinline__ double wide(float x) {
    const uint32_t u = __float_as_uint(x);
    return __hiloint2double((int)(((u & 0x7fffffffu) >> 3) + 0x38000000u | (u & 0x80000000u)), (int)(u << 29));
  }
  __device__ __forceinline__ u64 operator()(float x) const { return (*this)(x, below(top, x) * per_bin); }
  // at: the distance in bins
  __device__ __forceinline__ u64 operator()(float x, float at) const {
    const double z = (top64 - wide(x)) * c;
    const double y = z + POLY[10];                 // 1.5 * 2^52: the sum's low bits are the nearest whole number
    const double r = (y - POLY[10]) - z;
    double p = POLY[9];
#pragma unroll
    for (int i = 8; i >= 0; --i) p = fma(p, r, POLY[i]);
    p = __hiloint2double(__double2hiint(p) + ((45 - __double2loint(y)) << 20), __double2loint(p));
    const u64 w = (u64)__double_as_longlong(p + POLY[11]) & 0xfffffffffffffull;
    return at <= NOTHING ? w : 0;                  // nothing, too, where the distance is no number
  }
};

// A run of 2^shift bins among those that follow bin `base`.
struct Group {
  float top, per_bin;
  int base, shift, g;
  __device__ __forceinline__ int of(float x) const { return (bin_of(below(top, x), per_bin) - base) >> shift; }
  __device__ __forceinline__ bool has(float x) const { return of(x) == g; }
};

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
  const S mine = warp_scan((threadIdx.x & 31) < WARPS ? red[threadIdx.x & 31] : S(0));
  const S before = __shfl_sync(0xffffffffu, mine, w ? w - 1 : 0);
  total = __shfl_sync(0xffffffffu, mine, 31);
  return v + (w ? before : S(0));
}
__device__ __forceinline__ u64 cta_sum(u64 v, u64* red) {
  u64 total;
  cta_scan<u64>(v, red, total);
  return total;
}

// The i-th of n running sums in which `goal` lies (before < goal <= after, of values that are there) to s.i0, what comes before it to s.u0; s.i0 stays
// as it is if there is none. A thread looks at n / TH neighbours. Returns the whole sum.
template <int N, typename V>
__device__ __forceinline__ u64 find(Work& s, V&& value, double goal) {
  constexpr int E = N / TH;
  u64 v[E], sum = 0, all;
#pragma unroll
  for (int i = 0; i < E; ++i) sum += v[i] = value(E * threadIdx.x + i);
  u64 before = cta_scan<u64>(sum, s.red, all) - sum;
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (v[i] && (double)before < goal && goal <= (double)(before + v[i])) {
      s.i0 = E * threadIdx.x + i;
      s.u0 = before;
    }
    before += v[i];
  }
  __syncthreads();
  return all;
}
// Which of the counted digits (s.cnt, s.mass) the cut lies in: the last one that is there, if sums fall short of it. What lies before it is taken from r
// or `want`.
template <bool MASS>
__device__ __forceinline__ int digit(Work& s, uint32_t& r, double& want) {
  if (threadIdx.x == 0) s.i0 = -1;
  __syncthreads();
  const u64 all = find<ND>(s, [&](int i) { return MASS ? s.mass[i] : (u64)s.cnt[i]; }, MASS ? want : (double)r);
  const bool none = s.i0 < 0;
  __syncthreads();
  if (none) {                                                          // everything is kept, up to the last token there is
    for (int i = threadIdx.x; i < ND; i += TH)
      if (s.cnt[i]) atomicMax(&s.i0, i);
    if (threadIdx.x == 0) s.u0 = MASS ? all : all - 1;
    __syncthreads();
  }
  if (MASS) want -= (double)s.u0;
  else r -= (uint32_t)s.u0;
  return s.i0;
}

// The last token kept of a group's n tokens at or above `floor`: the r-th in order (MASS false), or the first at which the weights reach `want`.
template <bool MASS, typename T>
__device__ __noinline__ u64 last_kept(const Row<T> row, Work& s, const Weigh weigh, const Group group, u64 floor, uint32_t n, uint32_t r, double want) {
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
        const bool in = base + j < row.V && group.has(x[j]) && place(x[j], base + j) >= floor &&
                        (shift == 32 || key_of(x[j]) >> shift == prefix);
        body(c, base + j, x[j], in);
      }
    }
  };
  while (n > LIST && shift > 0) {
    const int wide = min(11, shift), low = shift - wide;
    const uint32_t mask = (1u << wide) - 1;
    for (int i = tid; i < ND; i += TH) {
      s.cnt[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    each([&](int, int, float x, bool in) {
      if (in) {
        const uint32_t d = mask - (key_of(x) >> low & mask);
        atomicAdd(&s.cnt[d], 1u);
        if (MASS) atomicAdd(&s.mass[d], weigh(x));
      }
    });
    __syncthreads();
    const int at = digit<MASS>(s, r, want);
    n = s.cnt[at];
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
          s.lw[k] = MASS ? weigh(x) : 1;
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
    const double w = (double)weigh(logit_of((u64)prefix << 32));
    r = w > 0 ? (uint32_t)fmin(fmax(ceil(want / w), 1.0), (double)n) : n;
  }
  r = min(max(r, 1u), n);
  for (int c = 0; c < chunks; ++c) {
    const int base = c * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
    uint32_t k = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      k += base + j < row.V && key_of(x[j]) == prefix && place(x[j], base + j) >= floor;
    k = __reduce_add_sync(0xffffffffu, k);
    if ((tid & 31) == 0) s.cw[c * WARPS + (tid >> 5)] = k;
  }
  __syncthreads();
  find<GROUPS>(s, [&](int i) { return i < chunks * WARPS ? s.cw[i] : 0; }, (double)r);
  const int g = s.i0;
  if ((tid >> 5) == g % WARPS) {
    const int base = g / WARPS * CHUNK + tid * PER;
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

// The same among those of the list's n tokens (s.wc).
template <bool MASS>
__device__ __noinline__ u64 ranked(Work& s, uint32_t n, const Group group, u64 floor, uint32_t r, double want) {
  const int tid = threadIdx.x;
  int shift = 64;
  u64 prefix = 0;
  auto in = [&](u64 c) { return c >= floor && group.has(logit_of(c)) && (shift == 64 || c >> shift == prefix); };
  // their numbers in the list, in place of the counts
  auto gather = [&]() {
    if (tid == 0) s.n = 0;
    __syncthreads();
    for (uint32_t i = tid; i < n; i += TH)
      if (in(s.wc[i])) {
        const uint32_t k = atomicAdd(&s.n, 1u);
        if (k < ND) s.cnt[k] = i;
      }
    __syncthreads();
    const uint32_t m = s.n;
    __syncthreads();
    return m;
  };
  uint32_t m = gather();
  while (m > LIST && shift > 0) {                                      // too many to compare each with each: 11 more bits
    const int wide = min(11, shift), low = shift - wide;
    const uint32_t mask = (1u << wide) - 1;
    for (int i = tid; i < ND; i += TH) {
      s.cnt[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    for (uint32_t i = tid; i < n; i += TH) {
      const u64 c = s.wc[i];
      if (in(c)) {
        const uint32_t d = mask - ((uint32_t)(c >> low) & mask);
        atomicAdd(&s.cnt[d], 1u);
        if (MASS) atomicAdd(&s.mass[d], s.ww[i]);
      }
    }
    __syncthreads();
    const int at = digit<MASS>(s, r, want);
    prefix = prefix << wide | (mask - (uint32_t)at);
    shift = low;
    m = gather();
  }
  if (tid == 0) s.u0 = s.u1 = ~0ull;
  __syncthreads();
  for (uint32_t i = tid; i < m; i += TH) {
    const u64 mine = s.wc[s.cnt[i]];
    u64 before = 0;
    uint32_t rank = 0;
    for (uint32_t j = 0; j < m; ++j) {
      const uint32_t e = s.cnt[j];
      if (s.wc[e] > mine) {
        before += s.ww[e];
        ++rank;
      }
    }
    if (MASS ? (double)before < want && want <= (double)(before + s.ww[s.cnt[i]]) : rank == r - 1) s.u0 = mine;
    if (rank == m - 1) s.u1 = mine;                                    // sums that fall short of `want` keep all
  }
  __syncthreads();
  const u64 got = s.u0 != ~0ull ? s.u0 : s.u1;
  __syncthreads();
  return got;
}

// Where top-p ends: the group in which the weights (s.mass, by group) reach `goal`, -1 if they do not; what is left of goal there.
__device__ __forceinline__ int reached(Work& s, double& goal) {
  if (threadIdx.x == 0) s.i0 = -1;
  __syncthreads();
  find<ND>(s, [&](int i) { return s.mass[i]; }, goal);
  const int g = s.i0;
  if (g >= 0) goal -= (double)s.u0;
  __syncthreads();
  return g;
}

// Both cuts where the list is too short. by_k: the bin in which top-k ends, k_count its tokens; by_p: the bins in which top-p can, from its base to `to`.
template <typename T>
__device__ __noinline__ u64 cut_by_division(const Row<T> row, Work& s, const Weigh weigh, bool k_on, Group by_k, uint32_t k_count, uint32_t k_left, bool p_on, Group by_p, int to,
                                            float tp) {
  const int tid = threadIdx.x, V = row.V;
  const int chunks = (V + CHUNK - 1) / CHUNK;
  u64 floor = 0;
  if (k_on) floor = last_kept<false>(row, s, weigh, by_k, 0ull, k_count, k_left, 0.0);
  if (!p_on) return floor;
  for (int i = tid; i < ND; i += TH) {
    s.cnt[i] = 0;
    s.mass[i] = 0;
  }
  __syncthreads();
  u64 whole = 0, above = 0;
  const int groups = ((to - by_p.base) >> by_p.shift) + 1;
  for (int c = 0; c < chunks; ++c) {
    const int base = c * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (base + j < V && place(x[j], base + j) >= floor) {
        const u64 w = weigh(x[j]);
        const int g = by_p.of(x[j]);
        whole += w;
        if (g < 0) above += w;
        else if (g < groups) {
          atomicAdd(&s.mass[g], w);
          atomicAdd(&s.cnt[g], 1u);
        }
      }
  }
  whole = cta_sum(whole, s.red);
  above = cta_sum(above, s.red);
  double want = fmax((double)tp * (double)whole, 0.5) - (double)above;
  by_p.g = reached(s, want);
  if (by_p.g < 0) return floor;                                        // nothing is cut
  const uint32_t n = s.cnt[by_p.g];
  __syncthreads();
  return last_kept<true>(row, s, weigh, by_p, floor, n, 0u, want);
}

// The weights of a row: sums of the tokens before bin f_first, by 256 tokens (of at least `least`) and altogether, and of all; the tokens of the bins
// from there to f_last go to the list. EVERY: top-k is off, every token's weight counts. SUM: for top-p's sum. CUT: min-p is on.
template <bool SHARED, bool EVERY, bool SUM, bool CUT, typename T>
__device__ __noinline__ void weights(const Row<T> row, Work& s, const Weigh weigh, float f_first, float f_last, u64 least, u64& whole_, u64& sure_) {
  u64 whole = 0, sure = 0;
  row.each_chunk([&](int c, int base, const float (&x)[PER]) {
    u64 kept = 0;
    auto count = [&](u64 w, float at) {
      const u64 before = at < f_first ? w : 0;
      if (SUM) whole += w;
      if (CUT) {
        sure += before;
        kept += before >= least ? before : 0;
      } else {
        kept += before;
      }
    };
    auto list = [&](u64 w, float at, int j) {
      if (at >= f_first && at < f_last && base + j < row.V) {
        const uint32_t i = take_place<SHARED>(&s.n);
        store_first<SHARED>(&s.wc[i], place(x[j], base + j));
        store_first<SHARED>(&s.ww[i], w);
      }
    };
    if constexpr (EVERY) {                                             // nothing in between: eight chains of operations side by side
      u64 w[PER];
      float at[PER];
      bool near = false;
#pragma unroll
      for (int j = 0; j < PER; ++j) {                                  // those behind the end are -inf: no weight
        at[j] = below(weigh.top, x[j]) * weigh.per_bin;
        near |= at[j] >= f_first && at[j] < f_last;
        w[j] = weigh(x[j], at[j]);
      }
#pragma unroll
      for (int j = 0; j < PER; ++j) count(w[j], at[j]);
      if (near) {
#pragma unroll
        for (int j = 0; j < PER; ++j) list(w[j], at[j], j);
      }
    } else {                                                           // few count: most warps see none
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const float at = below(weigh.top, x[j]) * weigh.per_bin;
        if (__any_sync(0xffffffffu, at < f_last)) {
          const u64 w = at < f_last ? weigh(x[j], at) : 0;
          count(w, at);
          list(w, at, j);
        }
      }
    }
    if (!CUT) sure += kept;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, o);
    if ((threadIdx.x & 31) == 0) store_first<SHARED>(&s.cw[c * WARPS + (threadIdx.x >> 5)], kept);
  });
  whole_ = whole;
  sure_ = sure;
}

// SHARED: a cluster for each row
template <typename T, bool SHARED>
__global__ void __launch_bounds__(TH, 1) sample_given_kernel(const T* __restrict__ logits, long long ld, int V, const double* __restrict__ u,
                                                             const float* __restrict__ temperature, const int* __restrict__ top_k,
                                                             const float* __restrict__ top_p, const float* __restrict__ min_p,
                                                             long long* __restrict__ out, float* __restrict__ out_logprob) {
  extern __shared__ __align__(16) unsigned char raw[];
  Work& s = *reinterpret_cast<Work*>(raw);
  const int rank = SHARED ? cluster_rank() : 0, ctas = SHARED ? cluster_size() : 1;
  const int b = blockIdx.x / ctas, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const T* p = logits + (long long)b * ld;
  const Row<T> row{p, V, (reinterpret_cast<uintptr_t>(p) & 15) == 0, rank, ctas};
  const int chunks = (V + CHUNK - 1) / CHUNK;

  // the largest logit, at its lowest index
  float mine_top = -INFINITY;
  int mine_at = tid * PER;
  row.each_chunk([&](int, int base, const float (&x)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (x[j] > mine_top) {
        mine_top = x[j];
        mine_at = base + j;
      }
  });
  if (tid == 0) s.n = 0;
  u64 best = place(mine_top, mine_at);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if (lane == 0) s.red[warp] = best;
  __syncthreads();
  best = lane < WARPS ? s.red[lane] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if constexpr (SHARED) {
    if (tid == 0) s.best = best;
    cluster_barrier();
    best = remote_u64(&s.best, lane % ctas);
#pragma unroll
    for (int o = MOST_CTAS / 2; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  }
  const int arg = (int)(0xffffffffu - (uint32_t)best);
  const float top = logit_of(best);
  __syncthreads();
  if (top == -INFINITY) {                                              // nothing is left: no token is more likely than another
    if (tid == 0 && rank == 0) {
      out[b] = 0;
      if (out_logprob) out_logprob[b] = -INFINITY;
    }
    if constexpr (SHARED) cluster_barrier();                           // nobody leaves while others read its memory
    return;
  }
  const float t = temperature ? temperature[b] : 0.f;
  const bool drawn = t > 0.f;
  const int k = drawn && top_k ? top_k[b] : 0;
  const bool k_on = k > 0 && k < V;
  const float tp = drawn && top_p ? top_p[b] : 1.f;
  const bool p_on = tp < 1.f;
  const float tt = fmaxf(t, 1e-30f);                                   // the distances of a row in units of T stay finite
  const Weigh weigh(top, drawn ? tt : 1.f);
  const float per_bin = weigh.per_bin;

  if (k_on || p_on) {
    for (int i = tid; i < NB; i += TH) s.bins[i] = 0;
    __syncthreads();
  }
  double sum1 = 0.0;                                                   // of sums of eight in 32 bits: the same for any share, to a rounding
  if (out_logprob || k_on || p_on)
    row.each_chunk([&](int, int base, const float (&x)[PER]) {
      if (out_logprob) {
        float some = 0.f;
#pragma unroll
        for (int j = 0; j < PER; ++j) some += expf(-below(top, x[j]));   // nothing for those behind the end
        sum1 += (double)some;
      }
      if (k_on || p_on) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
          if (base + j < V) atomicAdd(&s.bins[bin_of(below(top, x[j]), per_bin)], 1u);
      }
    });
  float log_sum = 0.f;
  double whole1 = 0.0;
  if (out_logprob) {
    double v = sum1;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) s.red[warp] = __double_as_longlong(v);
    __syncthreads();
    v = lane < WARPS ? __longlong_as_double(s.red[lane]) : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    whole1 = v;
  }
  if constexpr (SHARED) {
    if (tid == 0) s.sum1 = whole1;
    cluster_barrier();
    if (out_logprob) {
      whole1 = lane % MOST_CTAS < ctas ? __longlong_as_double((long long)remote_u64(&s.sum1, lane % MOST_CTAS)) : 0.0;
#pragma unroll
      for (int o = MOST_CTAS / 2; o > 0; o >>= 1) whole1 += __shfl_xor_sync(0xffffffffu, whole1, o);
    }
  }
  if (out_logprob) log_sum = (float)log(whole1);
  if (!drawn) {
    if (tid == 0 && rank == 0) {
      out[b] = arg;
      if (out_logprob) out_logprob[b] = -log_sum;
    }
    if constexpr (SHARED) cluster_barrier();
    return;
  }
  __syncthreads();

  // a kept token weighs at least `least`
  const float mp = min_p ? min_p[b] : 0.f;
  const u64 least = mp > 0.f ? (u64)ceil(fmin((double)mp, 1.0) * UNIT) : 0;
  constexpr int MINE = NB / TH;                                        // bins of a thread
  uint32_t cnt[MINE];
  if (k_on || p_on) {
    if constexpr (SHARED) {                                            // a CTA adds up its share of the bins, then everyone reads the sums
      const int share = NB / ctas;
      for (int i = rank * share + 4 * tid; i < (rank + 1) * share; i += 4 * TH) {
        uint4 c = make_uint4(0, 0, 0, 0), v[MOST_CTAS];
#pragma unroll
        for (int r = 0; r < MOST_CTAS; ++r) v[r] = r < ctas ? remote_u32x4(&s.bins[i], r) : make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int r = 0; r < MOST_CTAS; ++r) c = make_uint4(c.x + v[r].x, c.y + v[r].y, c.z + v[r].z, c.w + v[r].w);
        *reinterpret_cast<uint4*>(&s.bins[i]) = c;
      }
      cluster_barrier();
      const int owner = MINE * tid / share;
#pragma unroll
      for (int i = 0; i < MINE; i += 4) {
        const uint4 v = remote_u32x4(&s.bins[MINE * tid + i], owner);
        cnt[i] = v.x;
        cnt[i + 1] = v.y;
        cnt[i + 2] = v.z;
        cnt[i + 3] = v.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < MINE; ++i) cnt[i] = s.bins[MINE * tid + i];
    }
  }
  int k_bin = NB - 1;
  uint32_t k_left = 0, k_count = 0;                                    // tokens of k_bin that top-k keeps; its tokens
  if (k_on) {
    u64 sum = 0, all;
#pragma unroll
    for (int i = 0; i < MINE; ++i) sum += cnt[i];
    u64 before = cta_scan<u64>(sum, s.red, all) - sum;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      if (before < (u64)k && (u64)k <= before + cnt[i]) {
        s.i0 = MINE * tid + i;
        s.i1 = (int)cnt[i];
        s.u0 = before;
      }
      before += cnt[i];
    }
    __syncthreads();
    k_bin = s.i0;
    k_count = (uint32_t)s.i1;
    k_left = (uint32_t)k - (uint32_t)s.u0;
    __syncthreads();
  }
  int from = NB, to = -1, near_from = NB, near_to = -1;                // bins in which top-p can end, and does most of the time
  if (p_on) {
    // a bin's weight lies between its count times its least and its largest weight; so do the running sums, and with them the bins in which the
    // sum can reach top_p of the whole
    const float step = RANGE / NB, fall = __expf(-step);
    float hi[MINE], lo[MINE], hs = 0.f, ls = 0.f, w = __expf(-step * (MINE * tid));
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int at = MINE * tid + i;
      const float c = (float)(k_on && at >= k_bin ? at == k_bin ? k_left : 0u : cnt[i]);
      hi[i] = c * w * 1.0001f;
      w *= fall;
      lo[i] = at == NB - 1 ? 0.f : c * w * 0.9999f;                    // the last bin has no least weight
      hs += hi[i];
      ls += lo[i];
    }
    float most, lowest;
    float ah = cta_scan<float>(hs, s.fred, most) - hs;
    float al = cta_scan<float>(ls, s.fred, lowest) - ls;
    const float pp = fmaxf(tp, 0.f);
    const float lo_goal = pp * lowest * 0.9999f, hi_goal = pp * most * 1.0001f;
    // The mean of both bounds is far nearer (a bin's tokens lie evenly in it): where the bounds leave many tokens, a narrow range around it is
    // looked at first, and the weights themselves tell whether top-p ends there.
    const float mid_goal = pp * 0.5f * (most + lowest);
    if (tid == 0) {
      s.i0 = s.i1 = k_bin;
      s.g0 = s.g1 = k_bin;
    }
    __syncthreads();
    // only threads near where a goal is reached look for it (all those behind it would queue for the same word)
    const float mid0 = 0.5f * (ah + al);
    bool h_done = ah > lo_goal * 1.0001f, l_done = al > hi_goal * 1.0001f, a_done = mid0 > mid_goal, b_done = mid0 > mid_goal * 1.001f;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      ah += hi[i];
      al += lo[i];
      if (!h_done && ah >= lo_goal) { atomicMin(&s.i0, MINE * tid + i); h_done = true; }
      if (!l_done && al >= hi_goal) { atomicMin(&s.i1, MINE * tid + i); l_done = true; }
      const float mid = 0.5f * (ah + al);
      if (!a_done && mid >= mid_goal * (1.f - NEAR)) { atomicMin(&s.g0, MINE * tid + i); a_done = true; }
      if (!b_done && mid >= mid_goal * (1.f + NEAR)) { atomicMin(&s.g1, MINE * tid + i); b_done = true; }
    }
    __syncthreads();
    from = s.i0;
    to = max(s.i1, from);
    near_from = min(max(from, s.g0), to);
    near_to = min(to, max(s.g1, near_from));
    __syncthreads();
  }
  // bins first .. last are looked at token by token; those before are kept, those behind are not (but count for top-p's sum, without top-k)
  const Group by_k{top, per_bin, 0, 0, k_bin};
  Group by_p{top, per_bin, from, 0, 0};
  while (((to - from) >> by_p.shift) >= ND) ++by_p.shift;
  int first = p_on ? from : k_on ? k_bin : NB, last = k_on ? k_bin : to;
  uint32_t n_list = 0, n_before = 0;                                   // their tokens, and those before them (with top-k; else those of the near bins)
  if (first <= last) {
    u64 c = 0;
#pragma unroll
    for (int i = 0; i < MINE; ++i) {
      const int at = MINE * tid + i;
      if (at <= last && at >= first) c += cnt[i];
      if (k_on ? at < first : at >= near_from && at <= near_to) c += (u64)cnt[i] << 32;
    }
    c = cta_sum(c, s.red);
    n_list = (uint32_t)c;
    n_before = (uint32_t)(c >> 32);
  }
  const bool guess = !k_on && n_list > TH;
  if (guess) {
    first = near_from;
    last = near_to;
    n_list = n_before;
  }
  Group near = by_p;
  if (guess) {
    near.base = near_from;
    near.shift = 0;
    while (((near_to - near_from) >> near.shift) >= ND) ++near.shift;
  }
  bool again = n_list > WINDOW;
  u64 whole = 0, sure = 0;                                             // weight of everything that top-p's sum counts; of the tokens before `first`
  if (!again) {
    if (tid == 0) s.u0 = 0;
    __syncthreads();
    const float f_first = (float)first, f_last = last == NB - 1 ? INFINITY : (float)(last + 1);
    if (k_on) {
      if (least) weights<SHARED, false, false, true>(row, s, weigh, f_first, f_last, least, whole, sure);
      else weights<SHARED, false, false, false>(row, s, weigh, f_first, f_last, least, whole, sure);
    } else if (p_on) {
      if (least) weights<SHARED, true, true, true>(row, s, weigh, f_first, f_last, least, whole, sure);
      else weights<SHARED, true, true, false>(row, s, weigh, f_first, f_last, least, whole, sure);
    } else {
      if (least) weights<SHARED, true, false, true>(row, s, weigh, f_first, f_last, least, whole, sure);
      else weights<SHARED, true, false, false>(row, s, weigh, f_first, f_last, least, whole, sure);
    }
    __syncthreads();
  }
  if constexpr (SHARED) {                                              // the first CTA goes on alone
    whole = cta_sum(whole, s.red);
    sure = cta_sum(sure, s.red);
    if (tid == 0) {
      s.part[0] = whole;
      s.part[1] = sure;
    }
    cluster_barrier();
    if (rank == 0) {
      const bool mine = tid < ctas;
      whole = mine ? remote_u64(&s.part[0], tid) : 0;
      sure = mine ? remote_u64(&s.part[1], tid) : 0;
    }
    cluster_barrier();
    if (rank) return;
  }
  if (!again) {
    n_list = s.n;
    if (first <= last && n_list <= TH) {                               // a token a thread: in order, with the weight before it
      constexpr int SORTED = WINDOW / 2;
      const u64 mine = tid < n_list ? s.wc[tid] : 0;
      if (warp * 32 < n_list) {
        uint32_t rank = 0;
        for (uint32_t j = 0; j < n_list; ++j) rank += s.wc[j] > mine;
        if (tid < n_list) {
          s.wc[SORTED + rank] = mine;
          s.ww[SORTED + rank] = s.ww[tid];
        }
      }
      __syncthreads();
      const u64 c = tid < n_list ? s.wc[SORTED + tid] : 0, w = tid < n_list ? s.ww[SORTED + tid] : 0;
      u64 all;
      const u64 after = cta_scan<u64>(w, s.red, all), before = after - w;
      const uint32_t limit = k_on ? min(n_list, (uint32_t)k - n_before) : n_list;
      if (tid + 1 == limit) s.u0 = after;
      double want = INFINITY;
      if (p_on) {
        sure = cta_sum(sure, s.red);
        whole = k_on ? sure + s.u0 : cta_sum(whole, s.red);            // with top-k, its sum counts what that keeps
        want = fmax((double)tp * (double)whole, 0.5) - (double)sure;
      }
      again = guess && !(want > 0.0 && want <= (double)s.u0);
      if (!again) {
        const bool keep = tid < limit && (double)before < want, next = tid + 1 < limit && (double)after < want;
        if (keep && w >= least) atomicAdd(&s.cw[(0xffffffffu - (uint32_t)c) / (32 * PER)], w);
        if (keep && !next) s.u1 = c;
        if (tid == 0 && !keep) s.u1 = c + 1;
      }
    } else if (first <= last) {
      const uint32_t n = n_list;
      u64 floor = 0;
      if (k_on) {
        floor = ranked<false>(s, n, by_k, 0ull, k_left, 0.0);
        if (p_on) {                                                    // of the list, top-p's sum counts what top-k keeps
          u64 w = 0;
          for (uint32_t i = tid; i < n; i += TH)
            if (s.wc[i] >= floor) w += s.ww[i];
          whole = sure + w;
        }
      }
      if (p_on) {
        whole = cta_sum(whole, s.red);
        sure = cta_sum(sure, s.red);
        for (int i = tid; i < ND; i += TH) s.mass[i] = 0;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += TH)
          if (s.wc[i] >= floor) {
            const int g = near.of(logit_of(s.wc[i]));
            if (g < ND) atomicAdd(&s.mass[g], s.ww[i]);
          }
        __syncthreads();
        double want = fmax((double)tp * (double)whole, 0.5) - (double)sure;
        again = guess && want <= 0.0;
        near.g = reached(s, want);
        again |= guess && near.g < 0;
        if (!again && near.g >= 0) floor = ranked<true>(s, n, near, floor, 0u, want);       // else nothing is cut
      }
      if (!again) {
        for (uint32_t i = tid; i < n; i += TH)
          if (s.wc[i] >= floor && s.ww[i] >= least) atomicAdd(&s.cw[(0xffffffffu - (uint32_t)s.wc[i]) / (32 * PER)], s.ww[i]);
        if (tid == 0) s.u1 = floor;
      }
    } else if (tid == 0) {
      s.u1 = 0;
    }
    __syncthreads();
  }
  if (again) {
    const u64 floor = cut_by_division(row, s, weigh, k_on, by_k, k_count, k_left, p_on, by_p, to, tp);
    for (int c = 0; c < chunks; ++c) {
      const int base = c * CHUNK + tid * PER;
      float x[PER];
      row.get(base, x);
      u64 kept = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (base + j < V && place(x[j], base + j) >= floor) {
          const u64 w = weigh(x[j]);
          kept += w >= least ? w : 0;
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) kept += __shfl_xor_sync(0xffffffffu, kept, o);
      if (lane == 0) s.cw[c * WARPS + warp] = kept;
    }
    if (tid == 0) s.u1 = floor;
  }
  __syncthreads();
  const u64 floor = s.u1;
  constexpr int E = GROUPS / TH;
  u64 group[E], sum = 0, all;
#pragma unroll
  for (int i = 0; i < E; ++i) sum += group[i] = E * tid + i < chunks * WARPS ? s.cw[E * tid + i] : 0;
  u64 before = cta_scan<u64>(sum, s.red, all) - sum;
  // a number that rounding takes to the whole sum falls on the last token
  const double goal = fmin(fmax(u[b], 0.0) * (double)all, (double)all * (1.0 - 2.3e-16));
  if (tid == 0) s.i0 = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < E; ++i) {
    if (group[i] && (double)before <= goal && goal < (double)(before + group[i])) {
      s.i0 = E * tid + i;
      s.u0 = before;
    }
    before += group[i];
  }
  __syncthreads();
  const int g = s.i0;
  if (warp == g % WARPS) {
    const int base = g / WARPS * CHUNK + tid * PER;
    float x[PER];
    row.get(base, x);
    u64 w[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      w[j] = base + j < V && place(x[j], base + j) >= floor ? weigh(x[j]) : 0;
      if (w[j] < least) w[j] = 0;
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
    DLTI_CUDA_CHECK(cudaFuncSetAttribute(sample_given_kernel<T, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Work)));
    DLTI_CUDA_CHECK(cudaFuncSetAttribute(sample_given_kernel<T, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Work)));
    set[dev & 63] = true;
  }
  // Several SMs for a row where there are few of them. What the CTAs tell each other takes time of its own, so a row has to be long (us for 1 / 2 / 4 / 8
  // CTAs, of bf16 rows: one row of 32,000 31 / 33 / 29, of 99,444 in fp32 84 / 59 / 43 / 35; 32 rows of 128,000 100 / 76 / 55; 64 rows 100 / 76), and
  // clusters of eight find room for no more than some eight rows at once (16 rows of 128,000 55 us by four, 88 by eight).
  const int chunks = (V + CHUNK - 1) / CHUNK;
  const int ctas = batch <= 8 && chunks >= 16 ? MOST_CTAS : batch <= 32 && chunks >= 8 ? 4 : batch <= 64 && chunks >= 16 ? 2 : 1;
  DLTI_CUDA_CHECK(dlti_launch_pdl_cluster(DLTI_PDL_MAX_ROWS + 1, ctas, ctas > 1 ? sample_given_kernel<T, true> : sample_given_kernel<T, false>,
                                          dim3((unsigned)(batch * ctas)), dim3(TH), sizeof(Work), st, (const T*)logits, ld, V, u, t, k, p, mp, out, lp));
  dlti_count_launch();
  return 0;
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
