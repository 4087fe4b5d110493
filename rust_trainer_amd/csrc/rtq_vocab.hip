// rtq_vocab.hip — operators on rows of vocabulary logits (included by rtq_kernels.hip): a teacher's
// top logits, distillation from them with its gradient, and the verification of drafted tokens.
// Rows are f32, f16 or bf16, V long, at any stride and any element alignment: they are read and
// written 16 bytes at a time through an unaligned vector type (gfx950 takes such accesses at any
// element boundary), the last partial vector element by element.

typedef uint32_t u4u __attribute__((ext_vector_type(4), aligned(2)));

enum { VT_F32 = 0, VT_F16 = 1, VT_BF16 = 2 };

template <int VT>
struct VRow {
  static constexpr int ES = VT == VT_F32 ? 4 : 2;
  static constexpr int E = 16 / ES;  // elements per 16-byte vector
  __device__ static __forceinline__ float one(const void* p, int64_t j) {
    if constexpr (VT == VT_F32) return static_cast<const float*>(p)[j];
    else if constexpr (VT == VT_F16) return (float)static_cast<const _Float16*>(p)[j];
    else return __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[j] << 16);
  }
  __device__ static __forceinline__ uint16_t bf(float v) {  // to nearest even, NaN kept quiet
    return __builtin_bit_cast(uint16_t, (__bf16)v);
  }
  __device__ static __forceinline__ void put(void* p, int64_t j, float v) {
    if constexpr (VT == VT_F32) static_cast<float*>(p)[j] = v;
    else if constexpr (VT == VT_F16) static_cast<_Float16*>(p)[j] = (_Float16)v;
    else static_cast<uint16_t*>(p)[j] = bf(v);
  }
  // element e of a raw vector
  __device__ static __forceinline__ float get(const u4v& r, int e) {
    // (a copy first: a bit cast of a vector's element itself reads element 0)
    const uint32_t u = r[VT == VT_F32 ? e : e >> 1];
    if constexpr (VT == VT_F32) return __builtin_bit_cast(float, u);
    else if constexpr (VT == VT_F16) return (float)__builtin_bit_cast(_Float16, (uint16_t)(u >> (16 * (e & 1))));
    else return __builtin_bit_cast(float, (e & 1) ? (u & 0xffff0000u) : (u << 16));
  }
  __device__ static __forceinline__ u4v pack(const float* v) {
    u4v r;
    if constexpr (VT == VT_F32) {
#pragma unroll
      for (int e = 0; e < 4; e++) r[e] = __builtin_bit_cast(uint32_t, v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        uint16_t lo, hi;
        if constexpr (VT == VT_F16) {
          lo = __builtin_bit_cast(uint16_t, (_Float16)v[2 * e]);
          hi = __builtin_bit_cast(uint16_t, (_Float16)v[2 * e + 1]);
        } else {
          lo = bf(v[2 * e]), hi = bf(v[2 * e + 1]);
        }
        r[e] = (uint32_t)lo | (uint32_t)hi << 16;
      }
    }
    return r;
  }
  __device__ static __forceinline__ u4v load(const void* row, int64_t j) {
    return *reinterpret_cast<const u4u*>(static_cast<const char*>(row) + j * ES);
  }
  __device__ static __forceinline__ void store(void* row, int64_t j, const u4v& r) {
    *reinterpret_cast<u4u*>(static_cast<char*>(row) + j * ES) = r;
  }
  // elements j .. j + E - 1 of a row of V; those past its end read as `fill`
  __device__ static __forceinline__ u4v load_upto(const void* row, int64_t j, int64_t V, float fill) {
    if (j + E <= V) return load(row, j);
    float v[E];
#pragma unroll
    for (int e = 0; e < E; e++) v[e] = j + e < V ? one(row, j + e) : fill;
    return pack(v);
  }
};

// exp(t / T) for t <= 0 as exp2(t c), c = log2(e) / T given as ch + cl: the product's rounding and
// cl enter to first order, so the result is near the exponential instruction's own last place at
// every t (the plain product is off by |t c| 2^-24, which a small divergence would show)
__device__ __forceinline__ float exp_scaled(float t, float ch, float cl) {
  const float y = t * ch;
  const float d = fmaf(t, cl, fmaf(t, ch, -y));
  const float e = __builtin_amdgcn_exp2f(y);
  return y < -150.0f ? 0.0f : fmaf(e, d * 0.693147181f, e);  // -inf and overflows of t ch among them
}

// whether row i has logits (rows formed at positions: the position is one of the sequence's)
template <class Args>
__device__ __forceinline__ bool row_ok(const Args& a, int i) {
  return !a.pos || (a.pos[i] >= 0 && a.pos[i] < a.t);
}

template <class T>
__device__ __forceinline__ T wave_sum_any(T v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}

// sum / maximum over a workgroup of W waves (red: W values of LDS); every thread gets the result
template <int W, class T>
__device__ __forceinline__ T group_sum(T v, T* red) {
  v = wave_sum_any(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  T s = red[0];
#pragma unroll
  for (int w = 1; w < W; w++) s += red[w];
  return s;
}
template <int W>
__device__ __forceinline__ float group_max(float v, float* red) {
  v = wave_max(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = red[0];
#pragma unroll
  for (int w = 1; w < W; w++) s = fmaxf(s, red[w]);
  return s;
}

// ============================================================== top logits
// A logit's rank as one whole number: its order-preserving bits above, the complement of its index
// below, so that larger is better, equal values go by the lower index (-0 equals 0) and NaN is above
// every number.  0 is no logit.
__device__ __forceinline__ uint64_t rank_key(float x, int j) {
  uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  u = x != x ? 0xffffffffu : (u >> 31) ? ~u : u | 0x80000000u;
  return (uint64_t)u << 32 | (uint32_t)~j;
}
__device__ __forceinline__ float key_value(uint64_t k) {
  const uint32_t u = (uint32_t)(k >> 32);
  if (u == 0xffffffffu) return __builtin_nanf("");
  return __builtin_bit_cast(float, (u >> 31) ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_index(uint64_t k) { return (int)~(uint32_t)k; }

// (max, sum of exp((x - max) / T)) of two sets
__device__ __forceinline__ void join_sums(float& m, double& s, float m2, double s2, double invt) {
  if (m2 == -__builtin_inff()) return;
  if (m == -__builtin_inff()) {
    m = m2, s = s2;
    return;
  }
  const float mm = fmaxf(m, m2);
  s = s * exp(((double)m - mm) * invt) + s2 * exp(((double)m2 - mm) * invt);
  m = mm;
}
__device__ __forceinline__ float lse_of(float m, double s, double invt) {
  if (m == -__builtin_inff() || m == __builtin_inff()) return m;
  return (float)((double)m * invt + log(s));
}

// keys[0 .. P) sorted from the largest, P a power of two
template <int B>
__device__ __forceinline__ void sort_keys(uint64_t* keys, int P) {
  for (int k = 2; k <= P; k <<= 1)
    for (int j = k >> 1; j > 0; j >>= 1) {
      __syncthreads();
      for (int p = threadIdx.x; p < P / 2; p += B) {
        const int i = 2 * p - (p & (j - 1)), q = i | j;
        const uint64_t a = keys[i], b = keys[q];
        if ((a < b) == ((i & k) == 0)) keys[i] = b, keys[q] = a;
      }
    }
  __syncthreads();
}

// lane i's value of the wave's 64 sorted from the largest
__device__ __forceinline__ float wave_sort(float v) {
  const int l = threadIdx.x & 63;
#pragma unroll
  for (int k = 2; k <= 64; k <<= 1)
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const float o = __shfl_xor(v, j);
      const bool up = ((l & k) == 0) == ((l & j) == 0);  // this lane keeps the larger
      v = up ? fmaxf(v, o) : fminf(v, o);
    }
  return v;
}

constexpr int kTopB = 1024, kTopW = kTopB / 64, kTopCap = 2048;

// the outputs of a row without logits
__device__ __forceinline__ void top_none(const TopArgs& a, int i) {
  for (int s = threadIdx.x; s < a.k; s += kTopB) a.vals[(int64_t)i * a.k + s] = __builtin_nanf(""), a.ids[(int64_t)i * a.k + s] = -1;
  if (threadIdx.x == 0 && a.rest) a.rest[i] = __builtin_nanf("");
}

// The k largest of slice g of row i, in order, and (max, sum) of the slice's others.  The slice stays
// in registers (NV vectors a thread).  A bound below the k-th largest comes from the lanes' maxima:
// with r = ceil(k / waves), every wave has r maxima at or above its own r-th, so the least of those r-ths
// has k logits at or above it.  What reaches the bound (about 1.5 to 4 k of them in a row without
// structure) is gathered and sorted.  Where more than kTopCap reach it (ties, masks, sorted rows), the
// bound is found digit by digit over the whole keys instead.
template <int VT, int NV>
__device__ __forceinline__ void top_slice(const TopArgs& a) {
  using R = VRow<VT>;
  __shared__ uint64_t cand[kTopCap];
  __shared__ float redf[kTopW];
  __shared__ double redd[kTopW];
  __shared__ int hist[256];
  __shared__ int cnt, pick, above;
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  if (!row_ok(a, i)) {
    if (g == 0) top_none(a, i);
    return;
  }
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);  // L <= kTopB * NV * E
  const float ninf = -__builtin_inff();
  u4v raw[NV];
#pragma unroll
  for (int q = 0; q < NV; q++) {
    const int j = j0 + (q * kTopB + tid) * R::E;
    float f[R::E];
#pragma unroll
    for (int e = 0; e < R::E; e++) f[e] = ninf;
    raw[q] = j < j1 ? R::load_upto(row, j, j1, ninf) : R::pack(f);
  }
  float lm = ninf;
#pragma unroll
  for (int q = 0; q < NV; q++)
#pragma unroll
    for (int e = 0; e < R::E; e++) lm = fmaxf(lm, R::get(raw[q], e));
  if (tid == 0) cnt = 0;
  const int r = (a.k + kTopW - 1) / kTopW;
  const float ws = wave_sort(lm);
  if ((tid & 63) == r - 1) redf[tid >> 6] = ws;
  __syncthreads();
  float thr = redf[0];
#pragma unroll
  for (int w = 1; w < kTopW; w++) thr = fminf(thr, redf[w]);
  __syncthreads();
  // gather what is not below the bound (NaN is not); an index at or past j1 is padding
  float nm = ninf;
  auto gather = [&](auto&& in) {
    nm = ninf;
#pragma unroll
    for (int q = 0; q < NV; q++)
#pragma unroll
      for (int e = 0; e < R::E; e++) {
        const int j = j0 + (q * kTopB + tid) * R::E + e;
        const float x = R::get(raw[q], e);
        const bool c = j < j1 && in(x, j);
        if (!c) nm = fmaxf(nm, x);
        const uint64_t m = __ballot(c);
        if (m) {
          int at = 0;
          if ((tid & 63) == __builtin_ctzll(m)) at = atomicAdd(&cnt, __popcll(m));
          at = __shfl(at, __builtin_ctzll(m)) + __popcll(m & ((1ull << (tid & 63)) - 1));
          if (c && at < kTopCap) cand[at] = rank_key(x, j);
        }
      }
  };
  gather([&](float x, int) { return !(x < thr); });
  __syncthreads();
  int n = cnt;
  uint64_t low = 0;
  const bool many = n > kTopCap;
  if (many) {
    uint64_t mask = 0;
    int need = a.k;
    for (int sh = 56; sh >= 0; sh -= 8) {
      for (int b = tid; b < 256; b += kTopB) hist[b] = 0;
      __syncthreads();
#pragma unroll
      for (int q = 0; q < NV; q++)
#pragma unroll
        for (int e = 0; e < R::E; e++) {
          const int j = j0 + (q * kTopB + tid) * R::E + e;
          const uint64_t key = rank_key(R::get(raw[q], e), j);
          const bool in = j < j1 && (key & mask) == low;
          const int d = (int)(key >> sh) & 255;
          // equal digits of a wave (ties, the index's upper digits) are counted with one atomic
          const uint64_t m = __ballot(in);
          if (m) {
            const int first = __shfl(d, __builtin_ctzll(m));
            if (__ballot(in && d != first) == 0) {
              if ((tid & 63) == __builtin_ctzll(m)) atomicAdd(&hist[d], __popcll(m));
            } else if (in) {
              atomicAdd(&hist[d], 1);
            }
          }
        }
      __syncthreads();
      if (tid == 0) {
        int s = 0, b = 255;
        while (b > 0 && s + hist[b] < need) s += hist[b--];
        pick = b, above = s;
      }
      __syncthreads();
      const int inbin = hist[pick];
      need -= above;
      low |= (uint64_t)pick << sh;
      mask |= (uint64_t)255 << sh;
      const bool done = a.k - need + inbin <= kTopCap;
      __syncthreads();
      if (done) break;
    }
    if (tid == 0) cnt = 0;
    __syncthreads();
    gather([&](float x, int j) { return rank_key(x, j) >= low; });
    __syncthreads();
    n = cnt;
  }
  // others: the maximum and the sum of what was not gathered, then the gathered beyond the k-th
  nm = group_max<kTopW>(nm, redf);
  double ns = 0.0;
  if (nm != ninf && (a.rest || a.G > 1)) {
#pragma unroll
    for (int q = 0; q < NV; q++) {
      float s = 0.0f;
#pragma unroll
      for (int e = 0; e < R::E; e++) {
        const int j = j0 + (q * kTopB + tid) * R::E + e;
        const float x = R::get(raw[q], e);
        const bool c = j >= j1 || (many ? rank_key(x, j) >= low : !(x < thr));
        s += c ? 0.0f : exp_scaled(x - nm, a.ch, a.cl);
      }
      ns += (double)s;
    }
  }
  ns = group_sum<kTopW>(ns, redd);
  int P = 2;
  while (P < n || P < a.k) P <<= 1;
  for (int p = n + tid; p < P; p += kTopB) cand[p] = 0;
  sort_keys<kTopB>(cand, P);
  const double invt = 1.0 / (double)a.temp;
  const float cm = a.k < n ? key_value(cand[a.k]) : ninf;
  double cs = 0.0;
  for (int p = a.k + tid; p < n; p += kTopB) cs += cm == ninf ? 0.0 : exp(((double)key_value(cand[p]) - cm) * invt);
  cs = group_sum<kTopW>(cs, redd);
  join_sums(nm, ns, cm, cs, invt);
  if (a.G > 1) {
    for (int s = tid; s < a.k; s += kTopB) a.lists[((int64_t)i * a.G + g) * a.k + s] = cand[s];
    if (tid == 0) a.pm[(int64_t)i * a.G + g] = nm, a.ps[(int64_t)i * a.G + g] = ns;
    return;
  }
  for (int s = tid; s < a.k; s += kTopB) {
    a.vals[(int64_t)i * a.k + s] = key_value(cand[s]);
    a.ids[(int64_t)i * a.k + s] = key_index(cand[s]);
  }
  if (tid == 0 && a.rest) a.rest[i] = lse_of(nm, ns, invt);
}

// row i's k largest of its G slices' sorted lists (lists[g][s], 0 where a slice has fewer), by the
// same bound: the least of the lists' r-ths, r = ceil(k / G), or the largest of their k-ths
extern "C" __global__ __launch_bounds__(kTopB) void rtq_top_merge(TopArgs a) {
  extern __shared__ uint64_t mkeys[];  // G * k rounded up to a power of two
  __shared__ float redf[kTopW];
  __shared__ double redd[kTopW];
  __shared__ int cnt;
  __shared__ uint64_t bound;
  const int tid = threadIdx.x, i = blockIdx.x, r = (a.k + a.G - 1) / a.G, total = a.G * a.k;
  const uint64_t* L = a.lists + (int64_t)i * total;
  if (!row_ok(a, i)) return;  // written by slice 0
  if (tid < 64) {
    uint64_t lo = ~0ull, hi = 0;
    for (int g = tid; g < a.G; g += 64) {
      const uint64_t x = L[g * a.k + r - 1], y = L[g * a.k + a.k - 1];
      lo = x < lo ? x : lo, hi = y > hi ? y : hi;
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const uint64_t x = __shfl_xor(lo, m), y = __shfl_xor(hi, m);
      lo = x < lo ? x : lo, hi = y > hi ? y : hi;
    }
    if (tid == 0) bound = hi > lo ? hi : lo, cnt = 0;
  }
  __syncthreads();
  const uint64_t low = bound > 1 ? bound : 1;
  for (int p = tid; p < total; p += kTopB) {
    const uint64_t key = L[p];
    if (key >= low) mkeys[atomicAdd(&cnt, 1)] = key;
  }
  __syncthreads();
  const int n = cnt;
  int P = 2;
  while (P < n || P < a.k) P <<= 1;
  for (int p = n + tid; p < P; p += kTopB) mkeys[p] = 0;
  sort_keys<kTopB>(mkeys, P);
  for (int s = tid; s < a.k; s += kTopB) {
    a.vals[(int64_t)i * a.k + s] = key_value(mkeys[s]);
    a.ids[(int64_t)i * a.k + s] = key_index(mkeys[s]);
  }
  if (!a.rest) return;
  // the others: the slices' own, and every list entry after the k-th
  const double invt = 1.0 / (double)a.temp;
  const uint64_t kth = mkeys[a.k - 1];
  float m = -__builtin_inff();
  bool nan = false;
  for (int p = tid; p < total; p += kTopB) {
    const uint64_t key = L[p];
    if (key == 0 || key >= kth) continue;
    m = fmaxf(m, key_value(key));
    nan |= key_value(key) != key_value(key);
  }
  for (int g = tid; g < a.G; g += kTopB) m = fmaxf(m, a.pm[(int64_t)i * a.G + g]);
  m = group_max<kTopW>(m, redf);
  double s = nan ? (double)__builtin_nanf("") : 0.0;
  if (m != -__builtin_inff()) {
    for (int p = tid; p < total; p += kTopB) {
      const uint64_t key = L[p];
      if (key != 0 && key < kth) s += exp(((double)key_value(key) - m) * invt);
    }
    for (int g = tid; g < a.G; g += kTopB) {
      const float pm = a.pm[(int64_t)i * a.G + g];
      if (pm != -__builtin_inff()) s += a.ps[(int64_t)i * a.G + g] * exp(((double)pm - m) * invt);
    }
  }
  s = group_sum<kTopW>(s, redd);
  if (tid == 0) a.rest[i] = s != s && m != __builtin_inff() ? __builtin_nanf("") : lse_of(m, s, invt);
}

#define RTQ_TOP(name, VT, NV) \
  extern "C" __global__ __launch_bounds__(kTopB) void name(TopArgs a) { top_slice<VT, NV>(a); }
RTQ_TOP(rtq_top_f32_s, VT_F32, 2)
RTQ_TOP(rtq_top_f16_s, VT_F16, 2)
RTQ_TOP(rtq_top_bf16_s, VT_BF16, 2)
RTQ_TOP(rtq_top_f32_l, VT_F32, 8)
RTQ_TOP(rtq_top_f16_l, VT_F16, 4)
RTQ_TOP(rtq_top_bf16_l, VT_BF16, 4)

// ============================================================== distillation
// Row i: the teacher's distribution p over its listed tokens and the rest (one bucket), the student's
// q = softmax(z / T) over the same buckets.  The unlisted logits have their own maximum m and sums
// sT = sum exp((z - m) / T), s1 = sum exp(z - m), so the rest's probability is no difference of two
// sums.  Gradient at an unlisted token: C exp((z - m) / T) + D exp(z - m) with one C and D a row.
constexpr int kDisB = 256, kDisW = kDisB / 64;

// grid (G, n): the statistics of slice g's unlisted logits; the listed tokens' and the label's logits are
// kept aside (the gradient may overwrite them)
template <int VT>
__device__ __forceinline__ void distill_stats(const DistillArgs& a) {
  using R = VRow<VT>;
  extern __shared__ uint32_t mask[];  // a bit per logit of the slice: listed
  __shared__ float redf[kDisW];
  __shared__ double redd[kDisW];
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  if (!row_ok(a, i)) return;
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);
  const float ninf = -__builtin_inff();
  for (int w = tid; w < a.L / 32; w += kDisB) mask[w] = 0;
  __syncthreads();
  int twice = 0;
  for (int s = tid; s < a.k; s += kDisB) {
    const int id = a.ids[(int64_t)i * a.k + s];
    if (id >= j0 && id < j1) {
      const uint32_t bit = 1u << ((id - j0) & 31);
      twice |= (atomicOr(&mask[(id - j0) >> 5], bit) & bit) != 0;
      a.zs[(int64_t)i * a.k + s] = R::one(row, id);
    }
  }
  if (tid == 0 && a.tok) {
    const int t = a.tok[i];
    if (t >= j0 && t < j1) a.zt[i] = R::one(row, t);
  }
  twice = __syncthreads_or(twice);
  auto each = [&](auto&& f) {
    for (int j = j0 + tid * R::E; j < j1; j += kDisB * R::E) {
      const u4v r = R::load_upto(row, j, j1, ninf);
      const uint32_t bits = mask[(j - j0) >> 5] >> ((j - j0) & 31);
#pragma unroll
      for (int e = 0; e < R::E; e++) f((bits >> e) & 1 ? ninf : R::get(r, e));
    }
  };
  float m = ninf;
  each([&](float x) { m = fmaxf(m, x); });
  m = group_max<kDisW>(m, redf);
  const float ref = m == ninf ? 0.0f : m;
  double sT = 0.0, s1 = 0.0;
  each([&](float x) { sT += (double)exp_scaled(x - ref, a.ch, a.cl); });
  if (a.tok) each([&](float x) { s1 += (double)exp_scaled(x - ref, 1.44269502f, 1.92596303e-8f); });
  sT = group_sum<kDisW>(sT, redd);  // NaN if a logit is
  s1 = group_sum<kDisW>(s1, redd);
  if (tid == 0) {
    const int64_t o = (int64_t)i * a.G + g;
    a.pm[o] = m, a.psT[o] = sT, a.ps1[o] = s1, a.twice[o] = twice;
  }
}

// grid (G, n): row i's scalars from its slices' statistics and the teacher's list (each workgroup forms
// them again: k <= 256 = one slot a thread), the losses by slice 0, the gradient over slice g
template <int VT>
__device__ __forceinline__ void distill_grad(const DistillArgs& a) {
  using R = VRow<VT>;
  __shared__ float redf[kDisW];
  __shared__ double redd[kDisW];
  __shared__ int idl[kDisB];
  __shared__ double pl[kDisB];
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  const float ninf = -__builtin_inff();
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);
  void* out = static_cast<char*>(a.dz) + (int64_t)i * a.ldd * R::ES;
  if (!row_ok(a, i)) {
    if (g == 0 && tid == 0) {
      a.kl[i] = __builtin_nanf("");
      if (a.logp) a.logp[i] = __builtin_nanf("");
    }
    for (int j = j0 + tid; a.w && j < j1; j += kDisB) R::put(out, j, 0.0f);
    return;
  }
  const double invt = 1.0 / (double)a.temp;
  // the unlisted
  float mu = ninf;
  int twice = 0;
  for (int q = tid; q < a.G; q += kDisB) mu = fmaxf(mu, a.pm[(int64_t)i * a.G + q]), twice |= a.twice[(int64_t)i * a.G + q];
  mu = group_max<kDisW>(mu, redf);
  twice = __syncthreads_or(twice);
  double sT = 0.0, s1 = 0.0;
  for (int q = tid; q < a.G; q += kDisB) {
    const int64_t o = (int64_t)i * a.G + q;
    const float pm = a.pm[o];
    const double f = pm == ninf ? 1.0 : exp(((double)pm - mu) * invt), f1 = pm == ninf ? 1.0 : exp((double)pm - mu);
    sT += a.psT[o] * f;
    s1 += a.ps1[o] * f1;
  }
  sT = group_sum<kDisW>(sT, redd);
  s1 = group_sum<kDisW>(s1, redd);
  // the teacher's slots
  const int id = tid < a.k ? a.ids[(int64_t)i * a.k + tid] : -1;
  const bool held = id >= 0 && id < a.V;
  const float tv = held ? a.tv[(int64_t)i * a.k + tid] : ninf;
  const float zs = held ? a.zs[(int64_t)i * a.k + tid] : ninf;
  const double rest = a.rest ? (double)a.rest[i] : -__builtin_inf();
  const double tmax = fmax((double)group_max<kDisW>(tv, redf) * invt, rest);
  const bool nant = __syncthreads_or(tv != tv);
  const bool taught = tmax != -__builtin_inf() || nant || rest != rest;
  double pe = tv == ninf ? 0.0 : exp((double)tv * invt - tmax);
  const double re = rest == -__builtin_inf() ? 0.0 : exp(rest - tmax);
  const double tsum = group_sum<kDisW>(pe, redd) + re;
  const double ps = taught ? pe / tsum : 0.0, pr = taught ? re / tsum : 0.0;
  // tokens listed twice: the first slot stands for the token, with the sum of its slots
  bool first = held;
  double pt = ps;
  if (twice) {
    idl[tid] = held ? id : -1, pl[tid] = ps;
    __syncthreads();
    if (held) {
      pt = 0.0;
      for (int s = 0; s < a.k; s++)
        if (idl[s] == id) {
          if (s < tid) first = false;
          pt += pl[s];
        }
    }
  }
  // the student over all logits
  const float ml = group_max<kDisW>(zs, redf);
  const float M = fmaxf(mu, ml);
  const double fu = mu == ninf ? 0.0 : exp(((double)mu - M) * invt), fu1 = mu == ninf ? 0.0 : exp((double)mu - M);
  const double es = first && zs != ninf ? exp(((double)zs - M) * invt) : 0.0;
  const double es1 = first && zs != ninf && a.tok ? exp((double)zs - M) : 0.0;
  const bool bad = __syncthreads_or(zs != zs);  // a NaN among the listed
  const double nanv = (double)__builtin_nanf("");
  double ZT = group_sum<kDisW>(es, redd) + (mu == ninf && sT == sT ? 0.0 : sT * fu);
  double Z1 = group_sum<kDisW>(es1, redd) + (mu == ninf && s1 == s1 ? 0.0 : s1 * fu1);
  if (bad || M == ninf) ZT = nanv, Z1 = nanv;
  const double lT = log(ZT);
  const int tk = a.tok ? a.tok[i] : -1;
  const bool label = tk >= 0 && tk < a.V;
  const float zt = label ? a.zt[i] : ninf;
  if (g == 0) {
    double kl = ps > 0.0 || ps != ps ? ps * (log(ps) - ((((double)zs - M) * invt) - lT)) : 0.0;
    kl = group_sum<kDisW>(kl, redd);
    if (pr > 0.0 || pr != pr) kl += pr * (log(pr) - ((((double)mu - M) * invt + log(sT)) - lT));
    if (tid == 0) {
      a.kl[i] = taught ? (float)kl : 0.0f;
      if (a.logp) a.logp[i] = label ? (float)((double)zt - M - log(Z1)) : __builtin_nanf("");
    }
  }
  if (!a.w) return;
  const double w = (double)a.w[i];
  const double wT = taught ? w * (1.0 - (double)a.hard) * (double)a.temp : 0.0, w1 = label ? w * (double)a.hard : 0.0;
  const bool empty = mu == ninf;
  const float C = w == 0.0 || wT == 0.0 || (empty && ZT == ZT) ? 0.0f : (float)(wT * (fu / ZT - (pr > 0.0 ? pr / sT : 0.0)));
  const float D = w == 0.0 || w1 == 0.0 || (empty && Z1 == Z1) ? 0.0f : (float)(w1 * (fu1 / Z1));
  const float ref = empty ? 0.0f : mu;
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  for (int j = j0 + tid * R::E; j < j1; j += kDisB * R::E) {
    const u4v r = R::load_upto(row, j, j1, ninf);
    float f[R::E];
#pragma unroll
    for (int e = 0; e < R::E; e++) {
      const float t = R::get(r, e) - ref;
      float v = 0.0f;
      if (C != 0.0f) v = C * exp_scaled(t, a.ch, a.cl);
      if (D != 0.0f) v = fmaf(D, exp_scaled(t, 1.44269502f, 1.92596303e-8f), v);
      f[e] = v;
    }
    if (j + R::E <= j1) {
      R::store(out, j, R::pack(f));
    } else {
#pragma unroll
      for (int e = 0; e < R::E; e++)
        if (j + e < j1) R::put(out, j + e, f[e]);
    }
  }
  __syncthreads();  // the listed tokens and the label are written over the rows' formula
  if (w == 0.0) return;
  if (first && id >= j0 && id < j1) {
    double v = 0.0;
    if (wT != 0.0) v = wT * (exp(((double)zs - M) * invt) / ZT - pt);
    if (w1 != 0.0) v += w1 * (exp((double)zs - M) / Z1 - (id == tk ? 1.0 : 0.0));
    R::put(out, id, (float)v);
  }
  const bool listed = __syncthreads_or(held && id == tk);
  if (tid == 0 && label && !listed && w1 != 0.0 && tk >= j0 && tk < j1) {
    double v = w1 * (exp((double)zt - M) / Z1 - 1.0);
    if (wT != 0.0) v += wT * exp(((double)zt - M) * invt) / ZT - (pr > 0.0 ? wT * pr * exp(((double)zt - mu) * invt) / sT : 0.0);
    R::put(out, tk, (float)v);
  }
}

#define RTQ_DISTILL(ty, VT)                                                                                     \
  extern "C" __global__ __launch_bounds__(kDisB) void rtq_distill_stats_##ty(DistillArgs a) { distill_stats<VT>(a); } \
  extern "C" __global__ __launch_bounds__(kDisB) void rtq_distill_grad_##ty(DistillArgs a) { distill_grad<VT>(a); }
RTQ_DISTILL(f32, VT_F32)
RTQ_DISTILL(f16, VT_F16)
RTQ_DISTILL(bf16, VT_BF16)

// ============================================================== drafted tokens
// Sequence i: accept its drafted tokens x_0, x_1, ... while u_j q_j(x_j) < p_j(x_j) (p the target's
// softmax(z / T), q the draft's, or all of it on x_j without draft logits); the token after the accepted ones is
// drawn from max(p - q, 0) at the first rejection, from p after all: the first index whose running sum
// passes u_d times the total.  T = 0: accept while x_j is the target's largest logit (the lowest index
// of equals), which is also the token after.  Steps of the running sum over a flat tail lie nearer
// than 2^-24 of the total, so exponentials and sums are in 64 bits.
constexpr int kVdB = 256, kVdW = kVdB / 64;

template <int VT>
__device__ __forceinline__ const void* vd_row(const VerifyArgs& a, bool draft, int64_t row) {
  return static_cast<const char*>(draft ? a.q : a.z) + row * (draft ? a.ldq : a.ld) * VRow<VT>::ES;
}

// grid (G, b (d + 1) + b d): maximum (the lowest index of it) and sum exp((z - max) / T) of a slice of a target
// row, then of the draft rows; rows past a sequence's length are not read
template <int VT>
__device__ __forceinline__ void verify_stats(const VerifyArgs& a) {
  using R = VRow<VT>;
  __shared__ uint64_t redk[kVdW];
  __shared__ double redd[kVdW];
  const int tid = threadIdx.x, g = blockIdx.x;
  const int64_t rr = blockIdx.y + (int64_t)blockIdx.z * 65535, tr = (int64_t)a.b * (a.d + 1);
  if (rr >= tr + (a.q ? (int64_t)a.b * a.d : 0)) return;
  const bool draft = rr >= tr;
  const int64_t row = draft ? rr - tr : rr;
  const int i = (int)(row / (draft ? a.d : a.d + 1)), j = (int)(row % (draft ? a.d : a.d + 1));
  const int len = a.lens ? min(max(a.lens[i], 0), a.d) : a.d;
  if (draft ? j >= len : j > len) return;
  const void* z = vd_row<VT>(a, draft, row);
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);
  uint64_t best = 0;
  for (int v = j0 + tid * R::E; v < j1; v += kVdB * R::E) {
    const u4v r = R::load_upto(z, v, j1, -__builtin_inff());
#pragma unroll
    for (int e = 0; e < R::E; e++) {
      const uint64_t key = v + e < j1 ? rank_key(R::get(r, e), v + e) : 0;
      best = key > best ? key : best;
    }
  }
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(best, m);
    best = o > best ? o : best;
  }
  if ((tid & 63) == 0) redk[tid >> 6] = best;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kVdW; w++) best = redk[w] > best ? redk[w] : best;
  double s = 0.0;
  const double m = (double)key_value(best);
  if (a.temp > 0.0f && m != -__builtin_inf()) {
    const double invt = 1.0 / (double)a.temp;
    for (int v = j0 + tid * R::E; v < j1; v += kVdB * R::E) {
      const u4v r = R::load_upto(z, v, j1, -__builtin_inff());
#pragma unroll
      for (int e = 0; e < R::E; e++) s += exp(((double)R::get(r, e) - m) * invt);
    }
  }
  s = group_sum<kVdW>(s, redd);
  if (tid == 0) a.pk[rr * a.G + g] = best, a.ps[rr * a.G + g] = s;
}

struct VdRow {
  double m, s;
  int best;
};
// a row's maximum and sum from its slices, by one wave
__device__ __forceinline__ VdRow vd_join(const VerifyArgs& a, int64_t rr) {
  const int l = threadIdx.x & 63;
  const double invt = a.temp > 0.0f ? 1.0 / (double)a.temp : 0.0;
  uint64_t best = 0;
  for (int g = l; g < a.G; g += 64) best = a.pk[rr * a.G + g] > best ? a.pk[rr * a.G + g] : best;
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) {
    const uint64_t o = __shfl_xor(best, m);
    best = o > best ? o : best;
  }
  const double m = (double)key_value(best);
  double s = 0.0;
  for (int g = l; g < a.G; g += 64) {
    const double pm = (double)key_value(a.pk[rr * a.G + g]);
    if (pm != -__builtin_inf()) s += a.ps[rr * a.G + g] * exp((pm - m) * invt);
  }
  return VdRow{m, wave_sum_any(s), key_index(best)};
}

// grid b, one wave: how many of sequence i's drafted tokens are accepted, and the row to draw from
template <int VT>
__device__ __forceinline__ void verify_accept(const VerifyArgs& a) {
  using R = VRow<VT>;
  const int i = blockIdx.x, l = threadIdx.x;
  const int len = a.lens ? min(max(a.lens[i], 0), a.d) : a.d;
  const double invt = a.temp > 0.0f ? 1.0 / (double)a.temp : 0.0;
  const int64_t tr = (int64_t)a.b * (a.d + 1);
  int acc = 0;
  VdRow p{}, q{};
  bool rejected = false;
  int x = -1;
  for (; acc <= len; acc++) {
    const int64_t prow = (int64_t)i * (a.d + 1) + acc, qrow = (int64_t)i * a.d + acc;
    p = vd_join(a, prow);
    if (acc == len) break;
    x = a.drafted[qrow];
    const bool in = x >= 0 && x < a.V;
    bool ok;
    if (a.temp > 0.0f) {
      const double px = in ? exp(((double)R::one(vd_row<VT>(a, false, prow), x) - p.m) * invt) / p.s : 0.0;
      double qx = 1.0;
      if (a.q) {
        q = vd_join(a, tr + qrow);
        qx = in ? exp(((double)R::one(vd_row<VT>(a, true, qrow), x) - q.m) * invt) / q.s : 0.0;
      }
      ok = (double)a.u[(int64_t)i * (a.d + 1) + acc] * qx < px;
    } else {
      ok = in && x == p.best;
    }
    if (!ok) {
      rejected = true;
      break;
    }
  }
  for (int j = l; j <= a.d; j += 64)
    a.tokens[(int64_t)i * (a.d + 1) + j] = j < acc ? a.drafted[(int64_t)i * a.d + j] : (j == acc && a.temp == 0.0f) ? p.best : -1;
  if (l == 0) {
    a.accepted[i] = acc;
    VerifyPick v;
    v.pm = p.m, v.ps = 1.0 / p.s, v.qm = q.m, v.qs = rejected && a.q ? 1.0 / q.s : 0.0;
    v.row = acc, v.not_x = rejected && !a.q ? x : -1, v.minus_q = rejected && a.q ? 1 : 0, v.pad = 0;
    a.pick[i] = v;
  }
}

// the weight of token v: max(p - q, 0) after a rejection, or p
__device__ __forceinline__ double vd_weight(const VerifyPick& k, float zp, float zq, int v, double invt, double& p) {
  p = exp(((double)zp - k.pm) * invt) * k.ps;
  if (k.minus_q) return fmax(p - exp(((double)zq - k.qm) * invt) * k.qs, 0.0);
  return v == k.not_x ? 0.0 : p;
}

// grid (G, b): the weights' sum over slice g of sequence i's row, and p's
template <int VT>
__device__ __forceinline__ void verify_mass(const VerifyArgs& a) {
  using R = VRow<VT>;
  __shared__ double redd[kVdW];
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  const VerifyPick k = a.pick[i];
  const void* zp = vd_row<VT>(a, false, (int64_t)i * (a.d + 1) + k.row);
  const void* zq = k.minus_q ? vd_row<VT>(a, true, (int64_t)i * a.d + k.row) : zp;
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);
  const double invt = 1.0 / (double)a.temp;
  double sw = 0.0, sp = 0.0;
  for (int v = j0 + tid * R::E; v < j1; v += kVdB * R::E) {
    const u4v r = R::load_upto(zp, v, j1, -__builtin_inff()), rq = R::load_upto(zq, v, j1, -__builtin_inff());
#pragma unroll
    for (int e = 0; e < R::E; e++) {
      double p;
      sw += vd_weight(k, R::get(r, e), R::get(rq, e), v + e, invt, p);
      sp += p;
    }
  }
  sw = group_sum<kVdW>(sw, redd);
  sp = group_sum<kVdW>(sp, redd);
  if (tid == 0) a.mass[((int64_t)i * a.G + g) * 2] = sw, a.mass[((int64_t)i * a.G + g) * 2 + 1] = sp;
}

// grid b: the slice that holds u_d times the total, then the token in it
template <int VT>
__device__ __forceinline__ void verify_pick(const VerifyArgs& a) {
  using R = VRow<VT>;
  __shared__ double part[kVdB];
  __shared__ int sslice, sall, token;
  __shared__ double starget;
  const int tid = threadIdx.x, i = blockIdx.x;
  VerifyPick k = a.pick[i];
  const double* mass = a.mass + (int64_t)i * a.G * 2;
  if (tid == 0) {
    double tot = 0.0;
    for (int g = 0; g < a.G; g++) tot += mass[2 * g];
    const int all = tot > 0.0 ? 0 : 1;  // p - q is nowhere positive: drawn from p
    if (all) {
      tot = 0.0;
      for (int g = 0; g < a.G; g++) tot += mass[2 * g + 1];
    }
    const double t = (double)a.u[(int64_t)i * (a.d + 1) + a.d] * tot;
    double c = 0.0, before = 0.0;
    int s = -1;
    for (int g = 0; g < a.G; g++) {
      const double w = mass[2 * g + all];
      if (w > 0.0) s = g, before = c;
      c += w;
      if (c > t) break;
    }
    sslice = tot > 0.0 ? s : -1, sall = all, starget = t - before, token = -1;  // NaN: no token
  }
  __syncthreads();
  if (sslice < 0) return;
  if (sall) k.minus_q = 0, k.not_x = -1;
  const void* zp = vd_row<VT>(a, false, (int64_t)i * (a.d + 1) + k.row);
  const void* zq = k.minus_q ? vd_row<VT>(a, true, (int64_t)i * a.d + k.row) : zp;
  const double invt = 1.0 / (double)a.temp;
  const int j0 = sslice * a.L, j1 = min(a.V, j0 + a.L), per = (a.L + kVdB - 1) / kVdB;
  const int v0 = j0 + tid * per, v1 = min(j1, v0 + per);
  auto weight = [&](int v) {
    double p;
    return vd_weight(k, R::one(zp, v), R::one(zq, v), v, invt, p);
  };
  double s = 0.0;
  int last = -1;
  for (int v = v0; v < v1; v++) {
    const double w = weight(v);
    s += w;
    if (w > 0.0) last = v;
  }
  part[tid] = s;
  __syncthreads();
  double before = 0.0;
  for (int q = 0; q < tid; q++) before += part[q];
  // the first thread whose running sum passes the target; rounding may leave none: then the last
  // token of the slice that has weight
  int mine = 1 << 30;
  if (before + s > starget && last >= 0) {
    double c = before;
    for (int v = v0; v < v1; v++) {
      c += weight(v);
      if (c > starget) {
        mine = v;
        break;
      }
    }
    if (mine == 1 << 30) mine = last;
  }
  __shared__ int first, lastw;
  if (tid == 0) first = 1 << 30, lastw = -1;
  __syncthreads();
  atomicMin(&first, mine);
  atomicMax(&lastw, last);
  __syncthreads();
  if (tid == 0) a.tokens[(int64_t)i * (a.d + 1) + k.row] = first < (1 << 30) ? first : lastw;
}

#define RTQ_VERIFY(ty, VT)                                                                                              \
  extern "C" __global__ __launch_bounds__(kVdB) void rtq_verify_stats_##ty(VerifyArgs a) { verify_stats<VT>(a); }       \
  extern "C" __global__ __launch_bounds__(64) void rtq_verify_accept_##ty(VerifyArgs a) { verify_accept<VT>(a); }       \
  extern "C" __global__ __launch_bounds__(kVdB) void rtq_verify_mass_##ty(VerifyArgs a) { verify_mass<VT>(a); }         \
  extern "C" __global__ __launch_bounds__(kVdB) void rtq_verify_pick_##ty(VerifyArgs a) { verify_pick<VT>(a); }
RTQ_VERIFY(f32, VT_F32)
RTQ_VERIFY(f16, VT_F16)
RTQ_VERIFY(bf16, VT_BF16)
