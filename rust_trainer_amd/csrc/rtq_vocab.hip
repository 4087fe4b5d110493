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
  __device__ static __forceinline__ float get_at(const u4v& r, int e) {  // e not known to the compiler
    const int d = VT == VT_F32 ? e : e >> 1;
    const uint32_t u = d == 0 ? r[0] : d == 1 ? r[1] : d == 2 ? r[2] : r[3];
    return get(u4v{u, u, u, u}, VT == VT_F32 ? 0 : e & 1);
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
  // elements j .. j + E - 1 of a row of V; those past its end read as -inf (the rare path is kept small: it
  // stands beside unrolled code)
  __device__ static __forceinline__ u4v load_upto(const void* row, int64_t j, int64_t V) {
    if (j + E <= V) return load(row, j);
    const uint32_t none = VT == VT_F32 ? 0xff800000u : VT == VT_F16 ? 0xfc00fc00u : 0xff80ff80u;
    u4v r = {none, none, none, none};
#pragma unroll 1
    for (int e = 0; j + e < V; e++) {
      const int d = VT == VT_F32 ? e : e >> 1, sh = VT == VT_F32 ? 0 : 16 * (e & 1);
      uint32_t u, keep = 0;
      if constexpr (VT == VT_F32) u = static_cast<const uint32_t*>(row)[j + e];
      else u = (uint32_t) static_cast<const uint16_t*>(row)[j + e] << sh, keep = 0xffff0000u >> sh;
#pragma unroll
      for (int w = 0; w < 4; w++) r[w] = d == w ? (r[w] & keep) | u : r[w];
    }
    return r;
  }
};

// whether row i has logits (rows formed at positions: the position is one of the sequence's)
template <class Args>
__device__ __forceinline__ bool row_ok(const Args& a, int i) {
  return !a.pos || (a.pos[i] >= 0 && a.pos[i] < a.t);
}

// the value of lane ^ J (J = 1, 2, 4, 8 by DPP controls within rows of 16 lanes)
template <int J>
__device__ __forceinline__ float lane_xor(float v) {
  if constexpr (J == 1) return dpp_f<0xB1>(v);
  else if constexpr (J == 2) return dpp_f<0x4E>(v);
  else if constexpr (J == 4) return dpp_f<0x1B>(dpp_f<0x141>(v));  // mirrored in eight, then in four
  else if constexpr (J == 8) return dpp_f<0x128>(v);               // rotated by eight
  else return __shfl_xor(v, J);
}
template <int J>
__device__ __forceinline__ double lane_xor(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = __builtin_bit_cast(uint32_t, lane_xor<J>(__builtin_bit_cast(float, (uint32_t)u)));
  const uint32_t hi = __builtin_bit_cast(uint32_t, lane_xor<J>(__builtin_bit_cast(float, (uint32_t)(u >> 32))));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}

// a barrier that orders LDS alone: loads and stores of memory stay in flight across it
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <class T>
__device__ __forceinline__ T wave_sum_any(T v) {
  v += lane_xor<1>(v);
  v += lane_xor<2>(v);
  v += lane_xor<4>(v);
  v += lane_xor<8>(v);
  v += lane_xor<16>(v);
  return v + lane_xor<32>(v);
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
__device__ __forceinline__ float wave_max_any(float v) {
  v = fmaxf(v, lane_xor<1>(v));
  v = fmaxf(v, lane_xor<2>(v));
  v = fmaxf(v, lane_xor<4>(v));
  v = fmaxf(v, lane_xor<8>(v));
  v = fmaxf(v, lane_xor<16>(v));
  return fmaxf(v, lane_xor<32>(v));
}
template <int W>
__device__ __forceinline__ float group_max(float v, float* red) {
  v = wave_max_any(v);
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

__device__ __forceinline__ float lse_of(float m, double s, double invt) {  // s is NaN for a NaN alone
  if (s != s) return __builtin_nanf("");
  return fabsf(m) == __builtin_inff() ? m : (float)((double)m * invt + log(s));
}

// maximum / sum over each eight neighbouring lanes; every lane gets it
__device__ __forceinline__ float oct_max(float v) {
  v = fmaxf(v, dpp_f<0xB1>(v));
  v = fmaxf(v, dpp_f<0x4E>(v));
  return fmaxf(v, dpp_f<0x141>(v));
}
__device__ __forceinline__ float oct_sum(float v) {
  v += dpp_f<0xB1>(v);
  v += dpp_f<0x4E>(v);
  return v + dpp_f<0x141>(v);
}

// lane i's value of the wave's 64 sorted from the largest (a bitonic network; K: sorted runs, J: distance)
template <int K, int J>
__device__ __forceinline__ float sort_step(float v) {
  const int l = threadIdx.x & 63;
  const float o = lane_xor<J>(v);
  const bool up = ((l & K) == 0) == ((l & J) == 0);  // this lane keeps the larger
  v = up ? fmaxf(v, o) : fminf(v, o);
  if constexpr (J > 1) return sort_step<K, J / 2>(v);
  else if constexpr (K < 64) return sort_step<K * 2, K>(v);
  else return v;
}
__device__ __forceinline__ float wave_sort(float v) { return sort_step<2, 1>(v); }

// The row is read once, by groups of eight lanes' vectors (32 f32 or 64 16-bit logits, contiguous):
// of each group its maximum and the sum of exp((z - maximum) / T) are kept.  The k largest logits lie
// in the k groups of the largest maxima, so rtq_top_pick_* reads only those again; every other group
// enters the rest as a whole, so that nothing is subtracted.  A group that holds a NaN has maximum NaN.
//
// grid (chunks / 4, n), a wave per chunk of 64 groups: kTopU vectors a lane, all loaded at once
constexpr int kTopU = 8;

template <int VT>
__device__ __forceinline__ void top_scan(const TopArgs& a) {
  using R = VRow<VT>;
  constexpr int E = R::E, C = 64 * E * kTopU;
  const int l = threadIdx.x & 63, i = blockIdx.y;
  const int q = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (q * 64 >= a.NG || !row_ok(a, i)) return;
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  const float ninf = -__builtin_inff();
  const int j0 = q * C + l * E;
  u4v raw[kTopU];
  if ((q + 1) * C <= a.V) {
#pragma unroll
    for (int u = 0; u < kTopU; u++) raw[u] = R::load(row, j0 + u * 64 * E);
  } else {
#pragma unroll
    for (int u = 0; u < kTopU; u++) raw[u] = R::load_upto(row, j0 + u * 64 * E, a.V);
  }
  float gm = ninf, gs = 0.0f;
#pragma unroll
  for (int u = 0; u < kTopU; u++) {
    float m = R::get(raw[u], 0);
#pragma unroll
    for (int e = 1; e < E; e++) m = fmaxf(m, R::get(raw[u], e));
    m = oct_max(m);
    const float ref = m == ninf ? 0.0f : m;
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) s += __builtin_amdgcn_exp2f((R::get(raw[u], e) - ref) * a.c);
    s = oct_sum(s);
    if (__ballot(s != s)) {  // a NaN, or infinity less itself
      float bad = 0.0f;
#pragma unroll
      for (int e = 0; e < E; e++) bad = R::get(raw[u], e) != R::get(raw[u], e) ? 1.0f : bad;
      if (oct_max(bad) > 0.0f) m = __builtin_nanf("");
    }
    gm = (l & 7) == u ? m : gm;
    gs = (l & 7) == u ? s : gs;
  }
  const int64_t o = (int64_t)i * a.NG + q * 64 + (l & 7) * 8 + (l >> 3);
  a.gm[o] = gm;
  a.gs[o] = gs;
}

// the K-th largest of the keys f(0) .. f(N - 1) (0: none; the others differ), eight bits at a time
template <int B, class F>
__device__ __forceinline__ uint64_t radix_kth(int N, int K, int* hist, int* out, F&& f) {
  const int tid = threadIdx.x;
  uint64_t low = 0, mask = 0;
  int need = K;
  for (int sh = 56; sh >= 0; sh -= 8) {
    for (int b = tid; b < 256; b += B) hist[b] = 0;
    __syncthreads();
    for (int p = tid; p < (N + 63) / 64 * 64; p += B) {
      const uint64_t key = p < N ? f(p) : 0;
      const bool in = key != 0 && (key & mask) == low;
      const int d = (int)(key >> sh) & 255;
      // a wave's equal digits (ties, the index's upper digits) are counted with one atomic
      const uint64_t m = __ballot(in);
      if (m == 0) continue;
      const int lead = __builtin_ctzll(m);
      if (__ballot(in && d != __shfl(d, lead)) == 0) {
        if ((tid & 63) == lead) atomicAdd(&hist[d], __popcll(m));
      } else if (in) {
        atomicAdd(&hist[d], 1);
      }
    }
    __syncthreads();
    if (tid < 64) {  // lane l: bins 4 l .. 4 l + 3; the bin where the count from the top reaches `need`
      int h[4], s = 0;
#pragma unroll
      for (int b = 0; b < 4; b++) h[b] = hist[4 * tid + b], s += h[b];
      int above = s;  // of this lane and all above it
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) {
        const int o = __shfl_down(above, d);
        above += tid + d < 64 ? o : 0;
      }
      above -= s;
#pragma unroll
      for (int b = 3; b >= 0; b--) {
        if (above < need && need <= above + h[b]) out[0] = 4 * tid + b, out[1] = above, out[2] = h[b];
        above += h[b];
      }
    }
    __syncthreads();
    need -= out[1];
    low |= (uint64_t)out[0] << sh;
    mask |= (uint64_t)255 << sh;
    if (out[2] == need) return low;  // the whole bin belongs
  }
  return low;
}

// (m, s) of a set joined by N others: x[e] with exponential sum w[e] (0: no member).  A NaN makes s NaN, and
// nothing else does: beside +inf nothing is summed
template <int N>
__device__ __forceinline__ void join_rest(float& m, double& s, const float* x, const float* w, const TopArgs& a) {
  float b = m;
  bool nan = false;
#pragma unroll
  for (int e = 0; e < N; e++) {
    b = fmaxf(b, w[e] != 0.0f ? x[e] : b);
    nan |= w[e] != 0.0f && x[e] != x[e];
  }
  if (nan) s = (double)__builtin_nanf("");
  if (b == -__builtin_inff()) return;
  if (b > m) {
    s *= (double)__builtin_amdgcn_exp2f((m - b) * a.c);
    m = b;
  }
  if (b == __builtin_inff()) return;
  float t = 0.0f;
#pragma unroll
  for (int e = 0; e < N; e++) t += w[e] != 0.0f ? w[e] * __builtin_amdgcn_exp2f((x[e] - m) * a.c) : 0.0f;
  s += (double)t;
}

// grid n: row i's k largest logits and the rest's log-sum-exp, from its groups.  A bound
// below the k-th largest comes from the threads' maxima over the groups: with r = ceil(k / waves),
// every wave has r at or above its own r-th, so the least of those r-ths has k logits at or above
// it.  The groups that reach it (1.5 to 4 k of them in a row without structure) are read again, and what
// reaches it there is ranked by counting.  Where too many do, a second bound comes from the
// logits of those groups; where that does not help either (ties, masks, sorted rows), exactly the k
// groups and then exactly the k logits are found digit by digit.  512 threads: alone on the chip 8.9 us
// at k = 20 of 151936 f32 logits, and 36 us for 1024 rows at k = 128 (lists filled by atomics took 8.4 and 38.8,
// 9.5 and 40.9 with 256 threads, 10.2 and 67.6 with 1024).
constexpr int kPickB = 512;

template <int VT>
__device__ __forceinline__ void top_pick(const TopArgs& a) {
  using R = VRow<VT>;
  constexpr int E = R::E, GS = 8 * E, B = kPickB, W = B / 64, CAP = 4 * B, U = 5120 / B, UE = 4;
  __shared__ uint64_t cand[CAP];
  __shared__ alignas(16) uint32_t list[CAP];
  __shared__ float redf[W];
  __shared__ double redd[W];
  __shared__ int hist[256];
  __shared__ int out[3];
  __shared__ alignas(16) int wsum[2][W];
  __shared__ int fewer;
  const int tid = threadIdx.x, l = tid & 63, i = blockIdx.x;
  const float ninf = -__builtin_inff(), inf = __builtin_inff();
  if (!row_ok(a, i)) {
    for (int s = tid; s < a.k; s += B) a.vals[(int64_t)i * a.k + s] = __builtin_nanf(""), a.ids[(int64_t)i * a.k + s] = -1;
    if (tid == 0 && a.rest) a.rest[i] = __builtin_nanf("");
    return;
  }
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  const float* gm = a.gm + (int64_t)i * a.NG;
  const float* gs = a.gs + (int64_t)i * a.NG;
  const int held = (a.V + GS - 1) / GS;  // groups with a logit
  // the least over the first n / 64 waves (those whose lanes all have a maximum) of their r-ths
  auto bound = [&](float lm, int n) {
    const int full = min(W, n / 64), r = full ? (a.k + full - 1) / full : 65;
    const float ws = wave_sort(lm);
    if (l == r - 1) redf[tid >> 6] = ws;
    __syncthreads();
    float t = r > 64 ? ninf : redf[0];
    for (int w = 1; w < full; w++) t = r > 64 ? ninf : fminf(t, redf[w]);
    return t;
  };
  // this thread's first place for n entries of a list that has `all` so far, by thread (not in order of arrival: which
  // thread joins what to the rest decides its last bits); called by all threads.  Two buffers, so that one barrier will do
  int cnt = 0, groups = 0, turn = 0;
  auto places = [&](int n, int& all) {  // n <= 32
    int at = all, sum = 0;
#pragma unroll
    for (int b = 0; b < 6; b++) {  // the lanes below and all, by the digits of n
      const uint64_t m = __ballot((n >> b) & 1);
      at += (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0)) << b;
      sum += __popcll(m) << b;
    }
    if (l == 0) wsum[turn][tid >> 6] = sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; w++) {
      const int o = wsum[turn][w];
      at += w < tid >> 6 ? o : 0;
      all += o;
    }
    turn ^= 1;
    return at;
  };
  // the first U B groups stay in registers (V up to 163840 f32 or 327680 16-bit logits: all of them)
  float m0[U], s0[U];
  auto load_groups = [&](int g0, float* m, float* s) {
#pragma unroll
    for (int u = 0; u < U; u++) m[u] = g0 + u * B < held ? gm[g0 + u * B] : ninf;
#pragma unroll
    for (int u = 0; u < U; u++) s[u] = g0 + u * B < held && a.rest ? gs[g0 + u * B] : 0.0f;
  };
  auto largest = [&](const float* m) {
    float x = ninf;
#pragma unroll
    for (int u = 0; u < U; u++) x = fmaxf(x, m[u] != m[u] ? inf : m[u]);
    return x;
  };
  load_groups(tid, m0, s0);
  float lm = largest(m0);
  for (int g0 = tid + U * B; g0 < held; g0 += U * B) {
    float m[U], s[U];
    load_groups(g0, m, s);
    lm = fmaxf(lm, largest(m));
  }
  float thr = bound(lm, held);
  float rm = ninf;
  double rs = 0.0;
  // the groups in(m, g) takes go to the list, the others to the rest
  auto choose = [&](bool kept, auto&& in) {
    auto some = [&](int g0, const float* m, const float* s) {
      float w[U];
      uint32_t bits = 0;
#pragma unroll
      for (int u = 0; u < U; u++) {
        const bool c = g0 + u * B < held && in(m[u], g0 + u * B);
        bits |= c ? 1u << u : 0u;
        w[u] = c ? 0.0f : s[u];
      }
      int at = places(__popc(bits), groups);
      for (; bits; bits &= bits - 1, at++)
        if (at < CAP) list[at] = (uint32_t)(g0 + (__ffs(bits) - 1) * B);
      if (a.rest) join_rest<U>(rm, rs, m, w, a);
    };
    if (kept) some(tid, m0, s0);
    for (int b0 = kept ? U * B : 0; b0 < held; b0 += U * B) {
      float m[U], s[U];
      load_groups(b0 + tid, m, s);
      some(b0 + tid, m, s);
    }
  };
  choose(true, [&](float m, int) { return !(m < thr); });
  __syncthreads();
  // the listed groups' logits, UE vectors a thread at a time, all threads together: f(vectors, indexes of their
  // first); past the list's end the index is V or above
  auto each = [&](auto&& f) {
    const int n = groups * 8;
    for (int b0 = 0; b0 < n; b0 += B * UE) {
      u4v v[UE];
      int j[UE];
#pragma unroll
      for (int u = 0; u < UE; u++) {
        const int p = b0 + tid + u * B;
        j[u] = p < n ? (int)list[p >> 3] * GS + (p & 7) * E : a.V;
      }
#pragma unroll
      for (int u = 0; u < UE; u++) {
        v[u] = u4v{0, 0, 0, 0};
        if (j[u] < a.V) v[u] = R::load_upto(row, j[u], a.V);
      }
      f(v, j);
    }
  };
  // the logits that in(x, index) takes are the candidates, the others go to the rest
  auto collect = [&](auto&& in) {
    each([&](const u4v* v, const int* j) {
      uint32_t bits = 0;  // E for each vector
#pragma unroll
      for (int u = 0; u < UE; u++) {
        if (j[u] >= a.V) continue;
        float x[E], w[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
          x[e] = R::get(v[u], e);
          const bool c = j[u] + e < a.V && in(x[e], j[u] + e);
          bits |= c ? 1u << (u * E + e) : 0u;
          w[e] = j[u] + e < a.V && !c ? 1.0f : 0.0f;
        }
        if (a.rest) join_rest<E>(rm, rs, x, w, a);
      }
      int at = places(__popc(bits), cnt);
#pragma unroll
      for (int u = 0; u < UE; u++) {
        const uint32_t mine = bits >> (u * E) & ((1u << E) - 1);
        if (!mine) continue;
#pragma unroll
        for (int e = 0; e < E; e++)
          if ((mine >> e) & 1) {
            if (at < CAP) cand[at] = rank_key(R::get(v[u], e), j[u] + e);
            at++;
          }
      }
    });
    __syncthreads();
  };
  const float gm_rest = rm;
  const double gs_rest = rs;
  bool many = groups > CAP;
  if (!many) {
    // a bound from the listed groups' logits, where the groups gave none (few of them hold a row of a small
    // vocabulary) or too much reaches it: places are found by counting, n of n candidates each
    auto refine = [&]() {
      float em = ninf;
      each([&](const u4v* v, const int* j) {
#pragma unroll
        for (int u = 0; u < UE; u++)
#pragma unroll
          for (int e = 0; e < E; e++) em = j[u] + e < a.V ? fmaxf(em, R::get(v[u], e) != R::get(v[u], e) ? inf : R::get(v[u], e)) : em;
      });
      thr = fmaxf(thr, bound(em, groups * 8));
    };
    const bool none = thr == ninf && groups * GS > 2 * a.k + 128;
    if (none) refine();
    collect([&](float x, int) { return !(x < thr); });
    if (!none && cnt > 4 * a.k + 256) {
      refine();
      cnt = 0;
      rm = gm_rest, rs = gs_rest;
      collect([&](float x, int) { return !(x < thr); });
    }
    many = cnt > CAP;
  }
  if (many) {
    auto group_key = [&](float m, int g) { return rank_key(m, g); };
    const uint64_t gk = radix_kth<B>(held, min(a.k, held), hist, out, [&](int g) { return group_key(gm[g], g); });
    cnt = 0, groups = 0;
    rm = ninf, rs = 0.0;
    choose(false, [&](float m, int g) { return group_key(m, g) >= gk; });  // min(k, held) of them
    __syncthreads();
    const uint64_t ek = radix_kth<B>(groups * GS, a.k, hist, out, [&](int p) {
      const int j = (int)list[p / GS] * GS + p % GS;
      return j < a.V ? rank_key(R::one(row, j), j) : 0ull;
    });
    collect([&](float x, int j) { return rank_key(x, j) >= ek; });  // k of them
  }
  // Many candidates more than k (a small vocabulary, of which k is a large part): first exactly the k, found digit
  // by digit (2000 rows of 1000 f32 logits, k = 256: 61 us, 172 by counting all of them).
  const uint64_t* best = cand;
  int n = cnt;
  if (n > 2 * a.k + 128) {
    const uint64_t kth = radix_kth<B>(n, a.k, hist, out, [&](int p) { return cand[p]; });
    uint64_t* few = reinterpret_cast<uint64_t*>(list);
    if (tid == 0) fewer = 0;
    __syncthreads();
    for (int p = tid; p < n; p += B) {
      const uint64_t key = cand[p];
      if (key >= kth) {
        few[atomicAdd(&fewer, 1)] = key;  // (their places go by their keys)
      } else if (a.rest) {
        const float x = key_value(key), w = 1.0f;
        join_rest<1>(rm, rs, &x, &w, a);
      }
    }
    __syncthreads();
    best = few, n = a.k;
  }
  // a candidate's place is the number of larger ones
  const int n8 = (n + 7) & ~7;
  if (tid < n8 - n) const_cast<uint64_t*>(best)[n + tid] = 0;
  __syncthreads();
  for (int p = tid; p < n; p += B) {
    const uint64_t key = best[p];
    int place = 0;
    for (int q = 0; q < n8; q += 8)
#pragma unroll
      for (int e = 0; e < 8; e++) place += best[q + e] > key;
    if (place < a.k) {
      a.vals[(int64_t)i * a.k + place] = key_value(key);
      a.ids[(int64_t)i * a.k + place] = key_index(key);
    } else if (a.rest) {
      const float x = key_value(key), w = 1.0f;
      join_rest<1>(rm, rs, &x, &w, a);
    }
  }
  if (!a.rest) return;
  const float m = group_max<W>(rm, redf);
  rs = group_sum<W>(rm == m || rm == ninf ? rs : rs * (double)__builtin_amdgcn_exp2f((rm - m) * a.c), redd);
  if (tid == 0) a.rest[i] = lse_of(m, rs, 1.0 / (double)a.temp);
}

#define RTQ_TOP(ty, VT)                                                                                    \
  extern "C" __global__ __launch_bounds__(256) void rtq_top_scan_##ty(TopArgs a) { top_scan<VT>(a); }      \
  extern "C" __global__ __launch_bounds__(kPickB, 4) void rtq_top_pick_##ty(TopArgs a) { top_pick<VT>(a); }
RTQ_TOP(f32, VT_F32)
RTQ_TOP(f16, VT_F16)
RTQ_TOP(bf16, VT_BF16)

// ============================================================== distillation
// Row i: the teacher's distribution p over its listed tokens and the rest (one bucket), the student's
// q = softmax(z / T) over the same buckets.  The unlisted logits have their own maximum mu and sums
// sT = sum exp((z - mu) / T), s1 = sum exp(z - mu), so the rest's probability is no difference of two
// sums.  Gradient at an unlisted token: C exp((z - mu) / T) + D exp(z - mu) with one C and D a row; the
// listed tokens and the label are written over it.
//
// rtq_distill*_<type>: a row a workgroup, whose first wave does the row's scalars (the teacher's list, the
// losses, the gradient at the listed tokens) while the others hold their first kDisV vectors a thread in
// registers and the next kDisL in LDS from the statistics to the gradient: one read and one write of the row
// (what a longer row has beyond them is read twice: of 151936 f32 logits 39%, of 16 bits none).  2048 rows of 151936
// bf16 take 292 us, 4.3 TB/s; 256 of f32 83 us, 4.5 TB/s with the second read.
// rtq_distill_stats_* / _grad_* do the two halves for slices, of few long rows or without a gradient.
//
// Exponentials are exp2(fma(z, c, -K)), one FMA and the instruction: c = log2(e) / T rounded to f32, and a
// maximum m's reference is f32(m c), so that its rounding cancels between the sums and what is divided by
// them; an exponential below the maximum is off by 2^-24 of its argument for c's rounding.  The row's scalars are
// in 64 bits with log2(e) / T itself, so a large divergence carries none of that.
constexpr int kDisL = 8;
template <int VT>
constexpr int kDisV = VT == VT_F32 ? 16 : 14;  // as many as leave the sums their registers (4 waves a SIMD)

constexpr float kLog2eF = 1.44269502f;  // the f32 nearest log2(e)
constexpr double kLog2eD = 1.4426950408889634074;
constexpr double kLn2D = 0.69314718055994530942;

struct DisShared {
  int id[RTQ_TOP_MAX];     // the slots' tokens (-1: empty)
  float tv[RTQ_TOP_MAX];   // their logits: the teacher's, the student's
  float zs[RTQ_TOP_MAX];
  double p[RTQ_TOP_MAX];   // the teacher's probability, and its sum over the slots of the token
  double pt[RTQ_TOP_MAX];
  int first[RTQ_TOP_MAX];  // the slot stands for its token
  float wm[16];            // the waves' maxima and sums
  double wT[16], w1[16];
  // the row's scalars: C and D with the unlisted logits' references, the student's two normalisers
  // (2^tT sum at the list's scale and 2^t1 sum, kept apart: beside a maximum of -1e9 log2 of the sum would be lost)
  float C, D, KT, K1, base;
  double tT, LT, t1, L1, lu, pr, wgT, wg1;  // LT, L1: log2 of those sums; lu: log2 of the unlisted one's less tT
  float zt;
  int tok, taught;
  // log2 of a logit's probability
  __device__ __forceinline__ double log_qT(float z, double c) const { return ((double)z * c - tT) - LT; }
  __device__ __forceinline__ double log_q1(float z) const { return ((double)z * kLog2eD - t1) - L1; }
};

// a maximum's reference: K = f32(m c) for z c - K, or, where that product's rounding could overflow an exponential
// (masks of -1e9 and below: |m| c > 2^26 = big c, its last place 8), m itself for (z - m) c
__device__ __forceinline__ bool huge(float m, float big) { return fabsf(m) > big; }
__device__ __forceinline__ float ref_base(float m, float big) { return huge(m, big) && fabsf(m) < __builtin_inff() ? m : 0.0f; }
__device__ __forceinline__ float ref_of(float m, float c, float big) { return m == -__builtin_inff() || ref_base(m, big) != 0.0f ? 0.0f : m * c; }
__device__ __forceinline__ double ref_in(float m, float c, float big) { return (double)ref_base(m, big) * (double)c + (double)ref_of(m, c, big); }
// the same for the scale itself, of which c is the float: sums by the reference of m are 2^-(this) of those of exp2(z scale)
__device__ __forceinline__ double ref_exact(float m, float c, double scale, float big) {
  return ref_base(m, big) != 0.0f ? (double)m * scale : (double)ref_of(m, c, big) + (double)m * (scale - (double)c);
}
__device__ __forceinline__ float exp_ref(float z, float c, float K) { return __builtin_amdgcn_exp2f(fmaf(z, c, -K)); }

// which logits of a slice are listed: a bit each, and for every wave a bit per vector of its registers that
// holds one
template <int ST, int NV, int E>
struct DisMarks {
  uint32_t* mask;
  uint32_t* any;  // [ST / 64]
  // by all threads; a barrier follows
  __device__ __forceinline__ void clear(int len) {
    for (int w = threadIdx.x; w < len / 32 + 1; w += blockDim.x) mask[w] = 0;
    if (threadIdx.x < ST / 64) any[threadIdx.x] = 0;
  }
  __device__ __forceinline__ bool set(int o) {  // whether it was
    const int v = o / (ST * E);
    if (v < NV) atomicOr(&any[o % (ST * E) / (64 * E)], 1u << v);
    const uint32_t bit = 1u << (o & 31);
    return (atomicOr(&mask[o >> 5], bit) & bit) != 0;
  }
  __device__ __forceinline__ bool get(int o) const { return (mask[o >> 5] >> (o & 31)) & 1; }
  __device__ __forceinline__ uint32_t vec(int o) const { return mask[o >> 5] >> (o & 31); }  // the low E: of vector o / E
};

// a set of logits: their maximum and their two sums, by the references of that maximum
struct DisSum {
  float m = -__builtin_inff();
  double sT = 0.0, s1 = 0.0;
  __device__ __forceinline__ void raise(float m2, const DistillArgs& a) {  // to the reference of m2 >= m
    const bool none = m == -__builtin_inff();  // (a NaN sum stays)
    sT *= none ? 0.0 : (double)__builtin_amdgcn_exp2f((float)(ref_in(m, a.c, a.big) - ref_in(m2, a.c, a.big)));
    s1 *= none ? 0.0 : (double)__builtin_amdgcn_exp2f((float)(ref_in(m, kLog2eF, a.big) - ref_in(m2, kLog2eF, a.big)));
    m = m2;
  }
  // joined over the lanes of a wave; every lane gets it
  __device__ __forceinline__ void join_wave(const DistillArgs& a) {
    const float M = wave_max_any(m);
    if (m != M) raise(M, a);
    sT = wave_sum_any(sT);
    s1 = wave_sum_any(s1);
  }
};

// A slice [j0, j1) over ST threads (st: 0 .. ST - 1): of the vectors that a whole wave has, the first NV a thread
// stay in registers and the next NL in LDS; the others are read from memory where they are used.  The code for
// registers is unrolled, so what is rare goes another way: marked logits become -inf in the registers, and the
// gradient is written over them afterwards.
template <int VT, int ST, int NV, int NL>
struct DisSlice {
  using R = VRow<VT>;
  using Marks = DisMarks<ST, NV, R::E>;
  static constexpr int E = R::E, GV = 2, MV = 4;  // GV: vectors summed together, MV: loaded together from memory
  static_assert(NV % GV == 0 && MV % GV == 0, "whole groups");
  u4v raw[NV];
  u4v* lds;  // [NL][ST]
  int j0, j1, st, wave, held, kept;  // wave: the wave's first st; its vectors in registers; those and in LDS

  __device__ __forceinline__ void init(int j0_, int j1_, int st_, u4v* lds_) {
    j0 = j0_, j1 = j1_, st = st_, lds = lds_;
    wave = __builtin_amdgcn_readfirstlane(st_ & ~63);
    const int first = (wave + 64) * E, len = j1 - j0;
    const int full = len >= first ? (len - first) / (ST * E) + 1 : 0;
    held = min(NV, full);
    kept = min(NV + NL, full);
  }
  __device__ __forceinline__ int place(int v) const { return j0 + (v * ST + st) * E; }
  // (no branch between the loads, so that each is waited for by itself while the sums run: the first one again
  // instead of one that the row has not.  2048 rows of 151936 bf16: 337 -> 295 us)
  __device__ __forceinline__ void load(const void* row) {
    if (!held) return;
    const uint32_t at = place(0) * R::ES;
#pragma unroll
    for (int v = 0; v < NV; v++) raw[v] = R::load(static_cast<const char*>(row) + (v < held ? v * ST * 16 : 0) + at, 0);
  }
  // v with its marked elements at -inf
  __device__ __forceinline__ static u4v unmarked(u4v v, uint32_t bits) {
#pragma unroll
    for (int d = 0; d < 4; d++) {
      const uint32_t none = VT == VT_F32 ? 0xff800000u : VT == VT_F16 ? 0xfc00fc00u : 0xff80ff80u;
      uint32_t m;
      if constexpr (VT == VT_F32) m = 0u - ((bits >> d) & 1);
      else m = ((0u - ((bits >> (2 * d)) & 1)) & 0xffffu) | (0u - ((bits >> (2 * d + 1)) & 1)) << 16;
      v[d] = (v[d] & ~m) | (none & m);
    }
    return v;
  }
  __device__ __forceinline__ static void add(DisSum& d, const DistillArgs& a, const u4v* x, bool two) {
    float f[GV][E], m = d.m;
#pragma unroll
    for (int v = 0; v < GV; v++)
#pragma unroll
      for (int e = 0; e < E; e++) f[v][e] = R::get(x[v], e), m = fmaxf(m, f[v][e]);
    const float old = d.m == -__builtin_inff() ? m : d.m;  // without logits so far the reference is m's own
    const bool odd = __ballot(huge(m, a.big) || huge(old, a.big)) != 0;
    if (odd) {
      const float b = ref_base(m, a.big);
#pragma unroll
      for (int v = 0; v < GV; v++)
#pragma unroll
        for (int e = 0; e < E; e++) f[v][e] -= b;
    }
    auto sum = [&](double& s, float c) {
      const float K = ref_of(m, c, a.big);
      float t[GV];
#pragma unroll
      for (int v = 0; v < GV; v++) {
        float y[E];
#pragma unroll
        for (int e = 0; e < E; e++) y[e] = exp_ref(f[v][e], c, K);
#pragma unroll
        for (int w = E / 2; w >= 1; w /= 2)
#pragma unroll
          for (int e = 0; e < w; e++) y[e] += y[e + w];
        t[v] = y[0];
        __builtin_amdgcn_sched_barrier(0);  // a vector at a time: the registers hold the row
      }
      float up = ref_of(old, c, a.big) - K;
      if (odd) up = (float)(ref_in(old, c, a.big) - ref_in(m, c, a.big));
      s = fma(s, (double)__builtin_amdgcn_exp2f(up), (double)(t[0] + t[1]));
    };
    sum(d.sT, a.c);
    if (two) sum(d.s1, kLog2eF);
    d.m = m;
  }
  // the statistics of the unmarked logits, into LDS a wave
  __device__ __forceinline__ void stats(const DistillArgs& a, DisShared& sh, const void* row, const Marks& mk) {
    const float ninf = -__builtin_inff();
    const bool two = a.tok && a.temp != 1.0f;  // s1 is a sum of its own
    const uint32_t any = __builtin_amdgcn_readfirstlane(mk.any[wave >> 6]);
    float nothing[E];
#pragma unroll
    for (int e = 0; e < E; e++) nothing[e] = ninf;
    const u4v none = R::pack(nothing);
    DisSum d;
#pragma unroll
    for (int g = 0; g < NV; g += GV) {
      if (g >= held) break;
#pragma unroll
      for (int v = g; v < g + GV; v++) {
        if (v >= held) raw[v] = none;
        else if ((any >> v) & 1) raw[v] = unmarked(raw[v], mk.vec(place(v) - j0));
      }
      add(d, a, &raw[g], two);
    }
    for (int j = place(held); j < j1; j += MV * ST * E) {  // beyond the registers
      u4v x[MV];
#pragma unroll
      for (int v = 0; v < MV; v++) {
        const int o = j + v * ST * E;
        x[v] = o < j1 ? R::load_upto(row, o, j1) : none;
      }
#pragma unroll
      for (int v = 0; v < MV; v++) {
        const int o = j + v * ST * E;
        const uint32_t bits = o < j1 ? mk.vec(o - j0) & ((1u << E) - 1) : 0u;
        if (bits) x[v] = unmarked(x[v], bits);
      }
      if (NL > 0 && j - st * E - j0 < kept * ST * E) {  // (whole waves of vectors: the same for all lanes)
        const int at = (j - st * E - j0) / (ST * E);
#pragma unroll
        for (int v = 0; v < MV; v++)
          if (at + v < kept) lds[(at + v - held) * ST + st] = x[v];
      }
#pragma unroll
      for (int v = 0; v < MV; v += GV) add(d, a, x + v, two);
    }
    if (!two) d.s1 = d.sT;
    d.join_wave(a);
    if ((st & 63) == 0) sh.wm[st >> 6] = d.m, sh.wT[st >> 6] = d.sT, sh.w1[st >> 6] = d.s1;
  }
  // the row's formula.  MODE 0: zeros, 1: C exp2(c z - K), 2: that and D's
  template <int MODE>
  __device__ __forceinline__ void write(void* out, const void* row, float C, float c, float K, float D, float K1, float sub) {
    auto grad = [&](const u4v& x, float base) {
      float f[E];
#pragma unroll
      for (int e = 0; e < E; e++) {
        const float z = base != 0.0f ? R::get(x, e) - base : R::get(x, e);
        f[e] = MODE == 0 ? 0.0f : C * exp_ref(z, c, K);
        if constexpr (MODE == 2) f[e] = fmaf(D, exp_ref(z, kLog2eF, K1), f[e]);
      }
      return R::pack(f);
    };
    if (sub != 0.0f) held = kept = 0;  // from memory
    void* p = static_cast<char*>(out) + (int64_t)place(0) * R::ES;
#pragma unroll
    for (int v = 0; v < NV; v++)
      if (v < held) R::store(p, v * ST * E, grad(raw[v], 0.0f));
    for (int v = held; v < kept; v++) R::store(p, v * ST * E, grad(lds[(v - held) * ST + st], 0.0f));
    for (int j = place(kept); j < j1; j += MV * ST * E) {
      u4v x[MV];
#pragma unroll
      for (int v = 0; v < MV; v++) {
        const int o = j + v * ST * E;
        if (o < j1) x[v] = R::load_upto(row, o, j1);
      }
#pragma unroll
      for (int v = 0; v < MV; v++) {
        const int o = j + v * ST * E;
        if (o >= j1) break;
        const u4v y = grad(x[v], sub);
        if (o + E <= j1) {
          R::store(out, o, y);
        } else {
#pragma unroll 1
          for (int e = 0; o + e < j1; e++) R::put(out, o + e, R::get_at(y, e));
        }
      }
    }
  }
  __device__ __forceinline__ void write(const DistillArgs& a, const DisShared& sh, const void* row, void* out) {
    const float C = sh.C, D = sh.D;
    if (C == 0.0f && D == 0.0f) return write<0>(out, row, 0, 0, 0, 0, 0, 0);
    const bool one = D == 0.0f || C == 0.0f || a.temp == 1.0f, label = one && C == 0.0f;
    if (one) write<1>(out, row, C + D, label ? kLog2eF : a.c, label ? sh.K1 : sh.KT, 0, 0, sh.base);
    else write<2>(out, row, C, a.c, sh.KT, D, sh.K1, sh.base);
  }
};

struct DisTeacher {
  float ml;       // the largest of the student's listed logits
  double ZT, Z1;  // their sums of exp2((z - ml) c) at the two temperatures, each token once
  bool nan;       // one of them is
};

// By one wave, before the statistics are there: the teacher's distribution (sh.p by slots, sh.pt and sh.first by
// tokens, sh.pr, sh.taught) and the student's listed tokens.
__device__ __forceinline__ void distill_teacher(const DistillArgs& a, DisShared& sh, int i, bool twice, DisTeacher& st) {
  const int l = threadIdx.x & 63;
  const float ninf = -__builtin_inff();
  const double invt = 1.0 / (double)a.temp, rest = a.rest ? (double)a.rest[i] : -__builtin_inf();
  float tm = ninf;
  st.ml = ninf;
  bool nant = rest != rest;
  st.nan = false;
  for (int s = l; s < a.k; s += 64) {
    const float tv = sh.tv[s], zs = sh.id[s] >= 0 ? sh.zs[s] : ninf;
    tm = fmaxf(tm, tv);
    st.ml = fmaxf(st.ml, zs);
    nant |= tv != tv;
    st.nan |= zs != zs;
  }
  const double tmax = fmax((double)wave_max_any(tm) * invt, rest);
  st.ml = wave_max_any(st.ml);
  nant = __ballot(nant) != 0;
  st.nan = __ballot(st.nan) != 0;
  const bool taught = tmax != -__builtin_inf() || nant;
  double sum = 0.0;
  for (int s = l; s < a.k; s += 64) {
    const float tv = sh.tv[s];
    const double pe = tv == ninf ? 0.0 : exp((double)tv * invt - tmax);
    sh.p[s] = pe;
    sum += pe;
  }
  const double re = rest == -__builtin_inf() ? 0.0 : exp(rest - tmax);
  sum = wave_sum_any(sum) + re;
  if (l == 0) sh.taught = taught, sh.pr = taught ? re / sum : 0.0;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (all lanes read them)
  for (int s = l; s < a.k; s += 64) sh.p[s] = sh.pt[s] = taught ? sh.p[s] / sum : 0.0, sh.first[s] = sh.id[s] >= 0;
  if (twice) {  // a token's first slot stands for it, with the sum of its slots' probabilities in slot order
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (int s = l; s < a.k; s += 64) {
      const int id = sh.id[s];
      if (id < 0) continue;
      double pt = 0.0;
      for (int o = 0; o < a.k; o++)
        if (sh.id[o] == id) {
          if (o < s) sh.first[s] = 0;
          pt += sh.p[o];
        }
      sh.pt[s] = pt;
    }
  }
  st.ZT = st.Z1 = 0.0;
  for (int s = l; s < a.k; s += 64) {
    const float zs = sh.zs[s];
    if (!sh.first[s] || zs == ninf) continue;
    st.ZT += exp2(((double)zs - st.ml) * a.scale);
    if (a.tok) st.Z1 += exp2(((double)zs - st.ml) * kLog2eD);
  }
  st.ZT = wave_sum_any(st.ZT);
  st.Z1 = wave_sum_any(st.Z1);
}

// the student's normaliser at a scale and its float c: 2^top times what is returned, of the listed sum Z at ml and the unlisted sum
// s at mu's reference; *share is 2^(that reference - top) over it
__device__ __forceinline__ double distill_norm(const DistillArgs& a, float c, double scale, float ml, double Z, float mu, double s, bool bad, double* top, double* share) {
  const float ninf = -__builtin_inff();
  const double kl = ml == ninf ? -__builtin_inf() : (double)ml * scale, ku = mu == ninf ? -__builtin_inf() : ref_exact(mu, c, scale, a.big);
  *top = fmax(kl, ku);
  const double less = exp2(-fabs(kl - ku));  // (0 where one of them is -inf)
  const double fl = ml == ninf ? 0.0 : kl < ku ? less : 1.0, fu = mu == ninf ? 0.0 : ku < kl ? less : 1.0;
  double t = Z * fl + (mu == ninf && s == s ? 0.0 : s * fu);
  if (bad || (ml == ninf && mu == ninf)) t = (double)__builtin_nanf("");
  *share = fu / t;
  return t;
}

struct DisNorms {
  double top[2], sum[2];  // of the two temperatures
};

// with the unlisted logits' statistics: the gradient's constants into sh
__device__ __forceinline__ void distill_scalars(const DistillArgs& a, DisShared& sh, const DisTeacher& st, const DisSum& d, float w_, DisNorms& nm) {
  const bool empty = d.m == -__builtin_inff(), label = sh.tok >= 0;
  double fT, f1 = 0.0;
  nm.sum[0] = distill_norm(a, a.c, a.scale, st.ml, st.ZT, d.m, d.sT, st.nan, &nm.top[0], &fT);
  nm.sum[1] = 1.0, nm.top[1] = 0.0;
  if (a.tok) nm.sum[1] = distill_norm(a, kLog2eF, kLog2eD, st.ml, st.Z1, d.m, d.s1, st.nan, &nm.top[1], &f1);
  const double w = (double)w_, pr = sh.pr;
  const double wT = sh.taught && w != 0.0 ? w * (1.0 - (double)a.hard) * (double)a.temp : 0.0;
  const double w1 = label && w != 0.0 ? w * (double)a.hard : 0.0;
  if ((threadIdx.x & 63) == 0) {
    sh.C = wT == 0.0 || (empty && nm.sum[0] == nm.sum[0]) ? 0.0f : (float)(wT * (fT - (pr > 0.0 ? pr / d.sT : 0.0)));
    sh.D = w1 == 0.0 || (empty && nm.sum[1] == nm.sum[1]) ? 0.0f : (float)(w1 * f1);
    sh.KT = ref_of(d.m, a.c, a.big), sh.K1 = ref_of(d.m, kLog2eF, a.big), sh.base = ref_base(d.m, a.big), sh.wgT = wT, sh.wg1 = w1;
  }
}

// log2 of the two normalisers and of the unlisted sum, for the losses and the gradient at the listed tokens
__device__ __forceinline__ void distill_logs(const DistillArgs& a, DisShared& sh, const DisSum& d, const DisNorms& nm) {
  const double LT = log2(nm.sum[0]), L1 = log2(nm.sum[1]);
  const double lu = d.m == -__builtin_inff() ? -__builtin_inf() : (ref_exact(d.m, a.c, a.scale, a.big) - nm.top[0]) + log2(d.sT);
  if ((threadIdx.x & 63) == 0) sh.tT = nm.top[0], sh.LT = LT, sh.t1 = nm.top[1], sh.L1 = L1, sh.lu = lu;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// the losses, by the wave that formed the scalars
__device__ __forceinline__ void distill_losses(const DistillArgs& a, const DisShared& sh, int i) {
  const int l = threadIdx.x & 63;
  const double c = a.scale, pr = sh.pr;
  double kl = 0.0;
  for (int s = l; s < a.k; s += 64) {  // a token's slots are one bucket
    const double p = sh.first[s] ? sh.pt[s] : 0.0;
    if (p > 0.0 || p != p) kl += p * (log(p) - sh.log_qT(sh.zs[s], c) * kLn2D);
  }
  kl = wave_sum_any(kl);
  if (pr > 0.0 || pr != pr) kl += pr * (log(pr) - (sh.lu - sh.LT) * kLn2D);
  if (l == 0) {
    a.kl[i] = sh.taught ? (float)kl : 0.0f;
    if (a.logp) a.logp[i] = sh.tok >= 0 ? (float)(sh.log_q1(sh.zt) * kLn2D) : __builtin_nanf("");
  }
}

// the gradient at the listed tokens and the label of [j0, j1), over the row's formula; by one wave
template <int VT, class Marks>
__device__ __forceinline__ void distill_marked(const DistillArgs& a, const DisShared& sh, const Marks& mk, void* out, int j0, int j1) {
  using R = VRow<VT>;
  const int l = threadIdx.x & 63;
  const double c = a.scale;
  for (int s = l; s < a.k; s += 64) {
    const int id = sh.id[s];
    if (!sh.first[s] || id < j0 || id >= j1) continue;
    double v = 0.0;
    if (sh.wgT != 0.0) v = sh.wgT * (exp2(sh.log_qT(sh.zs[s], c)) - sh.pt[s]);
    if (sh.wg1 != 0.0) v += sh.wg1 * (exp2(sh.log_q1(sh.zs[s])) - (id == sh.tok ? 1.0 : 0.0));
    R::put(out, id, (float)v);
  }
  if (l == 0 && sh.tok >= j0 && sh.tok < j1 && !mk.get(sh.tok - j0)) {
    double v = 0.0;
    if (sh.wgT != 0.0) v = sh.wgT * (exp2(sh.log_qT(sh.zt, c)) - (sh.pr > 0.0 ? sh.pr * exp2(((double)sh.zt * c - sh.tT) - sh.lu) : 0.0));
    if (sh.wg1 != 0.0) v += sh.wg1 * (exp2(sh.log_q1(sh.zt)) - 1.0);
    R::put(out, sh.tok, (float)v);
  }
}

// by the row's wave: the slots of row i and its label into LDS
__device__ __forceinline__ void distill_ids(const DistillArgs& a, DisShared& sh, int i) {
  for (int s = threadIdx.x & 63; s < a.k; s += 64) {
    const int id = a.ids[(int64_t)i * a.k + s];
    const float tv = a.tv[(int64_t)i * a.k + s];
    const bool held = id >= 0 && id < a.V;
    sh.id[s] = held ? id : -1;
    sh.tv[s] = held ? tv : -__builtin_inff();
  }
  const int tk = a.tok ? a.tok[i] : -1;
  sh.tok = tk >= 0 && tk < a.V ? tk : -1;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}
// and the marks of those in [j0, j1); whether one was set before
template <class Marks>
__device__ __forceinline__ bool distill_marks(const DistillArgs& a, const DisShared& sh, Marks& mk, int j0, int j1) {
  bool twice = false;
  for (int s = threadIdx.x & 63; s < a.k; s += 64)
    if (sh.id[s] >= j0 && sh.id[s] < j1) twice |= mk.set(sh.id[s] - j0);
  return __ballot(twice) != 0;
}

// the outputs of a row without logits over [j0, j1)
template <int VT>
__device__ __forceinline__ void distill_none(const DistillArgs& a, int i, void* out, int j0, int j1) {
  if (j0 == 0 && threadIdx.x == 0) {
    a.kl[i] = __builtin_nanf("");
    if (a.logp) a.logp[i] = __builtin_nanf("");
  }
  for (int j = j0 + (int)threadIdx.x; a.w && j < j1; j += blockDim.x) VRow<VT>::put(out, j, 0.0f);
}

// grid n, B threads
template <int VT, int B>
__device__ __forceinline__ void distill_row(const DistillArgs& a) {
  using R = VRow<VT>;
  constexpr int ST = B - 64;
  using Slice = DisSlice<VT, ST, kDisV<VT>, kDisL>;
  extern __shared__ u4v dyn[];  // [kDisL][ST] vectors, then a bit per logit
  uint32_t* mask = reinterpret_cast<uint32_t*>(dyn + kDisL * ST);
  __shared__ uint32_t any[ST / 64];
  __shared__ DisShared sh;
  const int tid = threadIdx.x, i = blockIdx.x;
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  void* out = static_cast<char*>(a.dz) + (int64_t)i * a.ldd * R::ES;
  if (!row_ok(a, i)) return distill_none<VT>(a, i, out, 0, a.V);
  typename Slice::Marks mk{mask, any};
  if (tid >= 64) {
    Slice sl;
    sl.init(0, a.V, tid - 64, dyn);
    sl.load(row);
    mk.clear(a.V);
    lds_barrier();
    lds_barrier();  // marked
    sl.stats(a, sh, row, mk);
    lds_barrier();
    lds_barrier();  // the scalars are there
    if (a.w) sl.write(a, sh, row, out);
    __syncthreads();
  } else {
    mk.clear(a.V);
    distill_ids(a, sh, i);
    lds_barrier();
    const bool twice = distill_marks(a, sh, mk, 0, a.V);
    lds_barrier();
    for (int s = tid; s < a.k; s += 64)
      if (sh.id[s] >= 0) sh.zs[s] = R::one(row, sh.id[s]);
    const float zt = sh.tok >= 0 ? R::one(row, sh.tok) : 0.0f, w = a.w ? a.w[i] : 0.0f;
    DisTeacher st;
    distill_teacher(a, sh, i, twice, st);
    lds_barrier();
    DisSum d;
    if (tid < ST / 64) d.m = sh.wm[tid], d.sT = sh.wT[tid], d.s1 = sh.w1[tid];
    d.join_wave(a);
    DisNorms nm;
    distill_scalars(a, sh, st, d, w, nm);
    lds_barrier();
    sh.zt = zt;
    distill_logs(a, sh, d, nm);
    distill_losses(a, sh, i);
    __syncthreads();  // the row is written
    if (a.w) distill_marked<VT>(a, sh, mk, out, 0, a.V);
  }
}

// Slices of kSliceB - 64 threads by kSliceV vectors.  grid (G, n): the statistics of slice g; slice 0 keeps the
// listed tokens' and the label's logits (the gradient may be written over them).
constexpr int kSliceB = 320, kSliceV = 8;
template <int VT>
__device__ __forceinline__ void distill_stats(const DistillArgs& a) {
  using R = VRow<VT>;
  constexpr int ST = kSliceB - 64;
  using Slice = DisSlice<VT, ST, kSliceV, 0>;
  __shared__ uint32_t mask[kSliceV * ST * R::E / 32 + 1];
  __shared__ uint32_t any[ST / 64];
  __shared__ DisShared sh;
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  if (!row_ok(a, i)) return;
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);  // L = kSliceV ST E
  typename Slice::Marks mk{mask, any};
  if (tid >= 64) {
    Slice sl;
    sl.init(j0, j1, tid - 64, nullptr);
    sl.load(row);
    mk.clear(j1 - j0);
    lds_barrier();
    lds_barrier();  // marked
    sl.stats(a, sh, row, mk);
    lds_barrier();
  } else {
    mk.clear(j1 - j0);
    distill_ids(a, sh, i);
    lds_barrier();
    const bool twice = distill_marks(a, sh, mk, j0, j1);
    lds_barrier();
    if (g == 0) {
      for (int s = tid; s < a.k; s += 64)
        if (sh.id[s] >= 0) a.zs[(int64_t)i * a.k + s] = R::one(row, sh.id[s]);
      if (tid == 0 && sh.tok >= 0) a.zt[i] = R::one(row, sh.tok);
    }
    lds_barrier();
    DisSum d;
    if (tid < ST / 64) d.m = sh.wm[tid], d.sT = sh.wT[tid], d.s1 = sh.w1[tid];
    d.join_wave(a);
    const int64_t o = (int64_t)i * a.G + g;
    if (tid == 0) a.pm[o] = d.m, a.psT[o] = d.sT, a.ps1[o] = d.s1, a.twice[o] = twice;
  }
}

// grid (G, n) (n alone without weights): each workgroup joins the row's slices and forms its scalars again, slice 0
// writes the losses
template <int VT>
__device__ __forceinline__ void distill_grad(const DistillArgs& a) {
  using R = VRow<VT>;
  constexpr int ST = kSliceB - 64;
  using Slice = DisSlice<VT, ST, kSliceV, 0>;
  __shared__ uint32_t mask[kSliceV * ST * R::E / 32 + 1];
  __shared__ uint32_t any[ST / 64];
  __shared__ DisShared sh;
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);
  const void* row = static_cast<const char*>(a.z) + (int64_t)i * a.ld * R::ES;
  void* out = static_cast<char*>(a.dz) + (int64_t)i * a.ldd * R::ES;
  if (!row_ok(a, i)) return distill_none<VT>(a, i, out, j0, j1);
  typename Slice::Marks mk{mask, any};
  if (tid >= 64) {
    Slice sl;
    sl.init(j0, j1, tid - 64, nullptr);
    if (a.w) sl.load(row);
    mk.clear(j1 - j0);
    lds_barrier();
    lds_barrier();  // the scalars are there
    if (a.w) sl.write(a, sh, row, out);
    __syncthreads();
  } else {
    mk.clear(j1 - j0);
    distill_ids(a, sh, i);
    for (int s = tid; s < a.k; s += 64)
      if (sh.id[s] >= 0) sh.zs[s] = a.zs[(int64_t)i * a.k + s];
    const float zt = sh.tok >= 0 ? a.zt[i] : 0.0f, w = a.w ? a.w[i] : 0.0f;
    int t2 = 0;
    DisSum d;
    for (int q = tid; q < a.G; q += 64) {
      const int64_t o = (int64_t)i * a.G + q;
      DisSum e;
      e.m = a.pm[o], e.sT = a.psT[o], e.s1 = a.ps1[o];
      t2 |= a.twice[o];
      if (e.m > d.m) d.raise(e.m, a);
      if (e.m < d.m) e.raise(d.m, a);
      d.sT += e.sT, d.s1 += e.s1;
    }
    d.join_wave(a);
    lds_barrier();
    distill_marks(a, sh, mk, j0, j1);
    DisTeacher st;
    distill_teacher(a, sh, i, __ballot(t2) != 0, st);
    DisNorms nm;
    distill_scalars(a, sh, st, d, w, nm);
    lds_barrier();
    sh.zt = zt;
    distill_logs(a, sh, d, nm);
    if (g == 0) distill_losses(a, sh, i);
    __syncthreads();  // the slice is written
    if (a.w) distill_marked<VT>(a, sh, mk, out, j0, j1);
  }
}

#define RTQ_DISTILL(ty, VT)                                                                                                \
  extern "C" __global__ __launch_bounds__(256, 4) void rtq_distill256_##ty(DistillArgs a) { distill_row<VT, 256>(a); }     \
  extern "C" __global__ __launch_bounds__(512, 4) void rtq_distill512_##ty(DistillArgs a) { distill_row<VT, 512>(a); }     \
  extern "C" __global__ __launch_bounds__(1024, 4) void rtq_distill1024_##ty(DistillArgs a) { distill_row<VT, 1024>(a); }  \
  extern "C" __global__ __launch_bounds__(kSliceB) void rtq_distill_stats_##ty(DistillArgs a) { distill_stats<VT>(a); }        \
  extern "C" __global__ __launch_bounds__(kSliceB) void rtq_distill_grad_##ty(DistillArgs a) { distill_grad<VT>(a); }
RTQ_DISTILL(f32, VT_F32)
RTQ_DISTILL(f16, VT_F16)
RTQ_DISTILL(bf16, VT_BF16)

// ============================================================== drafted tokens
// Sequence i: accept its drafted tokens x_0, x_1, ... while u_j q_j(x_j) < p_j(x_j) (p the target's
// softmax(z / T), q the draft's, or all of it on x_j without draft logits); the token after the accepted ones is
// drawn from max(p - q, 0) at the first rejection, from p after all: the first index whose running sum
// passes u_d times the total.  T = 0: accept while x_j is the target's largest logit (the lowest index
// of equals), which is also the token after.  Steps of the running sum over a flat tail lie nearer
// than 2^-24 of the total, so exponentials and sums are in 64 bits, whose arithmetic bounds the statistics (384
// rows of 151936 bf16 logits: 51 us, 2.3 TB/s, the VALU busy 83% of it; in one pass with a running maximum, the loads
// ahead of the sums: 53).
constexpr int kVdB = 256, kVdW = kVdB / 64, kVdV = 8;

// 2^(y / 256) for y <= 0: y = 256 n + i + f with |f| <= 1/2, a table of 2^(i / 256), and the series of exp(x) to
// the fourth power for x = f ln 2 / 256, whose next term is below 4e-17: off by a few 2^-53, as the sums are.
// (verification of 64 x 5 drafted tokens of 151936 bf16: 88 us; 90 with 128 entries and the quartic nearest to the series,
// 91 with 64 and the fifth power).  -inf gives 0; a NaN is not kept.
struct VdExp {
  double tab[256];
  __device__ __forceinline__ void fill(int t) {  // by t = 0 .. 255; a barrier follows
    tab[t] = exp2((double)t / 256.0);
  }
  __device__ __forceinline__ double operator()(double y) const {
    const double whole = 6755399441055744.0;  // 1.5 2^52: a sum with it ends at the ones, in its low bits
    y = fmax(y, -281600.0);
    const double n = y + whole, f = y - (n - whole);
    const int i = (int)(uint32_t)__builtin_bit_cast(uint64_t, n);
    constexpr double g = 0.6931471805599453 / 256.0;
    double p = g * g * g * g / 24.0;
    p = fma(p, f, g * g * g / 6.0);
    p = fma(p, f, g * g / 2.0);
    p = fma(p, f, g);
    p = fma(p, f, 1.0);
    return ldexp(p * tab[i & 255], i >> 8);
  }
};
__device__ __forceinline__ double vd_scale(const VerifyArgs& a) { return a.temp > 0.0f ? 369.3299304675746 / (double)a.temp : 0.0; }  // 256 log2(e) / T

template <int VT>
__device__ __forceinline__ const void* vd_row(const VerifyArgs& a, bool draft, int64_t row) {
  return static_cast<const char*>(draft ? a.q : a.z) + row * (draft ? a.ldq : a.ld) * VRow<VT>::ES;
}
__device__ __forceinline__ int vd_len(const VerifyArgs& a, int i) { return a.lens ? min(max(a.lens[i], 0), a.d) : a.d; }

// grid (G, b (d + 1) + b d): maximum and sum exp((z - max) / T) (T = 0: the largest rank key) of a slice of a target
// row, then of the draft rows; rows past a sequence's length are not read
template <int VT>
__device__ __forceinline__ void verify_stats(const VerifyArgs& a) {
  using R = VRow<VT>;
  constexpr int E = R::E;
  __shared__ uint64_t redk[kVdW];
  __shared__ float redf[kVdW];
  __shared__ double redd[kVdW];
  __shared__ VdExp ex;
  const int tid = threadIdx.x, g = blockIdx.x;
  const int64_t rr = blockIdx.y + (int64_t)blockIdx.z * 65535, tr = (int64_t)a.b * (a.d + 1);
  if (rr >= tr + (a.q ? (int64_t)a.b * a.d : 0)) return;
  const bool draft = rr >= tr;
  const int64_t row = draft ? rr - tr : rr;
  const int i = (int)(row / (draft ? a.d : a.d + 1)), j = (int)(row % (draft ? a.d : a.d + 1));
  const int len = vd_len(a, i);
  if (draft ? j >= len : j > len) return;
  const void* z = vd_row<VT>(a, draft, row);
  const int j0 = g * a.L, j1 = min(a.V, j0 + a.L);  // L = kVdB kVdV E
  const float ninf = -__builtin_inff();
  if (a.temp == 0.0f) {
    uint64_t best = 0;
#pragma unroll 1
    for (int o = j0 + tid * E; o < j1; o += kVdB * E) {
      const u4v r = R::load_upto(z, o, j1);
#pragma unroll
      for (int e = 0; e < E; e++) {
        const uint64_t key = o + e < j1 ? rank_key(R::get(r, e), o + e) : 0;
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
    if (tid == 0) a.pk[rr * a.G + g] = best;
    return;
  }
  float m = ninf;
  bool nan = false;
  auto see = [&](const u4v& r) {
#pragma unroll
    for (int e = 0; e < E; e++) m = fmaxf(m, R::get(r, e)), nan |= R::get(r, e) != R::get(r, e);
  };
  if (j0 + a.L <= a.V) {
    u4v raw[kVdV];
#pragma unroll
    for (int v = 0; v < kVdV; v++) raw[v] = R::load(z, j0 + (v * kVdB + tid) * E);
#pragma unroll
    for (int v = 0; v < kVdV; v++) see(raw[v]);
  } else {
#pragma unroll 1
    for (int o = j0 + tid * E; o < j1; o += kVdB * E) see(R::load_upto(z, o, j1));
  }
  ex.fill(tid);
  m = group_max<kVdW>(m, redf);  // (and its barriers)
  // (z - m) c and not z c - m c, which is not small where both are the type's lowest value
  const double c = vd_scale(a), ref = m == ninf ? 0.0 : (double)m;
  double s = nan || m == __builtin_inff() ? (double)__builtin_nanf("") : 0.0;
#pragma unroll 1
  for (int o = j0 + tid * E; o < j1; o += kVdB * E) {  // (again from the cache: in f64 registers go to the exponentials)
    const u4v r = R::load_upto(z, o, j1);
#pragma unroll
    for (int e = 0; e < E; e++) s += ex(((double)R::get(r, e) - ref) * c);
  }
  s = group_sum<kVdW>(s, redd);
  if (tid == 0) a.pk[rr * a.G + g] = __builtin_bit_cast(uint32_t, m), a.ps[rr * a.G + g] = s;
}

struct VdRow {
  double m, s;  // maximum, and the sum of exp((z - m) / T); NaN without a distribution
  int best;     // T = 0: the largest logit's index, -1 without a distribution
};
// a row's from its slices, by one wave
__device__ __forceinline__ VdRow vd_join(const VerifyArgs& a, const VdExp& ex, int64_t rr) {
  const int l = threadIdx.x & 63;
  if (a.temp == 0.0f) {
    uint64_t best = 0;
    for (int g = l; g < a.G; g += 64) best = a.pk[rr * a.G + g] > best ? a.pk[rr * a.G + g] : best;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
      const uint64_t o = __shfl_xor(best, m);
      best = o > best ? o : best;
    }
    const float z = key_value(best);  // NaN or -inf: no token
    return VdRow{0.0, 0.0, z > -__builtin_inff() ? key_index(best) : -1};
  }
  const double c = vd_scale(a);
  float m = -__builtin_inff();
  double s = 0.0;
  for (int g = l; g < a.G; g += 64) {
    const float m2 = __builtin_bit_cast(float, (uint32_t)a.pk[rr * a.G + g]);
    const double s2 = a.ps[rr * a.G + g];
    if (m2 > m) {
      s = s * (m == -__builtin_inff() ? 0.0 : ex(((double)m - m2) * c)) + s2;
      m = m2;
    } else {
      s += s2 * (m2 == -__builtin_inff() ? 0.0 : ex(((double)m2 - m) * c));
    }
  }
  const float M = wave_max_any(m);
  if (m != M) s *= m == -__builtin_inff() ? 0.0 : ex(((double)m - M) * c);
  s = wave_sum_any(s);
  return VdRow{(double)M, M == -__builtin_inff() ? (double)__builtin_nanf("") : s, -1};
}

// How many of sequence i's drafted tokens are accepted, and the row to draw from: the workgroup's waves
// test a token each, as many at a time as there are waves.  `write`: the outputs too.
template <int VT>
__device__ __forceinline__ VerifyPick vd_decide(const VerifyArgs& a, const VdExp& ex, int i, VerifyPick* lds, int* stop, bool write) {
  using R = VRow<VT>;
  const int tid = threadIdx.x, l = tid & 63, wv = tid >> 6, len = vd_len(a, i);
  const double c = vd_scale(a);
  const int64_t tr = (int64_t)a.b * (a.d + 1);
  int at = 0, found = kVdW;
  for (;; at += kVdW) {
    const int j = at + wv;
    bool here = false;  // the accepted end before j
    if (j <= len) {
      const int64_t prow = (int64_t)i * (a.d + 1) + j, qrow = (int64_t)i * a.d + j;
      const int x = j < len ? a.drafted[qrow] : -1;
      const bool in = x >= 0 && x < a.V;
      const float zp = in && a.temp > 0.0f ? R::one(vd_row<VT>(a, false, prow), x) : 0.0f;
      const float zq = in && a.q && j < len ? R::one(vd_row<VT>(a, true, qrow), x) : 0.0f;
      const VdRow p = vd_join(a, ex, prow);
      VerifyPick v;
      v.row = j, v.pm = p.m, v.ps = 1.0 / p.s, v.qm = 0.0, v.qs = 0.0, v.not_x = -1, v.minus_q = 0, v.best = p.best;
      if (j == len) {
        here = true;
      } else if (a.temp > 0.0f) {
        // (a NaN row gives a NaN probability, which accepts nothing)
        const double px = in ? (p.s != p.s ? p.s : ex(((double)zp - p.m) * c) / p.s) : 0.0;
        double qx = 1.0;
        if (a.q) {
          const VdRow q = vd_join(a, ex, tr + qrow);
          qx = in ? (q.s != q.s ? q.s : ex(((double)zq - q.m) * c) / q.s) : 0.0;
          v.qm = q.m, v.qs = 1.0 / q.s, v.minus_q = 1;
        } else {
          v.not_x = x;
        }
        here = !((double)a.u[(int64_t)i * (a.d + 1) + j] * qx < px);
      } else {
        here = !(in && x == p.best);
      }
      if (here && l == 0) lds[wv] = v;
    }
    if (l == 0) stop[wv] = here;
    __syncthreads();
    found = kVdW;
#pragma unroll
    for (int w = kVdW - 1; w >= 0; w--) found = stop[w] ? w : found;
    if (found < kVdW) break;  // (the wave of j == len stops at the latest)
    __syncthreads();
  }
  const VerifyPick v = lds[found];
  if (write) {
    for (int j = tid; j <= a.d; j += kVdB)
      a.tokens[(int64_t)i * (a.d + 1) + j] = j < v.row ? a.drafted[(int64_t)i * a.d + j] : j == v.row && a.temp == 0.0f ? v.best : -1;
    if (tid == 0) a.accepted[i] = v.row, a.pick[i] = v;
  }
  return v;
}

// grid b: T = 0
template <int VT>
__device__ __forceinline__ void verify_greedy(const VerifyArgs& a) {
  __shared__ VerifyPick lds[kVdW];
  __shared__ int stop[kVdW];
  __shared__ VdExp none;  // (not read at T = 0)
  vd_decide<VT>(a, none, blockIdx.x, lds, stop, true);
}

// the weight of token v: max(p - q, 0) after a rejection, or p
__device__ __forceinline__ double vd_weight(const VerifyPick& k, const VdExp& ex, double c, float zp, float zq, int v, double& p) {
  p = ex(((double)zp - k.pm) * c) * k.ps;
  if (k.minus_q) return fmax(p - ex(((double)zq - k.qm) * c) * k.qs, 0.0);
  return v == k.not_x ? 0.0 : p;
}

// grid (G, b): the weights' sums over the quarters of slice g of sequence i's row, a wave each, and p's (each workgroup
// decides again which row)
template <int VT>
__device__ __forceinline__ void verify_mass(const VerifyArgs& a) {
  using R = VRow<VT>;
  constexpr int E = R::E;
  __shared__ VerifyPick lds[kVdW];
  __shared__ int stop[kVdW];
  __shared__ VdExp ex;
  const int tid = threadIdx.x, g = blockIdx.x, i = blockIdx.y;
  ex.fill(tid);
  __syncthreads();
  const VerifyPick k = vd_decide<VT>(a, ex, i, lds, stop, g == 0);
  const void* zp = vd_row<VT>(a, false, (int64_t)i * (a.d + 1) + k.row);
  const void* zq = k.minus_q ? vd_row<VT>(a, true, (int64_t)i * a.d + k.row) : zp;
  const int q = g * kVdW + (tid >> 6), j0 = q * (a.L / kVdW), j1 = min(a.V, j0 + a.L / kVdW);
  const double c = vd_scale(a);
  double sw = 0.0, sp = k.ps != k.ps ? k.ps : 0.0;
#pragma unroll 1
  for (int v = j0 + (tid & 63) * E; v < j1; v += 64 * E) {
    const u4v r = R::load_upto(zp, v, j1);
    u4v rq = r;
    if (k.minus_q) rq = R::load_upto(zq, v, j1);
#pragma unroll
    for (int e = 0; e < E; e++) {
      double p;
      sw += vd_weight(k, ex, c, R::get(r, e), R::get(rq, e), v + e, p);
      sp += p;
    }
  }
  sw = wave_sum_any(sw);
  sp = wave_sum_any(sp);
  if ((tid & 63) == 0) {
    double* out = a.mass + ((int64_t)i * a.G * kVdW + q) * 2;
    out[0] = sw, out[1] = sp;
  }
}

// the sum over the lanes below this one, and over all
__device__ __forceinline__ double wave_before(double v, double* all) {
  const int l = threadIdx.x & 63;
  double s = v;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const double o = __shfl_up(s, d);
    s += l >= d ? o : 0.0;
  }
  *all = __shfl(s, 63);
  const double b = __shfl_up(s, 1);
  return l ? b : 0.0;
}

// grid b: the quarter slice that holds u_d times the total, then the token in it (1024 threads, consecutive logits
// each)
constexpr int kPickVdB = 1024, kVdMass = 8;  // kVdMass: quarter slices a lane at most (2^20 logits of f32: 512)
template <int VT>
__device__ __forceinline__ void verify_pick(const VerifyArgs& a) {
  using R = VRow<VT>;
  constexpr int E = R::E, N = E / 2, W = kPickVdB / 64;  // L / 4 = kVdB kVdV E / 4 = kPickVdB N
  __shared__ double part[W];
  __shared__ VdExp ex;
  __shared__ int sslice, sall, first, lastw;
  __shared__ double starget;
  const int tid = threadIdx.x, i = blockIdx.x, Q = a.G * kVdW;
  VerifyPick k = a.pick[i];
  if (tid < 64) {  // lane l: quarters per l .. per l + per - 1
    const double* mass = a.mass + (int64_t)i * Q * 2;
    const int per = (Q + 63) / 64;
    double w[kVdMass], p[kVdMass], sw = 0.0, sp = 0.0;
#pragma unroll
    for (int q = 0; q < kVdMass; q++) {
      const int at = tid * per + q;
      const bool in = q < per && at < Q;
      w[q] = in ? mass[2 * at] : 0.0, p[q] = in ? mass[2 * at + 1] : 0.0;
    }
    const float u = a.u[(int64_t)i * (a.d + 1) + a.d];
#pragma unroll
    for (int q = 0; q < kVdMass; q++) sw += w[q], sp += p[q];
    double tot, totp, before = wave_before(sw, &tot), beforep = wave_before(sp, &totp);
    const int all = tot > 0.0 ? 0 : 1;  // p - q is nowhere positive: drawn from p
    if (all) tot = totp, before = beforep;
    const double t = (double)u * tot;
    // the first quarter whose running sum passes t, or (rounding) the last that has weight
    int pass = 1 << 30, has = -1;
    double lo = 0.0, at_pass = 0.0, at_has = 0.0;
#pragma unroll
    for (int q = 0; q < kVdMass; q++) {
      const double x = all ? p[q] : w[q];
      if (x > 0.0) {
        has = tid * per + q, at_has = before + lo;
        if (pass == 1 << 30 && before + lo + x > t) pass = has, at_pass = at_has;
      }
      lo += x;
    }
    const uint64_t mp = __ballot(pass < (1 << 30)), mh = __ballot(has >= 0);
    const int lane = mp ? __builtin_ctzll(mp) : mh ? 63 - __builtin_clzll(mh) : 0;
    const int slice = __shfl(mp ? pass : has, lane);
    const double base = __shfl(mp ? at_pass : at_has, lane);
    if (tid == 0) sslice = tot > 0.0 ? slice : -1, sall = all, starget = t - base, first = 1 << 30, lastw = -1;  // NaN: no token
  } else if (tid < 64 + 256) {
    ex.fill(tid - 64);
  }
  __syncthreads();
  if (sslice < 0) return;
  if (sall) k.minus_q = 0, k.not_x = -1;
  const void* zp = vd_row<VT>(a, false, (int64_t)i * (a.d + 1) + k.row);
  const void* zq = k.minus_q ? vd_row<VT>(a, true, (int64_t)i * a.d + k.row) : zp;
  const double c = vd_scale(a);
  const int j0 = sslice * (a.L / kVdW), j1 = min(a.V, j0 + a.L / kVdW), v0 = j0 + tid * N;
  float fp[N], fq[N];
#pragma unroll
  for (int e = 0; e < N; e++) fp[e] = v0 + e < j1 ? R::one(zp, v0 + e) : 0.0f, fq[e] = v0 + e < j1 && k.minus_q ? R::one(zq, v0 + e) : 0.0f;
  double w[N], s = 0.0;
  int last = -1;
#pragma unroll
  for (int e = 0; e < N; e++) {
    double p;
    w[e] = v0 + e < j1 ? vd_weight(k, ex, c, fp[e], fq[e], v0 + e, p) : 0.0;
    s += w[e];
    last = w[e] > 0.0 ? v0 + e : last;
  }
  double sum;
  double before = wave_before(s, &sum);
  if ((tid & 63) == 0) part[tid >> 6] = sum;
  __syncthreads();
  for (int q = 0; q < (tid >> 6); q++) before += part[q];
  // the first logit whose running sum passes the target; rounding may leave none: then the last of the
  // quarter that has weight
  if (last >= 0) {
    double t = before;
    int mine = 1 << 30;
#pragma unroll
    for (int e = 0; e < N; e++) {
      t += w[e];
      mine = w[e] > 0.0 && t > starget ? min(mine, v0 + e) : mine;
    }
    if (mine < (1 << 30)) atomicMin(&first, mine);
    atomicMax(&lastw, last);
  }
  __syncthreads();
  if (tid == 0) a.tokens[(int64_t)i * (a.d + 1) + k.row] = first < (1 << 30) ? first : lastw;
}

#define RTQ_VERIFY(ty, VT)                                                                                              \
  extern "C" __global__ __launch_bounds__(kVdB) void rtq_verify_stats_##ty(VerifyArgs a) { verify_stats<VT>(a); }       \
  extern "C" __global__ __launch_bounds__(kVdB) void rtq_verify_greedy_##ty(VerifyArgs a) { verify_greedy<VT>(a); }     \
  extern "C" __global__ __launch_bounds__(kVdB) void rtq_verify_mass_##ty(VerifyArgs a) { verify_mass<VT>(a); }         \
  extern "C" __global__ __launch_bounds__(kPickVdB) void rtq_verify_pick_##ty(VerifyArgs a) { verify_pick<VT>(a); }
RTQ_VERIFY(f32, VT_F32)
RTQ_VERIFY(f16, VT_F16)
RTQ_VERIFY(bf16, VT_BF16)
