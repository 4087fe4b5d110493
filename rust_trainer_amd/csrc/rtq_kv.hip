// rtq_kv.hip — operators on a paged cache of keys and values (included by rtq_kernels.hip after
// rtq_vocab.hip, whose row types it uses): appending new tokens, attention of runs and trees of new
// tokens over what is cached, and keeping a tree's accepted tokens.
//
// A page holds `ps` slots (a power of two, 32 at least) of every KV head of one layer.  Keys lie
// [page][head][slot][d]; values lie transposed, [page][head][d][slot]: the attention's second product
// contracts over slots, and so both products read 16-byte MFMA operands straight from the cache, with no
// transposition through LDS.  The price is paid once per token, by the append's 2-byte stores.
// Page ids out of range are neither written nor read: their slots are not there.

// ------------------------------------------------------------------ sequences
__device__ __forceinline__ int kv_start(const KvSeqs& s, int i) {
  if (!s.starts) return (int)((int64_t)s.n / s.b) * i;
  return min(max(s.starts[i], 0), s.n);
}
// tokens held by sequence i, as far as its table's slots go
__device__ __forceinline__ int kv_held(const int32_t* lens, int i, int ldt, int ps_shift) {
  return (int)min((int64_t)max(lens[i], 0), min((int64_t)ldt << ps_shift, (int64_t)RTQ_KV_SLOTS));
}

// ------------------------------------------------------------------ append
// y = x inv_rms (w + off), then pairs (y1, y2) turned by position x freq: (y1 c - y2 s, y2 c + y1 s).  Every element is read
// and written once: copies bound it (16384 tokens of 16 query and 8 KV heads of 128, f32: 103 us, 4.5 TB/s of a copy's
// 4.7), and a few tokens their launch (5.6 us).
//
// 16 lanes take a head, a lane eight of its elements at a time (a unit: the two sides of four pairs, or eight in a
// row), a wave four heads.  Few tokens take a workgroup each, its waves sharing the heads; many take a wave
// each.  The angles are turns: position x freq in 64 bits, of which the whole turns are dropped before sine and cosine
// are taken in 32 (at position 10^5 a 32-bit angle is off by 4e-3), once per lane and pair for all of its heads.
// Values are turned over in LDS, 32 tokens of a head at a time: a token's elements lie a page row apart, and
// stored by themselves they were 2-byte stores (200 us for the call above).
__device__ __forceinline__ void kv_turn(double pos, double freq, float& c, float& s) {
  double t = pos * freq;
  t -= rint(t);
  sincospif(2.0f * (float)t, &s, &c);
}

template <int XT, int CT, int NU>
__device__ __forceinline__ void kv_append_rows(const KvAppendArgs& a, int tok, int seq, int h0, int step) {
  typedef VRow<XT> X;
  typedef VRow<CT> C;
  typedef u2v u2u __attribute__((aligned(2)));
  const int lane = threadIdx.x & 63, l16 = lane & 15;
  const int half = a.rot / 2, units = a.d / 8;
  const int64_t slot = (int64_t)max(a.s.lens[seq], 0) + (tok - kv_start(a.s, seq)), p = slot >> a.ps_shift;
  const int ps = 1 << a.ps_shift;
  const int pid = p < a.s.ldt ? a.s.table[(int64_t)seq * a.s.ldt + p] : -1;
  const bool stored = (unsigned)pid < (unsigned)a.n_pages, whole = a.rot % 8 == 0;
  const double pos = a.pos ? (double)a.pos[tok] : (double)slot;
  const int nq = a.q ? a.nh : 0, heads = nq + a.nkv;
  uint16_t* const kp = a.k + (((int64_t)(stored ? pid : 0) * a.nkv << a.ps_shift) + (slot & (ps - 1))) * a.d;
  // this lane's units: l16 and, of heads above 128, l16 + 16
  float cs[NU][4], sn[NU][4];
#pragma unroll
  for (int u = 0; u < NU; u++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      cs[u][e] = 1.0f, sn[u][e] = 0.0f;
      if (whole && l16 + 16 * u < a.rot / 8) kv_turn(pos, a.freq[4 * (l16 + 16 * u) + e], cs[u][e], sn[u][e]);
    }
  for (int h = h0 + (lane >> 4); h < heads; h += step) {
    const bool isq = h < nq;
    const int hh = isq ? h : h - nq;
    const void* x = isq ? a.q : a.kx;
    const int64_t at = (int64_t)tok * (isq ? a.ldq : a.ldk) + (int64_t)hh * a.d, qd = (int64_t)tok * a.ldo + (int64_t)hh * a.d;
    const float* w = isq ? a.q_norm : a.k_norm;
    uint16_t* const kd = kp + ((int64_t)hh << a.ps_shift) * a.d;
    if (!whole) {  // a rotation that ends inside a unit: element by element
      const auto put = [&](int j, float y) {
        if (isq) X::put(a.qo, qd + j, y);
        else if (stored) C::put(kd, j, y);
      };
      float ir = 1.0f;
      if (w) {
        float s = 0.0f;
        for (int j = l16; j < a.d; j += 16) s += X::one(x, at + j) * X::one(x, at + j);
#pragma unroll
        for (int m = 1; m <= 8; m <<= 1) s += __shfl_xor(s, m);
        ir = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)a.d) + a.eps));
      }
      const auto get = [&](int j) { return w ? X::one(x, at + j) * (ir * (w[j] + a.off)) : X::one(x, at + j); };
      for (int j = a.rot + l16; j < a.d; j += 16) put(j, get(j));
#pragma unroll 1
      for (int i = l16; i < half; i += 16) {
        const int ia = a.neox ? i : 2 * i, ib = a.neox ? i + half : 2 * i + 1;
        float sv, cv;
        kv_turn(pos, a.freq[i], cv, sv);
        const float x1 = get(ia), x2 = get(ib);
        put(ia, x1 * cv - x2 * sv), put(ib, x2 * cv + x1 * sv);
      }
      continue;
    }
    // unit u covers elements o1 .. o1 + 3 and o2 .. o2 + 3
    float v[NU][8];
    int o1[NU], o2[NU];
#pragma unroll
    for (int u = 0; u < NU; u++) {
      const int un = l16 + 16 * u;
      if (un >= units) continue;
      const bool split = a.neox && un < a.rot / 8;
      o1[u] = split ? 4 * un : 8 * un;
      o2[u] = split ? half + 4 * un : 8 * un + 4;
      if constexpr (XT == VT_F32) {
        const u4v r1 = X::load(x, at + o1[u]), r2 = X::load(x, at + o2[u]);
#pragma unroll
        for (int e = 0; e < 4; e++) v[u][e] = X::get(r1, e), v[u][4 + e] = X::get(r2, e);
      } else {
        const uint16_t* b = static_cast<const uint16_t*>(x) + at;
        const u2v r1 = *reinterpret_cast<const u2u*>(b + o1[u]), r2 = *reinterpret_cast<const u2u*>(b + o2[u]);
#pragma unroll
        for (int e = 0; e < 8; e++) v[u][e] = X::get(u4v{r1.x, r1.y, r2.x, r2.y}, e);
      }
    }
    if (w) {  // RMS norm of the head: (x / rms) (w + off)
      float s = 0.0f;
#pragma unroll
      for (int u = 0; u < NU; u++)
        if (l16 + 16 * u < units)
#pragma unroll
          for (int e = 0; e < 8; e++) s += v[u][e] * v[u][e];
#pragma unroll
      for (int m = 1; m <= 8; m <<= 1) s += __shfl_xor(s, m);
      const float ir = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)a.d) + a.eps));
#pragma unroll
      for (int u = 0; u < NU; u++)
        if (l16 + 16 * u < units)
#pragma unroll
          for (int e = 0; e < 8; e++) v[u][e] *= ir * (w[(e < 4 ? o1[u] : o2[u] - 4) + e] + a.off);
    }
#pragma unroll
    for (int u = 0; u < NU; u++)
      if (l16 + 16 * u < a.rot / 8) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float x1 = a.neox ? v[u][e] : v[u][2 * e], x2 = a.neox ? v[u][4 + e] : v[u][2 * e + 1];
          const float y1 = x1 * cs[u][e] - x2 * sn[u][e], y2 = x2 * cs[u][e] + x1 * sn[u][e];
          if (a.neox) v[u][e] = y1, v[u][4 + e] = y2;
          else v[u][2 * e] = y1, v[u][2 * e + 1] = y2;
        }
      }
#pragma unroll
    for (int u = 0; u < NU; u++) {
      if (l16 + 16 * u >= units) continue;
      if (isq) {
        if constexpr (XT == VT_F32) {
          X::store(a.qo, qd + o1[u], X::pack(v[u])), X::store(a.qo, qd + o2[u], X::pack(v[u] + 4));
        } else {
          uint16_t* b = static_cast<uint16_t*>(a.qo) + qd;
          const u4v r = X::pack(v[u]);
          *reinterpret_cast<u2u*>(b + o1[u]) = u2v{r[0], r[1]}, *reinterpret_cast<u2u*>(b + o2[u]) = u2v{r[2], r[3]};
        }
      } else if (stored) {  // (rows of the cache are 16-byte aligned)
        const u4v r = C::pack(v[u]);
        *reinterpret_cast<u2v*>(kd + o1[u]) = u2v{r[0], r[1]}, *reinterpret_cast<u2v*>(kd + o2[u]) = u2v{r[2], r[3]};
      }
    }
  }
}

// the sequence that row tok belongs to (-1: none), found by the wave's lanes
__device__ __forceinline__ int kv_find(const KvSeqs& s, int tok) {
  if (!s.starts) return tok / (s.n / s.b);
  for (int i0 = 0; i0 < s.b; i0 += 64) {
    const int i = i0 + (threadIdx.x & 63);
    const uint64_t hit = __ballot(i < s.b && kv_start(s, i) <= tok && tok < kv_start(s, i + 1));
    if (hit) return i0 + __ffsll((unsigned long long)hit) - 1;
  }
  return -1;
}

template <int XT, int CT, int NU>
__device__ __forceinline__ void kv_append(const KvAppendArgs& a) {
  const int wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if ((int)blockIdx.x < a.tw) {
    const int tok = a.wave_tokens ? 4 * blockIdx.x + wv : blockIdx.x;
    if (tok >= a.s.n) return;
    const int seq = kv_find(a.s, tok);
    if (seq >= 0) kv_append_rows<XT, CT, NU>(a, tok, seq, a.wave_tokens ? 0 : 4 * wv, a.wave_tokens ? 4 : 16);
    return;
  }
  // values: 32 tokens of one KV head, through LDS, so that neighbouring slots are stored together
  __shared__ uint16_t tile[256][34];  // [element][token], rows off each other's banks
  __shared__ int64_t dst[32];
  const int wg = blockIdx.x - a.tw, hv = wg % a.nkv, t0 = wg / a.nkv * 32;
  const int nt = min(32, a.s.n - t0), ps = 1 << a.ps_shift;
  typedef VRow<XT> X;
  constexpr int E = X::E;
  const int vecs = a.d / E;
  // rows of no sequence, before the first and behind the last, are not read (nor stored)
  typedef const __attribute__((address_space(4))) int32_t* cptr;
  const cptr starts = reinterpret_cast<cptr>(reinterpret_cast<uintptr_t>(a.s.starts));
  const int lo = a.s.starts ? max(starts[0] - t0, 0) : 0, hi = a.s.starts ? min(starts[a.s.b] - t0, nt) : nt;
  for (int i = lo * vecs + threadIdx.x; i < hi * vecs; i += 256) {
    const int t = i / vecs, c = i % vecs * E;
    const u4v r = X::load(a.vx, (int64_t)(t0 + t) * a.ldv + (int64_t)hv * a.d + c);
#pragma unroll
    for (int e = 0; e < E; e++) VRow<CT>::put(tile[c + e], t, X::get(r, e));
  }
  if (threadIdx.x < 64) {
    // where the tile's tokens go: a wave finds their sequences
    const int lane = threadIdx.x;
    int seq = -1, idx = 0;
    if (a.s.starts) {
      for (int i0 = 0; i0 < a.s.b; i0 += 64) {
        const int i = i0 + lane, s0 = i < a.s.b ? kv_start(a.s, i) : 0, s1 = i < a.s.b ? kv_start(a.s, i + 1) : 0;
        uint64_t near = __ballot(s0 < t0 + nt && s1 > t0 && s1 > s0);
        while (near) {  // (each sequence that meets the tile)
          const int j = __ffsll((unsigned long long)near) - 1;
          near &= near - 1;
          const int b0 = __builtin_amdgcn_readlane(s0, j), b1 = __builtin_amdgcn_readlane(s1, j), t = t0 + lane;
          if (t >= b0 && t < b1) seq = i0 + j, idx = t - b0;
        }
      }
    } else {
      const int per = a.s.n / a.s.b;
      seq = (t0 + lane) / per, idx = (t0 + lane) % per;
    }
    if (lane < 32) {
      int64_t at = -1;
      if (lane >= lo && lane < hi && seq >= 0) {
        const int64_t slot = (int64_t)max(a.s.lens[seq], 0) + idx;
        const int64_t p = slot >> a.ps_shift;
        const int pid = p < a.s.ldt ? a.s.table[(int64_t)seq * a.s.ldt + p] : -1;
        if ((unsigned)pid < (unsigned)a.n_pages) at = (((int64_t)pid * a.nkv + hv) * a.d << a.ps_shift) + (slot & (ps - 1));
      }
      dst[lane] = at;
    }
  }
  __syncthreads();
  // eight tokens in neighbouring, aligned slots are one store
  const int t8 = (threadIdx.x & 3) * 8;
  bool run = dst[t8] >= 0 && dst[t8] % 8 == 0;
#pragma unroll
  for (int j = 1; j < 8; j++) run = run && dst[t8 + j] == dst[t8] + j;
  for (int c = threadIdx.x >> 2; c < a.d; c += 64) {
    if (run) {
      const uint32_t* r = reinterpret_cast<const uint32_t*>(&tile[c][t8]);
      *reinterpret_cast<u4v*>(a.v + dst[t8] + ((int64_t)c << a.ps_shift)) = u4v{r[0], r[1], r[2], r[3]};
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (dst[t8 + j] >= 0) a.v[dst[t8 + j] + ((int64_t)c << a.ps_shift)] = tile[c][t8 + j];
    }
  }
}

#define RTQ_KV_APPEND(NAME, XT, CT) \
  extern "C" __global__ __launch_bounds__(256) void NAME(KvAppendArgs a) { kv_append<XT, CT, 1>(a); } \
  extern "C" __global__ __launch_bounds__(256) void NAME##_256(KvAppendArgs a) { kv_append<XT, CT, 2>(a); }
RTQ_KV_APPEND(rtq_kv_append_f32_f16, VT_F32, VT_F16)
RTQ_KV_APPEND(rtq_kv_append_f32_bf16, VT_F32, VT_BF16)
RTQ_KV_APPEND(rtq_kv_append_f16, VT_F16, VT_F16)
RTQ_KV_APPEND(rtq_kv_append_bf16, VT_BF16, VT_BF16)

// ------------------------------------------------------------------ keep
// A few rows are moved within the cache: what bounds it is that a token's values are 2 bytes of each of d rows, so that a
// 64-byte piece is read and written for each (32 sequences, 8 tokens of 63 kept, 28 layers of 8 heads of 128: 22 us,
// 12.5 at a copy's rate for the bytes alone; one sequence: 4.4 us).
// Workgroup: one KV head of one sequence and layer.  Kept tokens ascend, so the j-th comes from a slot no
// earlier than its own: a wave that moves its elements in batches of eight tokens, in order, each batch's loads before its
// stores, never writes a slot that it has yet to read, and no two waves touch the same elements.  Values: eight
// lanes take an element's eight tokens (neighbouring slots of one row), keys: d / 8 lanes a token.
#define RTQ_KV_KEEP 1024
extern "C" __global__ __launch_bounds__(256) void rtq_kv_keep(KvKeepArgs a) {
  __shared__ int64_t from[RTQ_KV_KEEP], to[RTQ_KV_KEEP];  // page x slots + slot; from -1: not moved
  __shared__ int count;
  const int hv = blockIdx.x % a.nkv, seq = blockIdx.x / a.nkv, tid = threadIdx.x;
  const int32_t* kept = a.kept + (int64_t)seq * a.ldk;
  const int held = max(a.lens[seq], 0), ps = 1 << a.ps_shift;
  if (tid == 0) count = a.ldk;
  __syncthreads();
  for (int j = tid; j < a.ldk; j += 256) {  // the list ends at the first entry that does not ascend
    const int x = kept[j];
    if (x < 0 || (j && x <= kept[j - 1])) atomicMin(&count, j);
    const int64_t f = (int64_t)held + max(x, 0), t = (int64_t)held + j;
    const int64_t fp = f >> a.ps_shift, tp = t >> a.ps_shift;
    const int fi = fp < a.ldt ? a.table[(int64_t)seq * a.ldt + fp] : -1, ti = tp < a.ldt ? a.table[(int64_t)seq * a.ldt + tp] : -1;
    const bool ok = (unsigned)fi < (unsigned)a.n_pages && (unsigned)ti < (unsigned)a.n_pages && f != t;
    from[j] = ok ? ((int64_t)fi << 32 | (f & (ps - 1))) : -1;
    to[j] = (int64_t)ti << 32 | (t & (ps - 1));
  }
  __syncthreads();
  const int n = count;
  if (blockIdx.y == 0 && hv == 0 && tid == 0 && a.after) a.after[seq] = held + n;
  const int64_t row = (int64_t)a.d << a.ps_shift;  // elements of a head's page
  uint16_t* k = a.k + blockIdx.y * a.layer;
  uint16_t* v = a.v + blockIdx.y * a.layer;
  const auto page = [&](int64_t at) { return ((at >> 32) * a.nkv + hv) * row; };
  const int lane = tid & 63, wv = tid >> 6, lanes = a.d / 8;
  if (wv == 0) {  // keys, 16 bytes a lane: 64 / lanes tokens at once (2 .. 32; 5 .. 15 lanes leave some idle)
    const int per = min(64 / lanes, 8), jl = lane / lanes, e = lane % lanes * 8;
    for (int j0 = 0; j0 < n; j0 += 8) {
      u4v x[4];
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int j = j0 + i * per + jl;
        if (jl < per && i * per + jl < 8 && j < n && from[j] >= 0) x[i] = *reinterpret_cast<const u4v*>(k + page(from[j]) + (from[j] & 0xffffffff) * a.d + e);
      }
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // (a lane may write what another has read)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const int j = j0 + i * per + jl;
        if (jl < per && i * per + jl < 8 && j < n && from[j] >= 0) *reinterpret_cast<u4v*>(k + page(to[j]) + (to[j] & 0xffffffff) * a.d + e) = x[i];
      }
    }
  }
  const int jl = lane & 7;
  for (int j0 = 0; j0 < n; j0 += 8) {
    const int j = j0 + jl;
    if (j >= n || from[j] < 0) continue;
    const uint16_t* src = v + page(from[j]) + (from[j] & 0xffffffff);
    uint16_t* dst = v + page(to[j]) + (to[j] & 0xffffffff);
    for (int c0 = 8 * wv + (lane >> 3); c0 < a.d; c0 += 128) {
      uint16_t x[4];
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (c0 + 32 * i < a.d) x[i] = src[(int64_t)(c0 + 32 * i) << a.ps_shift];
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (c0 + 32 * i < a.d) dst[(int64_t)(c0 + 32 * i) << a.ps_shift] = x[i];
    }
  }
}

// ------------------------------------------------------------------ attention
// o = sum_j p_j v_j / sum_j p_j, p_j = exp(scale q k_j - m), m the running maximum: one pass over the keys and values.
// Rows of one (sequence, KV head): its new tokens x the head's group of query heads, token by token; a tile
// takes TM of them, so that a group reads its keys once.  The keys of a tile are split into ranges of C slots (one C for the
// call, chosen on the device from the sequences' lengths: the host does not know them); an item is a tile and a range.  Tiles
// of one range leave o directly, others an unnormalised sum, the maximum and the sum of the weights, which are
// joined by the tile's last workgroup or by a kernel behind.
//
// Small tiles (16 rows: single tokens and narrow trees) are bound by the reading of the cache: 64 sequences of up to
// 8192 tokens, 32 over 8 heads of 128, 1.15 GB: 259 us, 4.4 TB/s; one of 131072: 97 us, 5.5 TB/s (some of it still cached);
// one of 1000: 14 us, of which the reading takes 1: each item is a chain of dependent loads (lengths, page, keys, values).
// Large ones (128 rows) are bound by the matrix instructions: 2048 tokens behind 6144, 32 over 8 heads of 128, bf16: 316 us,
// 0.76 PFLOP/s, and 1.14 with the weights' second plane counted, of a large product's 1.2.
//
// A wave takes 32 slots at a time.  S^T = K q^T and o^T = V^T p^T, so that a lane holds one query row:
// key row m of tile t is slot 8 (m / 4) + 4 t + m % 4, and the lane that gets the scores of slots 8 g .. 8 g + 7
// holds them in the order in which it feeds them to the second product: the weights never leave their lane.
//
// Weights are rounded to the cache's 16 bits for the second product, in two planes (three of f32 rows over bf16) that keep
// 16 to 22 bits of them, in small tiles and in large ones: a row is as exact whatever other rows its call has.  Sums stay in 32 bits.
struct KvItem {
  int seq, row0, cnt, held, total, tile, hv, split, splits, slot, C;  // slot: of the tile's first part (-1: one part)
};
// workgroups of a split tile that have left their part, at half the tile's first slot (a tile has two or more); zero
// between launches: the last one clears it
constexpr int kKvCounters = RTQ_KV_TARGET;  // (slots are twice the items)
__device__ int kv_arrived[kKvCounters];

// inclusive sums over the wave's lanes (DPP: rows of 16, then across them)
__device__ __forceinline__ int kv_wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // the lane 1, 2, 4, 8 before, within the row
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row 0's and row 2's last lane to the row behind
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row 1's to rows 2 and 3
  return v;
}
__device__ __forceinline__ float kv_wave_total(float v) {
  const auto dpp = [&](auto c, auto rows) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), decltype(c)::value, decltype(rows)::value, 0xf, false));
  };
  v += dpp(std::integral_constant<int, 0x111>{}, std::integral_constant<int, 0xf>{});
  v += dpp(std::integral_constant<int, 0x112>{}, std::integral_constant<int, 0xf>{});
  v += dpp(std::integral_constant<int, 0x114>{}, std::integral_constant<int, 0xf>{});
  v += dpp(std::integral_constant<int, 0x118>{}, std::integral_constant<int, 0xf>{});
  v += dpp(std::integral_constant<int, 0x142>{}, std::integral_constant<int, 0xa>{});
  v += dpp(std::integral_constant<int, 0x143>{}, std::integral_constant<int, 0xc>{});
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), 63));
}

// item `block` of the plan (every wave finds it by itself; a lane looks after b / 64 sequences); false: none.
// Sequences that overlap in `starts` can name more than the host counted: then whole tiles are left out.
__device__ __forceinline__ bool kv_plan(const KvAttendArgs& a, const int TM, int block, KvItem& it) {
  const int lane = threadIdx.x & 63, group = a.group;
  const int per = (a.s.b + 63) / 64, i0 = min(lane * per, a.s.b), i1 = min(i0 + per, a.s.b);
  int row0 = 0, cnt = 0, held = 0, total = 0, tiles = 0;
  const auto look = [&](int i) {
    row0 = kv_start(a.s, i);
    cnt = max(kv_start(a.s, i + 1) - row0, 0);
    held = kv_held(a.s.lens, i, a.s.ldt, a.ps_shift);
    total = (int)min((int64_t)held + cnt, min((int64_t)a.s.ldt << a.ps_shift, (int64_t)RTQ_KV_SLOTS));
    tiles = (int)(((int64_t)cnt * group + TM - 1) / TM);
  };
  float w = 0.0f, whole = 0.0f;
  int longest = 0;
  for (int i = i0; i < i1; i++) {
    look(i);
    w += (float)tiles * (float)total, whole += (float)tiles;
    if (tiles) longest = max(longest, total);
  }
  // a sequence's slots a part, parts
  const auto cut = [&](int C, int& c, int& ns) {
    c = kv_range(total, (int)min((int64_t)max(cnt, 1) * a.group, (int64_t)TM), C, a.fused);
    if (TM == 16 && total <= a.whole) c = max(c, a.whole);
    ns = kv_parts(total, c);
  };
  // Ranges of about even x 128 slots share the slots out evenly over the items that run at once.  With few tiles
  // that is it.  With more, what their last ranges leave over makes a second turn of the CUs: then the shortest ranges (of
  // some) are taken with which all items run at once (32 sequences of 1000 to 7000, 64 rows: 174 -> 140 us).  Tiles that
  // nearly fill the CUs are not split at all, unless one is far longer than the others (32 of 250 to 1750, 4 rows: 42 -> 34
  // us).  Small tiles of long sequences, and large ones that have a CU each, are better off with ranges as short as the
  // items allow, a second turn or not (32 of 4000 to 28000: 457 us against 550 unsplit; 64 rows and a head size of 256:
  // 1676 against 2199 in even ranges).
  const float even = kv_wave_total(w) * (float)a.nkv / (float)a.once / 128.0f, most = kv_wave_total(whole) * (float)a.nkv;
  const auto range = [&](float f) { return max((int)fminf(ceilf(even * f), (float)(RTQ_KV_SLOTS / 128)) * 128, 128); };
  int C = range(1.0f), c, ns;
  if (TM > 16 && !__any(longest > a.whole)) {
    C = max(C, a.whole);
  } else if (C > 2048 && (TM == 16 || a.once < a.target)) {
    if (most * 2.0f >= (float)a.once) C = range((float)a.once / (float)a.target);
  } else if (most * 16.0f > (float)a.once) {
    constexpr float kTry[] = {1.0f, 1.25f, 1.5f, 2.0f, 3.0f, 4.0f};
    float n[6] = {}, inv[6];  // items of each (about)
#pragma unroll
    for (int f = 0; f < 6; f++) inv[f] = __builtin_amdgcn_rcpf((float)range(kTry[f]));
    for (int i = i0; i < i1; i++) {
      if (per > 1) look(i);
#pragma unroll
      for (int f = 0; f < 6; f++) n[f] += (float)tiles * (TM == 16 && total <= a.whole ? 1.0f : ceilf((float)total * inv[f]));
    }
#pragma unroll
    for (int f = 0; f < 6; f++) n[f] = kv_wave_total(n[f]) * (float)a.nkv;
    if (most * (TM == 16 ? 2.0f : 1.0f) >= (float)a.once && n[5] <= most) {
      C = range(kTry[5]);
    } else {
#pragma unroll
      for (int f = 4; f >= 0; f--)
        if (n[f] <= (float)a.once) C = range(kTry[f]);
    }
  }
  int items = 0, slots = 0;
  for (int i = i0; i < i1; i++) {
    if (per > 1) look(i);
    cut(C, c, ns);
    items += tiles * a.nkv * ns, slots += ns > 1 ? tiles * a.nkv * ns : 0;
  }
  int ei = kv_wave_scan(items) - items, es = kv_wave_scan(slots) - slots;
  if (!a.fused && block == 0 && threadIdx.x == 63) a.items[0] = es + slots;
  const uint64_t mine = __ballot(block >= ei && block < ei + items);
  if (!mine) return false;
  int ok = 0;
  if (block >= ei && block < ei + items) {
    for (int i = i0; i < i1; i++) {
      if (per > 1) look(i);
      cut(C, c, ns);
      const int n = tiles * a.nkv * ns;
      if (block < ei + n) {
        const int at = block - ei;  // tile by tile, so that a range's tiles are a multiple of the XCDs apart
        it.seq = i, it.row0 = row0, it.cnt = cnt, it.held = held, it.total = total, it.splits = ns, it.C = c;
        it.tile = at / (a.nkv * ns);
        it.hv = (at - it.tile * a.nkv * ns) / ns, it.split = at - (it.tile * a.nkv + it.hv) * ns;
        const bool found = at >= 0 && it.tile < tiles;  // (sums of sequences that overlap may pass 32 bits)
        // A run's later tiles have more slots: they start first, and where two workgroups a CU take all of them at once, the
        // n-th longest shares its CU with the n-th shortest.
        if (!a.parents) it.tile = n > a.once || 2 * it.tile < tiles ? tiles - 1 - it.tile : it.tile - (tiles + 1) / 2;
        it.slot = ns > 1 ? es + at - it.split : -1;
        ok = found && (ns == 1 || (it.slot >= 0 && it.slot + ns <= a.slots && block - it.split + ns <= (int)gridDim.x));
        break;
      }
      ei += n, es += ns > 1 ? n : 0;
    }
  }
  const int src = __ffsll((unsigned long long)mine) - 1;
#define RTQ_KV_GIVE(F) it.F = __builtin_amdgcn_readlane(it.F, src)
  RTQ_KV_GIVE(seq), RTQ_KV_GIVE(row0), RTQ_KV_GIVE(cnt), RTQ_KV_GIVE(held), RTQ_KV_GIVE(total), RTQ_KV_GIVE(tile);
  RTQ_KV_GIVE(hv), RTQ_KV_GIVE(split), RTQ_KV_GIVE(splits), RTQ_KV_GIVE(slot), RTQ_KV_GIVE(C);
#undef RTQ_KV_GIVE
  if (!__builtin_amdgcn_readlane(ok, src)) return false;
  if (!a.fused && it.slot >= 0 && threadIdx.x == 0)
    *reinterpret_cast<KvItem*>(a.items + (1 + it.slot + it.split) * RTQ_KV_ITEM) = it;
  return true;
}

template <int CT>
__device__ __forceinline__ f4 kv_mfma(u4v x, u4v y, f4 c) {
  if constexpr (CT == VT_F16) return mfma_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c);
  else return mfma_bf16(__builtin_bit_cast(bf8, x), __builtin_bit_cast(bf8, y), c);
}
template <int CT>
__device__ __forceinline__ f16v kv_mfma32(u4v x, u4v y, f16v c) {
  if constexpr (CT == VT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf8, x), __builtin_bit_cast(bf8, y), c, 0, 0, 0);
}

typedef float f8v __attribute__((ext_vector_type(8)));
// eight floats as N planes of 16 bits, each the rounding of what the ones before it leave: 11 (f16) or 8
// (bf16) bits of the value a plane: f32 rows take two (f16) or three, one plane of a 16-bit row is the row itself.
template <int CT, int N>
__device__ __forceinline__ void kv_planes(const float* v, u4v* out) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = v[e];
#pragma unroll
  for (int n = 0; n < N; n++) {
    const f8v x = {r[0], r[1], r[2], r[3], r[4], r[5], r[6], r[7]};  // (converted in pairs)
    if constexpr (CT == VT_F16) out[n] = __builtin_bit_cast(u4v, __builtin_convertvector(x, half8));
    else out[n] = __builtin_bit_cast(u4v, __builtin_convertvector(x, bf8));
    if (n + 1 < N)
#pragma unroll
      for (int e = 0; e < 8; e++) r[e] -= VRow<CT>::get(out[n], e);
  }
}

// the page of slot k of sequence seq (uniform: a scalar load, which no vector load in flight is waited for with)
__device__ __forceinline__ int kv_page(const KvSeqs& s, int seq, int k, int ps_shift) {
  typedef const __attribute__((address_space(4))) int32_t* cptr;
  if (s.ldt <= 0) return -1;
  return reinterpret_cast<cptr>(reinterpret_cast<uintptr_t>(s.table + (int64_t)seq * s.ldt))[min(k >> ps_shift, s.ldt - 1)];
}

#define RTQ_KV_TREE 1024  // most new tokens of a sequence that is a tree

// f16 weights are taken times 2^9 (as is their sum): small ones, of which a long context has many, keep their bits.
// Large tiles follow a row's maximum only once it has risen by kKvLag (a factor 2^6 of the weights, which f16 still
// holds): with the maxima of 32 rows some rises in most steps, and each rise costs a product per accumulator.
template <int CT>
constexpr float kKvUp = CT == VT_F16 ? 9.0f : 0.0f;
constexpr float kKvLag = 6.0f;

// What an item works on, beside the plan's: its rows and slots
struct KvTile {
  int row_lo, rows, k_lo, k_hi;
  bool tail;  // some of its slots hold new tokens (or are the last of a table that has none for them)
};
__device__ __forceinline__ KvTile kv_tile(const KvAttendArgs& a, int TM, const KvItem& it) {
  KvTile t;
  const int group = a.group;
  t.row_lo = it.tile * TM, t.rows = min((int)((int64_t)it.cnt * group - t.row_lo), TM);
  t.k_lo = it.split * it.C;
  // (no row of the tile sees a new token after its own)
  const int64_t last = (int64_t)it.held + (t.row_lo + t.rows - 1) / group + 1;
  t.k_hi = (int)min(min((int64_t)t.k_lo + it.C, (int64_t)it.total), last);
  t.tail = t.k_hi >= min(it.held + 1, it.total);
  return t;
}

// The tile's tokens' chains as bits, seen[token - the tile's first] (none, not even the token's own, where the chain meets
// what is no parent: nothing is seen).  up: room for RTQ_KV_TREE parents.  Ends with a barrier.
typedef uint32_t KvSeen[RTQ_KV_TREE / 32];
template <int TOK, int THREADS>
__device__ __forceinline__ void kv_tree(const KvAttendArgs& a, const KvItem& it, const KvTile& t, KvSeen* seen, uint16_t* up) {
  const int group = a.group, n = min(it.cnt, RTQ_KV_TREE);
  const int first = t.row_lo / group, toks = (t.row_lo + t.rows - 1) / group - first + 1;
  for (int i = threadIdx.x; i < TOK * (RTQ_KV_TREE / 32); i += THREADS) (&seen[0][0])[i] = 0;
  for (int i = threadIdx.x; i < n; i += THREADS) {  // 0: the cache, else the parent + 1; 65535: none
    const int p = a.parents[it.row0 + i];
    up[i] = p < -1 || p >= i ? 65535 : p + 1;
  }
  __syncthreads();
  for (int r = threadIdx.x; r < toks; r += THREADS) {
    int node = first + r, dead = it.cnt > RTQ_KV_TREE;
    while (!dead && node >= 0) {
      seen[r][node >> 5] |= 1u << (node & 31);
      const int p = up[node];
      dead = p == 65535;
      node = p - 1;
    }
    if (dead)
      for (int w = 0; w < RTQ_KV_TREE / 32; w++) seen[r][w] = 0;
  }
  __syncthreads();
}
__device__ __forceinline__ bool kv_dead(const uint32_t* seen, int tok) { return !(seen[(tok & (RTQ_KV_TREE - 1)) >> 5] >> (tok & 31) & 1); }
// 32 bits from new token nw0 on (held tokens before it are seen): what token tok sees of them
__device__ __forceinline__ uint32_t kv_run_bits(int nw0, int tok) {
  const int n = tok - nw0 + 1;
  return n >= 32 ? 0xffffffffu : n <= 0 ? 0u : (1u << n) - 1;
}
__device__ __forceinline__ uint32_t kv_tree_bits(int nw0, const uint32_t* seen) {
  const int w = nw0 >> 5, sh = nw0 & 31;
  const auto word = [&](int i) { return i < 0 ? 0xffffffffu : i < RTQ_KV_TREE / 32 ? seen[i] : 0u; };
  return (uint32_t)(((uint64_t)word(w + 1) << 32 | word(w)) >> sh);
}

// eight 16-bit elements, of which those from element n on are cleared
__device__ __forceinline__ u4v kv_clear(u4v x, int n) {
#pragma unroll
  for (int w = 0; w < 4; w++) x[w] = 2 * w >= n ? 0u : 2 * w + 1 >= n ? x[w] & 0xffffu : x[w];
  return x;
}

// f32 rows over an f16 cache are scaled by a power of two (whose exponent is returned) that brings the row's
// largest element, of which the caller has mx, to [2^13, 2^14): its planes then neither overflow nor lose bits
__device__ __forceinline__ int kv_row_shift(float mx) {
  const int ex = (int)(__builtin_bit_cast(uint32_t, mx) >> 23);
  return ex == 255 || ex == 0 ? 0 : min(max(140 - ex, -120), 120);
}

// ---- the end of an item
// A row whose products met infinity or NaN, by the formula: in the matrix instructions a value that the row does not see
// still meets its weight 0, and the lower planes of queries and weights, which may be 0 or of the other sign,
// meet infinities.  Here only what is seen is multiplied, in 32 bits; slow, and rare.
// (A row is read again as its call was given it: out may be q itself, whose rows no other workgroup writes.)
struct KvAgain {
  float qs[256], sc[256], mx[256];
  int64_t at[256];  // the keys' pages (-1: not seen), looked up once
  uint32_t seen[RTQ_KV_TREE / 32];
  int dead;
};
template <int QT, int CT>
__device__ __forceinline__ void kv_row_again(const KvAttendArgs& a, const KvItem& it, int row, KvAgain& sh) {
  float *qs = sh.qs, *sc = sh.sc, *mx = sh.mx;
  uint32_t* seen = sh.seen;
  int& dead = sh.dead;
  const int tid = threadIdx.x, group = a.group, tok = row / group, seq = it.seq, hv = it.hv, d = a.d, held = it.held;
  const int last = min(held + tok + 1, it.total);
  __syncthreads();
  if (tid < d) qs[tid] = VRow<QT>::one(a.q, (int64_t)(it.row0 + tok) * a.ldq + (int64_t)(hv * group + row % group) * d + tid);
  if (tid < RTQ_KV_TREE / 32) seen[tid] = 0;
  if (tid == 0) dead = a.parents && tok >= RTQ_KV_TREE;
  __syncthreads();
  if (tid == 0 && a.parents)
    for (int node = tok; node >= 0 && !dead;) {
      seen[node >> 5] |= 1u << (node & 31);
      const int p = a.parents[it.row0 + node];
      if (p < -1 || p >= node) dead = 1;
      node = p;
    }
  __syncthreads();
  const int64_t head = (int64_t)d << a.ps_shift;
  const int ps = 1 << a.ps_shift;
  const auto conv = [&](uint16_t x) { return VRow<CT>::get(u4v{x, x, x, x}, 0); };
  const auto page = [&](int key) {
    const int pg = a.s.table[(int64_t)seq * a.s.ldt + (key >> a.ps_shift)];
    return (unsigned)pg < (unsigned)a.n_pages ? ((int64_t)pg * a.nkv + hv) * head : -1;
  };
  float m = -INFINITY, l = 0.0f, o = 0.0f;
  for (int k0 = 0; k0 < last && !dead; k0 += 256) {
    const int key = k0 + tid, nw = key - held;
    float s = -INFINITY;
    int64_t at = -1;
    const bool vis = key < last && (nw < 0 || !a.parents || (seen[(nw & (RTQ_KV_TREE - 1)) >> 5] >> (nw & 31) & 1));
    if (vis) {
      at = page(key);
      if (at >= 0) {
        const uint16_t* k = a.k + at + (int64_t)(key & (ps - 1)) * d;
        s = 0.0f;
        for (int c = 0; c < d; c++) s = fmaf(qs[c], conv(k[c]), s);
        s *= a.scale2;
      }
    }
    mx[tid] = s, sh.at[tid] = at;
    __syncthreads();
    for (int n = 128; n > 0; n >>= 1) {
      if (tid < n) mx[tid] = fmaxf(mx[tid], mx[tid + n]);
      __syncthreads();
    }
    const float mn = fmaxf(m, mx[0]), mu = mn == -INFINITY ? 0.0f : mn, al = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    sc[tid] = __builtin_amdgcn_exp2f(s - mu);
    __syncthreads();
    l *= al, o *= al;
    for (int j = 0; j < 256; j++) {
      const float p = sc[j];
      if (sh.at[j] < 0) continue;
      l += p;
      if (tid < d) o = fmaf(p, conv(a.v[sh.at[j] + ((int64_t)tid << a.ps_shift) + ((k0 + j) & (ps - 1))]), o);
    }
    __syncthreads();
  }
  if (tid < d)
    VRow<QT>::put(a.o, (int64_t)(it.row0 + tok) * a.ldo + (int64_t)(hv * group + row % group) * d + tid, l == 0.0f ? 0.0f : o / l);
}


union KvEnd {
  struct {
    float m[RTQ_KV_JOINED], w[RTQ_KV_JOINED];  // [row][part]: maxima, sums; then weights
    f4 o[256];
  } j;
  KvAgain again;
};
// a part's values: through to memory where another workgroup of the launch reads them (through: kv_end)
__device__ __forceinline__ void kv_part_put(bool through, float* p, float x, float y) {
  const float2 v = {x, y};
  if (through) __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, v), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  else *reinterpret_cast<float2*>(p) = v;
}
__device__ __forceinline__ void kv_part_put(bool through, float* p, f4 v) {
  if (through) kv_part_put(true, p, v[0], v[1]), kv_part_put(true, p + 2, v[2], v[3]);
  else *reinterpret_cast<f4*>(p) = v;
}

// Joins the parts of a tile's rows first, first + step, ... (with 256 threads): what counts is how many loads are under way.
// nan: room for the tile's rows: those that are not numbers are marked, and left.
template <int QT>
__device__ __forceinline__ void kv_join(const KvAttendArgs& a, const KvItem& it, const KvTile& t, int TM, int D, int from, int step, int* nan, KvEnd& sh) {
  const int tid = threadIdx.x, lane = tid & 63, group = a.group, ns = it.splits, V = D / 4, G = 256 / V;
  const int rows = (t.rows - from + step - 1) / step;
  if (rows <= 0) return;
  __syncthreads();
  // A thread takes four elements of a row; of few rows some threads share a row's parts.
  int share = 1;
  while (2 * share * rows <= G) share *= 2;
  const int c = tid % V * 4, gr = tid / V, first = gr % share;
  f4 x[16];
  const auto fetch = [&](int r, int i) {
#pragma unroll
    for (int u = 0; u < 16; u++) {
      x[u] = f4{0.0f, 0.0f, 0.0f, 0.0f};
      if (r < rows && c < a.d && i + u * share < ns)
        x[u] = *reinterpret_cast<const f4*>(a.part + ((int64_t)(it.slot + i + u * share) * TM + from + r * step) * D + c);
    }
  };
  fetch(gr / share, first);  // (under way beside the weights)
  // the parts' weights: every maximum and sum at once, then a thread a row of few parts or a wave a row of many
  for (int i = tid; i < rows * ns; i += 256) {
    const float* ml = a.ml + ((int64_t)(it.slot + i % ns) * TM + from + i / ns * step) * 2;
    sh.j.m[i] = ml[0], sh.j.w[i] = ml[1];
  }
  __syncthreads();
  const bool few = ns <= 8;
  const int part0 = few ? 0 : lane, parts = few ? 1 : 64;
  for (int r = few ? tid : tid >> 6; r < rows; r += few ? 256 : 4) {
    float *m = sh.j.m + r * ns, *w = sh.j.w + r * ns;
    float mx = -INFINITY, ls = 0.0f;
    int dead = 0;
    for (int i = part0; i < ns; i += parts) mx = fmaxf(mx, m[i]), dead |= w[i] == -1.0f;
    if (!few) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) mx = fmaxf(mx, __shfl_xor(mx, d)), dead |= __shfl_xor(dead, d);
    }
    for (int i = part0; i < ns; i += parts) {
      const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[i] - mx);
      ls += f * w[i];
      m[i] = f;
    }
    if (!few) {
#pragma unroll
      for (int d = 1; d < 64; d <<= 1) ls += __shfl_xor(ls, d);
    }
    const bool bad = !dead && ls != ls;
    nan[from + r * step] = bad;
    const float inv = dead || ls == 0.0f ? 0.0f : 1.0f / ls;
    // (a row that sees nothing is 0, also where infinite scores of held keys, which are not its own, make m NaN)
    for (int i = part0; i < ns; i += parts) w[i] = bad ? NAN : inv == 0.0f ? 0.0f : m[i] * inv;
  }
  __syncthreads();
  for (int r0 = 0; r0 < rows; r0 += G / share) {
    const int r = r0 + gr / share;
    const float* w = sh.j.w + min(r, rows - 1) * ns;
    f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int i = first; i < ns; i += 16 * share) {
      if (r0 > 0 || i > first) fetch(r, i);
#pragma unroll
      for (int u = 0; u < 16; u++)
        if (i + u * share < ns && w[i + u * share] != 0.0f) o += w[i + u * share] * x[u];
    }
    if (share > 1) {
      __syncthreads();
      sh.j.o[tid] = o;
      __syncthreads();
      if (first == 0)
        for (int i = 1; i < share; i++) o += sh.j.o[tid + i * V];
    }
    if (first == 0 && r < rows && c < a.d && w[0] == w[0]) {
      const int row = t.row_lo + from + r * step;
      const int64_t out = (int64_t)(it.row0 + row / group) * a.ldo + (int64_t)(it.hv * group + row % group) * a.d + c;
#pragma unroll
      for (int e = 0; e < 4; e++) VRow<QT>::put(a.o, out + e, o[e]);
    }
  }
}

// the marked rows of a tile (first, first + step, ...) by the formula
template <int QT, int CT>
__device__ __forceinline__ void kv_rows_again(const KvAttendArgs& a, const KvItem& it, const KvTile& t, int from, int step, const int* nan, KvAgain& sh) {
  __syncthreads();
  uint32_t any = 0;
  for (int r = threadIdx.x & 63; r < t.rows; r += 64) any |= r % step == from && nan[r];
  if (!__any(any)) return;
  for (int r = from; r < t.rows; r += step)
    if (nan[r]) kv_row_again<QT, CT>(a, it, t.row_lo + r, sh);
}

// After a workgroup's item (of 256 threads): nan[r] marks rows of a tile of one part that are to be done again; a part of
// a split tile is counted, and the last joins the parts.  sh: the workgroup's shared memory, free by now.
template <int QT, int CT, int D, int TM>
__device__ __forceinline__ void kv_end(const KvAttendArgs& a, const KvItem& it, const KvTile& t, int* nan, int* last, KvEnd& sh) {
  if (it.slot >= 0) {
    if (!a.fused) return;
    // The part's stores go through to memory (kv_part_put): once a wave has none under way they are there for every XCD, and
    // the part may be counted.  (Ordinary stores and a release would write back all that the XCD's L2 holds, in every
    // workgroup: 30 us of a call of 512.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    int* count = kv_arrived + (it.slot >> 1);
    if (threadIdx.x == 0) {
      const int n = __hip_atomic_fetch_add(count, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      if (n == it.splits - 1) __hip_atomic_store(count, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      *last = n == it.splits - 1;
    }
    __syncthreads();
    if (!*last) return;
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    kv_join<QT>(a, it, t, TM, D, 0, 1, nan, sh);
  }
  kv_rows_again<QT, CT>(a, it, t, 0, 1, nan, sh.again);
}

// ---- small tiles: 16 rows, four waves that share the tile's slots, operands straight from the cache
template <int CT, bool QF, int D, bool FULL>
__device__ __forceinline__ void kv_attend(const KvAttendArgs& a) {
  constexpr int DC = D / 32, DT = D / 16, TM = 16, LDR = D + 4;
  constexpr int NS = QF ? (CT == VT_F16 ? 2 : 3) : 1, NP = QF ? NS : 2;
  typedef VRow<QF ? VT_F32 : CT> Q;
  struct Main {
    float o[4][TM][LDR];
    float ml[4][TM][2];
    KvSeen seen[TM];
    uint16_t up[RTQ_KV_TREE];
  };
  union Shared {
    Main m;
    KvEnd end;
  };
  __shared__ Shared all;
  __shared__ int nan_row[TM], is_last;
  Main& sh = all.m;
  KvItem it;
  if (!kv_plan(a, TM, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int group = a.group, d = FULL ? D : a.d, ps = 1 << a.ps_shift;
  const KvTile tl = kv_tile(a, TM, it);
  const int row_lo = tl.row_lo, rows = tl.rows, k_hi = tl.k_hi;
  const bool tree = a.parents != nullptr;
  const int row = row_lo + min(li, rows - 1), tok = row / group;  // of this lane's column (tok: among the sequence's new tokens)
  const int64_t head = (int64_t)d << a.ps_shift, pstride = head * a.nkv;
  const auto page_of = [&](int k0) { return kv_page(a.s, it.seq, k0, a.ps_shift); };
  const auto base_of = [&](int pg) { return ((unsigned)pg < (unsigned)a.n_pages ? pg : 0) * pstride + it.hv * head; };
  u4v kf[2][DC], vf[DT];
  const uint32_t k_at = (uint32_t)((8 * (li >> 2) + (li & 3)) * d + 8 * g) * 2, v_at = (uint32_t)((li << a.ps_shift) + 8 * g) * 2;
  const auto load_k = [&](int k0, int pg) {
    const char* base = reinterpret_cast<const char*>(a.k + base_of(pg) + (int64_t)(k0 & (ps - 1)) * d);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int c = 0; c < DC; c++) {
        kf[t][c] = u4v{0, 0, 0, 0};
        if (FULL || 32 * c + 8 * g < d) kf[t][c] = *reinterpret_cast<const u4v*>(base + k_at + (4 * t * d + 32 * c) * 2);
      }
  };
  const auto load_v = [&](int k0, int pg) {
    const char* base = reinterpret_cast<const char*>(a.v + base_of(pg) + (k0 & (ps - 1)));
#pragma unroll
    for (int t = 0; t < DT; t++)
      if (FULL || 16 * t < d) vf[t] = *reinterpret_cast<const u4v*>(base + ((int64_t)(32 * t) << a.ps_shift) + v_at);
  };
  int k0 = tl.k_lo + 32 * wv;
  int pg = 0, pn = 0;
  if (k0 < k_hi) {
    pg = page_of(k0);
    pn = page_of(k0 + 128);
    load_k(k0, pg);
    load_v(k0, pg);
  }
  constexpr bool SCALED = QF && CT == VT_F16;
  u4v qf[NS][DC];
  const int64_t at = (int64_t)(it.row0 + tok) * a.ldq + (int64_t)(it.hv * group + row % group) * d;
  float sc = a.scale2, x[QF ? DC : 1][8] = {};
#pragma unroll
  for (int c = 0; c < DC; c++) {
    const bool in = (FULL || 32 * c + 8 * g < d) && li < rows;
    if constexpr (QF) {
      if (in) {
        const u4v r1 = Q::load(a.q, at + 32 * c + 8 * g), r2 = Q::load(a.q, at + 32 * c + 8 * g + 4);
#pragma unroll
        for (int e = 0; e < 4; e++) x[c][e] = Q::get(r1, e), x[c][4 + e] = Q::get(r2, e);
      }
    } else {
      qf[0][c] = u4v{0, 0, 0, 0};
      if (in) qf[0][c] = Q::load(a.q, at + 32 * c + 8 * g);
    }
  }
  if constexpr (QF) {
    int up = 0;
    if constexpr (SCALED) {
      float mx = 0.0f;
#pragma unroll
      for (int c = 0; c < DC; c++)
#pragma unroll
        for (int e = 0; e < 8; e++) mx = fmaxf(mx, fabsf(x[c][e]));
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      up = kv_row_shift(mx);
      sc = ldexpf(a.scale2, -up);
    }
#pragma unroll
    for (int c = 0; c < DC; c++) {
      if constexpr (SCALED)
#pragma unroll
        for (int e = 0; e < 8; e++) x[c][e] = ldexpf(x[c][e], up);
      u4v pl[NS];
      kv_planes<CT, NS>(x[c], pl);
#pragma unroll
      for (int i = 0; i < NS; i++) qf[i][c] = pl[i];
    }
  }
  if (tree && tl.tail) kv_tree<TM, 256>(a, it, tl, sh.seen, sh.up);
  const int tok0 = row_lo / group;

  f4 acc[DT];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int t = 0; t < DT; t++) acc[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (; k0 < k_hi; k0 += 128) {
    f4 s[2];
#pragma unroll
    for (int t = 0; t < 2; t++) {
      s[t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < DC; c++)
#pragma unroll
        for (int p = 0; p < NS; p++) s[t] = kv_mfma<CT>(kf[t][c], qf[p][c], s[t]);
    }
    const int kn = k0 + 128 < k_hi ? k0 + 128 : k0;  // (the last step loads its own slots again)
    const int pgn = k0 + 128 < k_hi ? pn : pg;
    load_k(kn, pgn);
    pn = page_of(kn + 128);
    const bool there = (unsigned)pg < (unsigned)a.n_pages;
    if (k0 + 32 > it.held || k0 + 32 > k_hi || !there) {
      const int here = there ? min(max(k_hi - k0 - 8 * g, 0), 8) : 0;  // of the lane's eight slots
      uint32_t bits = tree && tl.tail ? kv_tree_bits(k0 - it.held, sh.seen[tok - tok0]) : kv_run_bits(k0 - it.held, tok);
      bits = bits >> (8 * g) & ((1u << here) - 1);
      if (li >= rows) bits = 0;
#pragma unroll
      for (int e = 0; e < 8; e++)
        if (!(bits >> e & 1)) s[e >> 2][e & 3] = -INFINITY;
      // what lies behind the last token may be anything, NaN too: zeros, so that its weight 0 makes 0 of it
#pragma unroll
      for (int t = 0; t < DT; t++)
        if (FULL || 16 * t < d) vf[t] = kv_clear(vf[t], here);
    }
    u4v pf[NP];
    float mx = s[0][0], p[8];
#pragma unroll
    for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[e >> 2][e & 3]);
    mx = fmaxf(mx, __shfl_xor(mx, 16));
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(m, mx * sc), mu = mn == -INFINITY ? 0.0f : mn;
    const float al = __builtin_amdgcn_exp2f(m - mu);
    m = mn;
    float sum = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) {
      p[e] = __builtin_amdgcn_exp2f(fmaf(s[e >> 2][e & 3], sc, kKvUp<CT> - mu));
      sum += p[e];
    }
    l = l * al + sum;
    if (__any(al != 1.0f)) {
#pragma unroll
      for (int t = 0; t < DT; t++) acc[t] *= al;
    }
    kv_planes<CT, NP>(p, pf);
#pragma unroll
    for (int t = 0; t < DT; t++)
      if (FULL || 16 * t < d)
#pragma unroll
        for (int q = 0; q < NP; q++) acc[t] = kv_mfma<CT>(vf[t], pf[q], acc[t]);
    load_v(kn, pgn);
    pg = pgn;
  }
  // the four waves' parts
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  int nan = 0;
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int r = 0; r < 4; r++) nan |= (FULL || 16 * t < d) && acc[t][r] != acc[t][r];
  nan |= __shfl_xor(nan, 16);
  nan |= __shfl_xor(nan, 32);
  if (g == 0) sh.ml[wv][li][0] = m, sh.ml[wv][li][1] = nan ? NAN : l;
  __syncthreads();
  float top = -INFINITY;
#pragma unroll
  for (int w = 0; w < 4; w++) top = fmaxf(top, sh.ml[w][li][0]);
  const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - top);
#pragma unroll
  for (int t = 0; t < DT; t++)
    if (FULL || 16 * t < d) *reinterpret_cast<f4*>(&sh.o[wv][li][16 * t + 4 * g]) = acc[t] * f;
  __syncthreads();
  const int vecs = d / 4, slot = it.slot + it.split;
  for (int i = threadIdx.x; i < rows * vecs; i += 256) {
    const int r = i / vecs, c = i % vecs * 4;
    float mx = -INFINITY, ls = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; w++) mx = fmaxf(mx, sh.ml[w][r][0]);
#pragma unroll
    for (int w = 0; w < 4; w++) ls += sh.ml[w][r][1] * (mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(sh.ml[w][r][0] - mx));
    f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 0; w < 4; w++) o += *reinterpret_cast<const f4*>(&sh.o[w][r][c]);
    const bool dead = tree && tl.tail && kv_dead(sh.seen[(row_lo + r) / group - tok0], (row_lo + r) / group);
    if (it.slot >= 0) {
      kv_part_put(a.fused, a.part + ((int64_t)slot * TM + r) * D + c, o);
      if (c == 0) kv_part_put(a.fused, a.ml + ((int64_t)slot * TM + r) * 2, mx, dead ? -1.0f : ls);
    } else {
      const bool again = !dead && ls != ls;
      if (c == 0) nan_row[r] = again;
      if (again) continue;
      const int tk = (row_lo + r) / group;
      const int64_t at = (int64_t)(it.row0 + tk) * a.ldo + (int64_t)(it.hv * group + (row_lo + r) % group) * d + c;
      const float inv = dead || ls == 0.0f ? 0.0f : 1.0f / ls;
#pragma unroll
      for (int e = 0; e < 4; e++) Q::put(a.o, at + e, inv == 0.0f ? 0.0f : o[e] * inv);
    }
  }
  kv_end<QF ? VT_F32 : CT, CT, D, TM>(a, it, tl, nan_row, &is_last, all.end);
}

// ---- large tiles: four waves of 32 rows, 64 slots at a time through LDS for all of them
//
// The tile's keys and values reach LDS by buffer loads with the LDS destination, into a ring of R buffers (what
// two workgroups a CU leave room for: 3 at a head size of 64, else 2): the next slots are on their way while these are multiplied.  A unit is 32 slots (of one page): keys [slot][d / 8] and
// values [d][4] of 16-byte chunks, a chunk's place swapped by its row so that 16 lanes' reads fall on different
// banks (64 of 4 bytes); loads past a head's page (rows of a smaller head size, pages that are not there) give zeros.
// MFMA 32x32x16, again S^T = K q^T and o^T = V^T p^T: key row m of a unit is slot 16 (m / 16) + 8 (m / 4 % 2) +
// 4 (m / 8 % 2) + m % 4, so a lane's 16 scores are its operands of the second product in order.
// the key rows of lanes 0 .. 15 (and 16 .. 31), by their slots, get 16 places of a row of 16 chunks or more, or eight of each
// of two neighbouring rows
template <int CH>
__device__ __forceinline__ int kv_swap(int slot) {
  const int row = (slot & 3) | (slot >> 1 & 4) | (slot << 1 & 8);  // the MFMA row of the slot, modulo 16
  return CH >= 16 ? row : row >> 1;
}

template <int CT, bool QF, int D, bool FULL, int R>
__device__ __forceinline__ void kv_attend_big(const KvAttendArgs& a) {
  constexpr int NW = 4, DK = D / 16, DT = D / 32, CH = D / 8, TM = 32 * NW, T = 64 * NW;
  static_assert(TM <= RTQ_KV_ROWS, "a join's tables");
  constexpr int NS = QF ? (CT == VT_F16 ? 2 : 3) : 1, NP = QF ? NS : 2;
  constexpr int UK = 32 * CH, UV = D * 4, UNIT = UK + UV;  // chunks
  typedef VRow<QF ? VT_F32 : CT> Q;
  struct Main {
    u4v st[R][2][UNIT];
    KvSeen seen[TM];
  };
  union Shared {
    Main m;
    struct {
      KvEnd e;
      int nan_row[TM], is_last;
    } end;
  };
  __shared__ Shared all;
  Main& sh = all.m;
  KvItem it;
  if (!kv_plan(a, TM, blockIdx.x, it)) return;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q32 = lane & 31, h = lane >> 5;
  const int group = a.group, d = FULL ? D : a.d, ps = 1 << a.ps_shift;
  const KvTile tl = kv_tile(a, TM, it);
  const int row_lo = tl.row_lo, rows = tl.rows, k_hi = tl.k_hi;
  const bool tree = a.parents != nullptr;
  const int row = 32 * wv + q32, rc = row_lo + min(row, rows - 1), tok = rc / group, tok0 = row_lo / group;
  const bool busy = 32 * wv < rows;  // (waves without rows only help with the loads)

  const int64_t head = (int64_t)d << a.ps_shift, pstride = head * a.nkv;
  // this wave's loads of a unit: chunk places (i NW + wv) 64 + lane of the keys, then of the values
  constexpr int LK = UK / T, LV = UV / T;
  static_assert(UK % T == 0 && UV % T == 0, "whole loads");
  uint32_t ko[LK], vo[LV];
#pragma unroll
  for (int i = 0; i < LK; i++) {
    const int p = (i * NW + wv) * 64 + lane, slot = p / CH, c = (p % CH) ^ kv_swap<CH>(slot);
    ko[i] = FULL || 8 * c < d ? (uint32_t)(slot * d + 8 * c) * 2 : 0x80000000u;
  }
#pragma unroll
  for (int i = 0; i < LV; i++) {
    const int p = (i * NW + wv) * 64 + lane, r = p / 4, c = (p % 4) ^ (r >> 2 & 3);
    vo[i] = FULL || r < d ? (uint32_t)((r << a.ps_shift) + 8 * c) * 2 : 0x80000000u;
  }
  uint32_t ahead = 0;  // of the slots under way: bit u, unit u's page is not there
  int page[2];         // of the slots to load next
  const auto pages = [&](int k0) {
#pragma unroll
    for (int u = 0; u < 2; u++) page[u] = kv_page(a.s, it.seq, k0 + 32 * u, a.ps_shift);
  };
  const auto issue = [&](int buf, int k0) {
    ahead = 0;
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int at = k0 + 32 * u, pg = page[u];
      const bool there = (unsigned)pg < (unsigned)a.n_pages;
      const int64_t base = (there ? pg : 0) * pstride + it.hv * head;
      const uint32_t bytes = there ? (uint32_t)head * 2 : 0u, in = there ? (uint32_t)(at & (ps - 1)) : 0u;
      ahead |= there ? 0u : 1u << u;
      const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.k + base), (short)0, bytes, 0x00020000);
      const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(a.v + base), (short)0, bytes, 0x00020000);
      u4v* s = sh.st[buf][u];
#pragma unroll
      for (int i = 0; i < LK; i++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, RTQ_LDSP(s + (i * NW + wv) * 64), 16, ko[i], in * (uint32_t)d * 2, 0, 0);
#pragma unroll
      for (int i = 0; i < LV; i++)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, RTQ_LDSP(s + UK + (i * NW + wv) * 64), 16, vo[i], in * 2, 0, 0);
    }
  };
  pages(tl.k_lo);
  if (tl.k_lo < k_hi) issue(0, tl.k_lo);
  uint32_t missing[R];  // ahead of the slots in turn
  missing[0] = ahead;
  pages(tl.k_lo + 64);

  constexpr bool SCALED = QF && CT == VT_F16;
  u4v qf[NS][DK];
  float sc = a.scale2;
  {
    const int64_t at = (int64_t)(it.row0 + tok) * a.ldq + (int64_t)(it.hv * group + rc % group) * d + 8 * h;
    int up = 0;
    if constexpr (SCALED) {
      float mx = 0.0f;
#pragma unroll
      for (int c = 0; c < DK; c++)
        if (FULL || 16 * c < d) {
          const u4v r1 = Q::load(a.q, at + 16 * c), r2 = Q::load(a.q, at + 16 * c + 4);
#pragma unroll
          for (int e = 0; e < 4; e++) mx = fmaxf(mx, fmaxf(fabsf(Q::get(r1, e)), fabsf(Q::get(r2, e))));
        }
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      up = kv_row_shift(mx);
      sc = ldexpf(a.scale2, -up);
    }
#pragma unroll
    for (int c = 0; c < DK; c++) {
      if constexpr (QF) {
        float x[8] = {};
        if (FULL || 16 * c < d) {
          const u4v r1 = Q::load(a.q, at + 16 * c), r2 = Q::load(a.q, at + 16 * c + 4);
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = Q::get(r1, e), x[4 + e] = Q::get(r2, e);
        }
        if constexpr (SCALED)
#pragma unroll
          for (int e = 0; e < 8; e++) x[e] = ldexpf(x[e], up);
        u4v pl[NS];
        kv_planes<CT, NS>(x, pl);
#pragma unroll
        for (int i = 0; i < NS; i++) qf[i][c] = pl[i];
      } else {
        qf[0][c] = u4v{0, 0, 0, 0};
        if (FULL || 16 * c < d) qf[0][c] = Q::load(a.q, at + 16 * c);
      }
    }
  }
  if (tree && tl.tail) kv_tree<TM, T>(a, it, tl, sh.seen, reinterpret_cast<uint16_t*>(sh.st[R - 1]));  // (not loaded into yet)

  f16v acc[DT];
  float m = -INFINITY, l = 0.0f;
#pragma unroll
  for (int t = 0; t < DT; t++) acc[t] = f16v{};
  // this lane's chunks: key row q32's slot, elements 16 c + 8 h; value row 32 t + q32, slots 16 s + 8 h
  const int kslot = 16 * (q32 >> 4) + 8 * (q32 >> 2 & 1) + 4 * (q32 >> 3 & 1) + (q32 & 3), kx = kv_swap<CH>(kslot), vx = q32 >> 2 & 3;
  if constexpr (R == 3) {
    if (tl.k_lo + 64 < k_hi) issue(1, tl.k_lo + 64);
    missing[1] = ahead;
    pages(tl.k_lo + 128);
  }
  int buf = 0, k0 = tl.k_lo;
  uint32_t lost = 0;
  const auto advance = [&] {
    asm volatile("" ::: "memory");
    if (R == 3 && k0 + 64 < k_hi) __builtin_amdgcn_s_waitcnt(vm_wait_imm(2 * (LK + LV)));
    else __builtin_amdgcn_s_waitcnt(vm_wait_imm(0));
    lds_barrier();  // these 64 slots have landed, and every wave is done with the buffer before them
    asm volatile("" ::: "memory");
    lost = missing[0];
    constexpr int A = R - 1;
    if (k0 + 64 * A < k_hi) issue(buf == 0 ? A : buf - 1, k0 + 64 * A);
#pragma unroll
    for (int i = 0; i + 1 < A; i++) missing[i] = missing[i + 1];
    missing[A - 1] = ahead;
    pages(k0 + 64 * A + 64);
  };
  const auto step = [&](auto some) {  // some: not every row sees all of the 64 slots
    constexpr bool MASKED = decltype(some)::value;
    f16v s[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const u4v* kt = sh.st[buf][u] + kslot * CH;
      s[u] = f16v{};
#pragma unroll
      for (int c = 0; c < DK; c++) {
        if (!FULL && 16 * c >= d) break;
        const u4v kf = kt[(2 * c + h) ^ kx];
#pragma unroll
        for (int p = 0; p < NS; p++) s[u] = kv_mfma32<CT>(kf, qf[p][c], s[u]);
      }
    }
    const int here = min(k_hi - k0, 64);  // slots that hold tokens
    if constexpr (MASKED) {
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int nw = k0 + 32 * u - it.held, left = min(max(here - 32 * u, 0), 32);
        uint32_t bits = tree && tl.tail ? kv_tree_bits(nw, sh.seen[tok - tok0]) : kv_run_bits(nw, tok);
        if (left < 32) bits &= (1u << left) - 1;
        if (lost >> u & 1) bits = 0;
#pragma unroll
        for (int e = 0; e < 16; e++)
          if (!(bits >> (16 * (e >> 3) + (e & 7)) >> (8 * h) & 1)) s[u][e] = -INFINITY;
      }
    }
    float mx = s[0][0];
#pragma unroll
    for (int e = 1; e < 32; e++) mx = fmaxf(mx, s[e >> 4][e & 15]);
    mx = fmaxf(mx, __shfl_xor(mx, 32));
    const float mn = fmaxf(m, mx * sc);
    if (__any(mn > m + kKvLag)) {
      const float al = __builtin_amdgcn_exp2f(m - (mn == -INFINITY ? 0.0f : mn));
      l *= al;
#pragma unroll
      for (int t = 0; t < DT; t++) acc[t] *= al;
      m = mn;
    }
    const float off = kKvUp<CT> - (m == -INFINITY ? 0.0f : m);
    u4v pf[4][NP];
    float sum = 0.0f;
#pragma unroll
    for (int g = 0; g < 4; g++) {
      float p[8];
#pragma unroll
      for (int e = 0; e < 8; e++) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(s[g >> 1][8 * (g & 1) + e], sc, off));
        sum += p[e];
      }
      kv_planes<CT, NP>(p, pf[g]);
    }
    l += sum;
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const u4v* vt = sh.st[buf][g >> 1] + UK + q32 * 4;
#pragma unroll
      for (int t = 0; t < DT; t++) {
        if (!FULL && 32 * t >= d) break;
        u4v vf = vt[128 * t + ((2 * (g & 1) + h) ^ vx)];
        if constexpr (MASKED) vf = kv_clear(vf, min(max(here - 16 * g - 8 * h, 0), 8));
#pragma unroll
        for (int p = 0; p < NP; p++) acc[t] = kv_mfma32<CT>(vf, pf[g][p], acc[t]);
      }
    }
  };
  // the slots that every row sees whole, then the others (and what lies behind a page that is not there)
  const int plain = min(tree ? it.held : it.held + tok0 + 1, k_hi);
  for (; k0 + 64 <= plain && !missing[0]; k0 += 64, buf = buf + 1 == R ? 0 : buf + 1) {
    advance();
    if (busy) step(std::false_type{});
  }
  for (; k0 < k_hi; k0 += 64, buf = buf + 1 == R ? 0 : buf + 1) {
    advance();
    if (busy) step(std::true_type{});
  }
  l += __shfl_xor(l, 32);
  int nan = 0;
#pragma unroll
  for (int t = 0; t < DT; t++)
#pragma unroll
    for (int e = 0; e < 16; e++) nan |= (FULL || 32 * t + 8 * (e >> 2) + 4 * h < d) && acc[t][e] != acc[t][e];
  nan |= __shfl_xor(nan, 32);
  if (nan) l = NAN;
  const bool dead = tree && tl.tail && kv_dead(sh.seen[tok - tok0], tok);
  __syncthreads();  // (the end's shared memory lies over the blocks')
  if (row < rows) {
    const int64_t slot = it.slot + it.split;
    const bool again = !dead && l != l;
    if (it.slot >= 0) {
      float* out = a.part + (slot * TM + row) * D;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          kv_part_put(a.fused, out + 32 * t + 8 * i + 4 * h, f4{acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]});
      if (h == 0) kv_part_put(a.fused, a.ml + (slot * TM + row) * 2, m, dead ? -1.0f : l);
    } else if (!again) {
      const int64_t at = (int64_t)(it.row0 + tok) * a.ldo + (int64_t)(it.hv * group + rc % group) * d + 4 * h;
      const float inv = dead || l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
      for (int t = 0; t < DT; t++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (FULL || 32 * t + 8 * i < d)
#pragma unroll
            for (int e = 0; e < 4; e++) Q::put(a.o, at + 32 * t + 8 * i + e, inv == 0.0f ? 0.0f : acc[t][4 * i + e] * inv);
    }
    if (h == 0) all.end.nan_row[row] = again;
  }
  kv_end<QF ? VT_F32 : CT, CT, D, TM>(a, it, tl, all.end.nan_row, &all.end.is_last, all.end.e);
}

#define RTQ_KV_ATTEND(SUF, CT, QF, D, FULL) \
  extern "C" __global__ __launch_bounds__(256, D > 128 ? 1 : 2) void rtq_kv_attend##SUF(KvAttendArgs a) { kv_attend<CT, QF, D, FULL>(a); }
#define RTQ_KV_BIG(SUF, CT, QF, D, FULL, R) \
  extern "C" __global__ __launch_bounds__(256, 2) void rtq_kv_attend##SUF(KvAttendArgs a) { kv_attend_big<CT, QF, D, FULL, R>(a); }
#define RTQ_KV_ATTENDS(SUF, CT, QF)                  \
  RTQ_KV_ATTEND(16_64_##SUF, CT, QF, 64, true)       \
  RTQ_KV_ATTEND(16_128_##SUF, CT, QF, 128, true)     \
  RTQ_KV_ATTEND(16_128p_##SUF, CT, QF, 128, false)   \
  RTQ_KV_ATTEND(16_256p_##SUF, CT, QF, 256, false)   \
  RTQ_KV_BIG(_big_64_##SUF, CT, QF, 64, true, 3)     \
  RTQ_KV_BIG(_big_128_##SUF, CT, QF, 128, true, 2)   \
  RTQ_KV_BIG(_big_128p_##SUF, CT, QF, 128, false, 2) \
  RTQ_KV_BIG(_big_256p_##SUF, CT, QF, 256, false, 2)
RTQ_KV_ATTENDS(f32_f16, VT_F16, true)
RTQ_KV_ATTENDS(f32_bf16, VT_BF16, true)
RTQ_KV_ATTENDS(f16, VT_F16, false)
RTQ_KV_ATTENDS(bf16, VT_BF16, false)

// the joining kernel: the workgroup of part i of n joins its tile's rows i, i + n, ...  It takes the item from the attention's
// workgroup of that part (making the plan again took 2 us of each launch).  Items that no workgroup has left (of tiles that the
// plan leaves out, where sequences overlap) are another call's: what does not name rows of this one is passed over.
template <int QT, int CT>
__device__ __forceinline__ void kv_join_rows(const KvAttendArgs& a) {
  __shared__ KvEnd sh;
  __shared__ int nan[128];
  typedef const __attribute__((address_space(4))) int32_t* cptr;
  const int at = blockIdx.x;
  const cptr items = reinterpret_cast<cptr>(reinterpret_cast<uintptr_t>(a.items));
  int f[RTQ_KV_ITEM];
#pragma unroll
  for (int i = 0; i < RTQ_KV_ITEM; i++) f[i] = items[(1 + at) * RTQ_KV_ITEM + i];
  if (at >= items[0]) return;
  const KvItem it = {f[0], f[1], f[2], f[3], f[4], f[5], f[6], f[7], f[8], f[9], f[10]};
  const bool sound = it.seq >= 0 && it.seq < a.s.b && it.row0 >= 0 && it.cnt >= 1 && it.cnt <= a.s.n - it.row0 && it.held >= 0 &&
                     it.total >= 0 && (it.total == 0 || (it.total - 1) >> a.ps_shift < a.s.ldt) && it.hv >= 0 && it.hv < a.nkv && it.tile >= 0 &&
                     (int64_t)it.tile * a.tm < (int64_t)it.cnt * a.group && it.splits >= 2 && it.splits <= RTQ_KV_JOIN && it.split >= 0 &&
                     it.split < it.splits && it.slot + it.split == at && it.slot + it.splits <= a.slots;
  if (!sound) return;
  const KvTile t = kv_tile(a, a.tm, it);
  if (it.split >= t.rows) return;
  kv_join<QT>(a, it, t, a.tm, a.D, it.split, it.splits, nan, sh);
  kv_rows_again<QT, CT>(a, it, t, it.split, it.splits, nan, sh.again);
}
extern "C" __global__ __launch_bounds__(256) void rtq_kv_join_f32_f16(KvAttendArgs a) { kv_join_rows<VT_F32, VT_F16>(a); }
extern "C" __global__ __launch_bounds__(256) void rtq_kv_join_f32_bf16(KvAttendArgs a) { kv_join_rows<VT_F32, VT_BF16>(a); }
extern "C" __global__ __launch_bounds__(256) void rtq_kv_join_f16(KvAttendArgs a) { kv_join_rows<VT_F16, VT_F16>(a); }
extern "C" __global__ __launch_bounds__(256) void rtq_kv_join_bf16(KvAttendArgs a) { kv_join_rows<VT_BF16, VT_BF16>(a); }
