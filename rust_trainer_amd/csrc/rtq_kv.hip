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
#define RTQ_KV_SLOTS (1 << 30)  // most slots of a sequence that are looked at
// tokens held by sequence i, no more than its table's slots
__device__ __forceinline__ int kv_held(const int32_t* lens, int i, int ldt, int ps_shift) {
  return (int)min((int64_t)max(lens[i], 0), min((int64_t)ldt << ps_shift, (int64_t)RTQ_KV_SLOTS));
}

// ------------------------------------------------------------------ append
// One token a workgroup (its KV heads' values beside, 32 tokens a workgroup): 16 lanes take a head, a lane
// eight elements at a time, four pairs of the rotation.  The angles are turns: position x freq in 64 bits,
// of which the whole turns are dropped before sine and cosine are taken in 32 (at position 10^5 a 32-bit
// angle is off by 4e-3), once per lane and pair for all of its heads.
template <int XT, int CT>
__device__ __forceinline__ void kv_append_rows(const KvAppendArgs& a, int tok, int held, int idx, int seq) {
  typedef VRow<XT> X;
  typedef VRow<CT> C;
  const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, l16 = lane & 15;
  const int half = a.rot / 2, units = a.d / 8;
  const int64_t slot = (int64_t)held + idx;
  const int p = (int)(slot >> a.ps_shift), ps = 1 << a.ps_shift;
  const int pid = p < a.s.ldt ? a.s.table[(int64_t)seq * a.s.ldt + p] : -1;
  const bool stored = (unsigned)pid < (unsigned)a.n_pages;
  const double pos = a.pos ? (double)a.pos[tok] : (double)slot;
  const int heads = (a.q ? a.nh : 0) + a.nkv, nq = a.q ? a.nh : 0;
  // this lane's units: l16 and l16 + 16 (d <= 256)
  float cs[2][4], sn[2][4];
  const bool whole = a.rot % 8 == 0;
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = 4 * (l16 + 16 * u) + e;
      cs[u][e] = 1.0f, sn[u][e] = 0.0f;
      if (i < half) {
        double t = pos * a.freq[i];
        t -= rint(t);
        float sv, cv;
        sincospif(2.0f * (float)t, &sv, &cv);
        cs[u][e] = cv, sn[u][e] = sv;
      }
    }
  for (int h = wv * 4 + (lane >> 4); h < heads; h += 16) {
    const bool isq = h < nq;
    const int hh = isq ? h : h - nq;
    const void* x = isq ? a.q : a.kx;
    const int64_t at = isq ? (int64_t)tok * a.ldq + (int64_t)hh * a.d : (int64_t)tok * a.ldk + (int64_t)hh * a.d;
    const float* w = isq ? a.q_norm : a.k_norm;
    uint16_t* kd = a.k + ((((int64_t)(stored ? pid : 0) * a.nkv + hh) << a.ps_shift) + (slot & (ps - 1))) * a.d;
    const int64_t qd = (int64_t)tok * a.ldo + (int64_t)hh * a.d;
    const auto put = [&](int j, float y) {
      if (isq) X::put(a.qo, qd + j, y);
      else if (stored) C::put(kd, j, y);
    };
    if (!whole) {  // a rotation that ends inside a unit of eight: element by element
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
      for (int i = l16; i < half; i += 16) {
        const int ia = a.neox ? i : 2 * i, ib = a.neox ? i + half : 2 * i + 1;
        double t = pos * a.freq[i];
        t -= rint(t);
        float sv, cv;
        sincospif(2.0f * (float)t, &sv, &cv);
        const float x1 = get(ia), x2 = get(ib);
        put(ia, x1 * cv - x2 * sv), put(ib, x2 * cv + x1 * sv);
      }
      continue;
    }
    // unit u covers elements o1 .. o1 + 3 and o2 .. o2 + 3: the two sides of four pairs, or eight in a row
    float v[2][8];
    int o1[2], o2[2];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const int un = l16 + 16 * u;
      if (un >= units) continue;
      const bool split = a.neox && un < a.rot / 8;
      o1[u] = split ? 4 * un : 8 * un;
      o2[u] = split ? half + 4 * un : 8 * un + 4;
      if constexpr (XT == VT_F32) {
        const u4v r1 = X::load(x, at + o1[u]), r2 = X::load(x, at + o2[u]);
#pragma unroll
        for (int e = 0; e < 4; e++) v[u][e] = X::get(r1, e), v[u][4 + e] = X::get(r2, e);
      } else if (split) {
#pragma unroll
        for (int e = 0; e < 4; e++) v[u][e] = X::one(x, at + o1[u] + e), v[u][4 + e] = X::one(x, at + o2[u] + e);
      } else {
        const u4v r = X::load(x, at + o1[u]);
#pragma unroll
        for (int e = 0; e < 8; e++) v[u][e] = X::get(r, e);
      }
    }
    if (w) {  // RMS norm of the head: (x / rms) (w + off)
      float s = 0.0f;
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (l16 + 16 * u < units)
#pragma unroll
          for (int e = 0; e < 8; e++) s += v[u][e] * v[u][e];
#pragma unroll
      for (int m = 1; m <= 8; m <<= 1) s += __shfl_xor(s, m);
      const float ir = __fdiv_rn(1.0f, __fsqrt_rn(__fdiv_rn(s, (float)a.d) + a.eps));
#pragma unroll
      for (int u = 0; u < 2; u++)
        if (l16 + 16 * u < units)
#pragma unroll
          for (int e = 0; e < 8; e++) v[u][e] *= ir * (w[(e < 4 ? o1[u] : o2[u] - 4) + e] + a.off);
    }
#pragma unroll
    for (int u = 0; u < 2; u++)
      if (l16 + 16 * u < a.rot / 8) {
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int ia = a.neox ? e : 2 * e, ib = a.neox ? 4 + e : 2 * e + 1;
          const float x1 = v[u][ia], x2 = v[u][ib];
          v[u][ia] = x1 * cs[u][e] - x2 * sn[u][e];
          v[u][ib] = x2 * cs[u][e] + x1 * sn[u][e];
        }
      }
#pragma unroll
    for (int u = 0; u < 2; u++) {
      if (l16 + 16 * u >= units) continue;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        put((e < 4 ? o1[u] : o2[u] - 4) + e, v[u][e]);
      }
    }
  }
}

// the sequence that row tok belongs to (-1: none), found by the workgroup's 256 threads
__device__ __forceinline__ int kv_find(const KvSeqs& s, int tok, int* found) {
  if (!s.starts) {
    const int per = s.n / s.b;
    return tok / per;
  }
  if (threadIdx.x == 0) *found = -1;
  __syncthreads();
  for (int i = threadIdx.x; i < s.b; i += 256)
    if (kv_start(s, i) <= tok && tok < kv_start(s, i + 1)) *found = i;
  __syncthreads();
  return *found;
}

template <int XT, int CT>
__device__ __forceinline__ void kv_append(const KvAppendArgs& a) {
  __shared__ int found;
  if ((int)blockIdx.x < a.s.n) {
    const int tok = blockIdx.x, seq = kv_find(a.s, tok, &found);
    if (seq < 0) return;
    kv_append_rows<XT, CT>(a, tok, kv_held(a.s.lens, seq, a.s.ldt, a.ps_shift), tok - kv_start(a.s, seq), seq);
    return;
  }
  // values: 32 tokens of one KV head, through LDS, so that neighbouring tokens are stored together
  __shared__ float tile[32][257];
  __shared__ int64_t dst[32];
  const int wg = blockIdx.x - a.s.n, hv = wg % a.nkv, t0 = wg / a.nkv * 32;
  const int nt = min(32, a.s.n - t0), ps = 1 << a.ps_shift;
  if (threadIdx.x < 32) dst[threadIdx.x] = -1;
  __syncthreads();
  if (a.s.starts) {  // each sequence names the tokens of this tile that are its own
    for (int i = threadIdx.x; i < a.s.b; i += 256) {
      const int s0 = kv_start(a.s, i), s1 = kv_start(a.s, i + 1);
      for (int t = max(s0, t0); t < min(s1, t0 + nt); t++) dst[t - t0] = (int64_t)i << 32 | (t - s0);
    }
  } else if ((int)threadIdx.x < nt) {
    const int per = a.s.n / a.s.b, t = t0 + threadIdx.x;
    dst[threadIdx.x] = (int64_t)(t / per) << 32 | (t % per);
  }
  __syncthreads();
  if (threadIdx.x < 32 && dst[threadIdx.x] >= 0) {
    const int seq = (int)(dst[threadIdx.x] >> 32), idx = (int)(dst[threadIdx.x] & 0xffffffff);
    const int64_t slot = (int64_t)kv_held(a.s.lens, seq, a.s.ldt, a.ps_shift) + idx;
    const int64_t p = slot >> a.ps_shift;
    const int pid = p < a.s.ldt ? a.s.table[(int64_t)seq * a.s.ldt + p] : -1;
    dst[threadIdx.x] = (unsigned)pid < (unsigned)a.n_pages
                           ? (((int64_t)pid * a.nkv + hv) * a.d << a.ps_shift) + (slot & (ps - 1))
                           : -1;
  }
  typedef VRow<XT> X;
  constexpr int E = X::E;
  const int vecs = a.d / E;
  for (int i = threadIdx.x; i < nt * vecs; i += 256) {
    const int t = i / vecs, c = i % vecs * E;
    const u4v r = X::load(a.vx, (int64_t)(t0 + t) * a.ldv + (int64_t)hv * a.d + c);
#pragma unroll
    for (int e = 0; e < E; e++) tile[t][c + e] = X::get(r, e);
  }
  __syncthreads();
  const int t = threadIdx.x & 31;
  if (t >= nt || dst[t] < 0) return;
  for (int c = threadIdx.x >> 5; c < a.d; c += 8) VRow<CT>::put(a.v, dst[t] + ((int64_t)c << a.ps_shift), tile[t][c]);
}

#define RTQ_KV_APPEND(NAME, XT, CT) \
  extern "C" __global__ __launch_bounds__(256) void NAME(KvAppendArgs a) { kv_append<XT, CT>(a); }
RTQ_KV_APPEND(rtq_kv_append_f32_f16, VT_F32, VT_F16)
RTQ_KV_APPEND(rtq_kv_append_f32_bf16, VT_F32, VT_BF16)
RTQ_KV_APPEND(rtq_kv_append_f16, VT_F16, VT_F16)
RTQ_KV_APPEND(rtq_kv_append_bf16, VT_BF16, VT_BF16)

// ------------------------------------------------------------------ keep
// Workgroup: one KV head of one sequence and layer.  Kept tokens ascend, so the j-th comes from a slot no
// earlier than its own: a thread that moves its elements in order, eight loads before their stores, never
// writes a slot that it has yet to read, and no two threads touch the same elements.
#define RTQ_KV_KEEP 1024
extern "C" __global__ __launch_bounds__(320) void rtq_kv_keep(KvKeepArgs a) {
  __shared__ int64_t from[RTQ_KV_KEEP], to[RTQ_KV_KEEP];  // page x slots + slot; from -1: not moved
  __shared__ int count;
  const int hv = blockIdx.x % a.nkv, seq = blockIdx.x / a.nkv;
  const int32_t* kept = a.kept + (int64_t)seq * a.ldk;
  const int held = kv_held(a.lens, seq, a.ldt, a.ps_shift), ps = 1 << a.ps_shift;
  if (threadIdx.x == 0) count = a.ldk;
  __syncthreads();
  for (int j = threadIdx.x; j < a.ldk; j += 320)  // the list ends at the first entry that does not ascend
    if (kept[j] < 0 || (j && kept[j] <= kept[j - 1])) atomicMin(&count, j);
  __syncthreads();
  const int n = count;
  for (int j = threadIdx.x; j < n; j += 320) {
    const int64_t f = (int64_t)held + kept[j], t = (int64_t)held + j;
    const int64_t fp = f >> a.ps_shift, tp = t >> a.ps_shift;
    const int fi = fp < a.ldt ? a.table[(int64_t)seq * a.ldt + fp] : -1, ti = tp < a.ldt ? a.table[(int64_t)seq * a.ldt + tp] : -1;
    const bool ok = (unsigned)fi < (unsigned)a.n_pages && (unsigned)ti < (unsigned)a.n_pages && f != t;
    from[j] = ok ? ((int64_t)fi << 32 | (f & (ps - 1))) : -1;
    to[j] = (int64_t)ti << 32 | (t & (ps - 1));
  }
  if (blockIdx.y == 0 && hv == 0 && threadIdx.x == 0 && a.after) a.after[seq] = a.lens[seq] + n;
  __syncthreads();
  const int64_t row = (int64_t)a.d << a.ps_shift;  // elements of a head's page
  uint16_t* k = a.k + blockIdx.y * a.layer;
  uint16_t* v = a.v + blockIdx.y * a.layer;
  const int c = threadIdx.x;
  const auto page = [&](int64_t at) { return ((at >> 32) * a.nkv + hv) * row; };
  if (c < a.d) {
    for (int j0 = 0; j0 < n; j0 += 8) {
      uint16_t x[8];
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j0 + j < n && from[j0 + j] >= 0) x[j] = v[page(from[j0 + j]) + ((int64_t)c << a.ps_shift) + (from[j0 + j] & 0xffffffff)];
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j0 + j < n && from[j0 + j] >= 0) v[page(to[j0 + j]) + ((int64_t)c << a.ps_shift) + (to[j0 + j] & 0xffffffff)] = x[j];
    }
  }
  const int e = (319 - c) * 8;  // keys: the last threads, 16 bytes each
  if (e < a.d) {
    for (int j0 = 0; j0 < n; j0 += 8) {
      u4v x[8];
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j0 + j < n && from[j0 + j] >= 0) x[j] = *reinterpret_cast<const u4v*>(k + page(from[j0 + j]) + (from[j0 + j] & 0xffffffff) * a.d + e);
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (j0 + j < n && from[j0 + j] >= 0) *reinterpret_cast<u4v*>(k + page(to[j0 + j]) + (to[j0 + j] & 0xffffffff) * a.d + e) = x[j];
    }
  }
}

// ------------------------------------------------------------------ attention
// Rows of one (sequence, KV head): its new tokens x the head's group of query heads, token by token; a tile
// takes TM of them.  The keys of a tile are split into ranges of C slots (one C for the call, chosen on the
// device from the sequences' lengths, so that about `target` items are made in all: the host does not
// know the lengths); an item is a tile and a range.  Tiles of one range leave o directly, others leave an
// unnormalised sum, the maximum and the sum of the weights, which rtq_kv_merge joins.
//
// A wave takes 32 slots at a time.  S^T = K q^T and o^T = V^T p^T, so that a lane holds one query row:
// key row m of tile t is slot 8 (m / 4) + 4 t + m % 4, and the lane that gets the scores of slots 8 g .. 8 g + 7
// holds them in the order in which it feeds them to the second product: the weights never leave their lane.
struct KvItem {
  int seq, row0, cnt, held, total, tile, hv, split, splits, slot, qid, C;
};

__device__ __forceinline__ int kv_wave_scan(int v) {  // inclusive
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(v, d);
    if (lane >= d) v += o;
  }
  return v;
}

// item `block` of the plan (every wave finds it by itself; a lane looks after b / 64 sequences); false: none.
// Sequences that overlap in `starts` can name more than the host counted: then nothing is joined.
template <int TM>
__device__ __forceinline__ bool kv_plan(const KvAttendArgs& a, int block, KvItem& it) {
  const int lane = threadIdx.x & 63, group = a.nh / a.nkv;
  const int per = (a.s.b + 63) / 64, i0 = lane * per, i1 = min(i0 + per, a.s.b);
  const auto look = [&](int i, int& row0, int& cnt, int& held, int& total, int& tiles) {
    row0 = kv_start(a.s, i);
    cnt = max(kv_start(a.s, i + 1) - row0, 0);
    held = kv_held(a.s.lens, i, a.s.ldt, a.ps_shift);
    total = (int)min((int64_t)held + cnt, min((int64_t)a.s.ldt << a.ps_shift, (int64_t)RTQ_KV_SLOTS));
    tiles = (int)(((int64_t)cnt * group + TM - 1) / TM);
  };
  int row0, cnt, held, total, tiles;
  double w = 0.0;
  for (int i = i0; i < i1; i++) {
    look(i, row0, cnt, held, total, tiles);
    w += (double)tiles * (double)total;
  }
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) w += __shfl_xor(w, m);
  const int C = (int)min(ceil(w * (double)a.nkv / (double)a.target / 128.0), (double)(RTQ_KV_SLOTS / 128)) * 128;
  it.C = max(C, 128);
  int items = 0, slots = 0, qids = 0;
  for (int i = i0; i < i1; i++) {
    look(i, row0, cnt, held, total, tiles);
    const int ns = max((total + it.C - 1) / it.C, 1), n = tiles * a.nkv;
    items += n * ns, qids += n, slots += ns > 1 ? n * ns : 0;
  }
  int ei = kv_wave_scan(items), es = kv_wave_scan(slots), eq = kv_wave_scan(qids);
  if (block == 0 && threadIdx.x == 63) a.desc[0] = eq <= a.qids && es <= a.slots && ei <= (int)gridDim.x ? eq : 0;
  ei -= items, es -= slots, eq -= qids;
  const uint64_t mine = __ballot(block >= ei && block < ei + items);
  if (!mine) return false;
  int ok = 0;
  if (block >= ei && block < ei + items) {
    for (int i = i0; i < i1; i++) {
      look(i, row0, cnt, held, total, tiles);
      const int ns = max((total + it.C - 1) / it.C, 1), n = tiles * a.nkv;
      if (block < ei + n * ns) {
        const int at = block - ei;  // tile by tile, so that a range's tiles are a multiple of the XCDs apart
        it.seq = i, it.row0 = row0, it.cnt = cnt, it.held = held, it.total = total, it.splits = ns;
        it.tile = at / (a.nkv * ns), it.hv = at / ns % a.nkv, it.split = at % ns;
        it.qid = eq + it.tile * a.nkv + it.hv;
        it.slot = ns > 1 ? es + at : -1;
        ok = 1;
        break;
      }
      ei += n * ns, eq += n, es += ns > 1 ? n * ns : 0;
    }
  }
  const int src = __ffsll((unsigned long long)mine) - 1;
#define RTQ_KV_GIVE(F) it.F = __builtin_amdgcn_readlane(it.F, src)
  RTQ_KV_GIVE(seq), RTQ_KV_GIVE(row0), RTQ_KV_GIVE(cnt), RTQ_KV_GIVE(held), RTQ_KV_GIVE(total), RTQ_KV_GIVE(tile);
  RTQ_KV_GIVE(hv), RTQ_KV_GIVE(split), RTQ_KV_GIVE(splits), RTQ_KV_GIVE(slot), RTQ_KV_GIVE(qid);
#undef RTQ_KV_GIVE
  ok = __builtin_amdgcn_readlane(ok, src);
  return ok && (unsigned)it.qid < (unsigned)a.qids && it.slot < a.slots;
}

template <int CT>
__device__ __forceinline__ f4 kv_mfma(u4v x, u4v y, f4 c) {
  if constexpr (CT == VT_F16) return mfma_f16(__builtin_bit_cast(half8, x), __builtin_bit_cast(half8, y), c);
  else return mfma_bf16(__builtin_bit_cast(bf8, x), __builtin_bit_cast(bf8, y), c);
}

// eight floats as N planes of 16 bits, each the rounding of what the ones before it leave: 11 (f16) or 8
// (bf16) bits of the value a plane: f32 rows take two (f16) or three, one plane of a 16-bit row is the row itself.
template <int CT, int N>
__device__ __forceinline__ void kv_planes(const float* v, u4v* out) {
  float r[8];
#pragma unroll
  for (int e = 0; e < 8; e++) r[e] = v[e];
#pragma unroll
  for (int n = 0; n < N; n++) {
    out[n] = VRow<CT>::pack(r);
    if (n + 1 < N)
#pragma unroll
      for (int e = 0; e < 8; e++) r[e] -= VRow<CT>::get(out[n], e);
  }
}

#define RTQ_KV_TREE 1024  // most new tokens of a sequence that is a tree

template <int CT, bool QF, int D, bool FULL, int NQ>
__device__ __forceinline__ void kv_attend(const KvAttendArgs& a) {
  constexpr int DC = D / 32, DT = D / 16, TM = 16 * NQ, LDR = D + 4;
  constexpr int NS = QF ? (CT == VT_F16 ? 2 : 3) : 1, NP = QF ? NS : 2;
  constexpr uint32_t EXP = CT == VT_F16 ? 0x7c00u : 0x7f80u;  // infinity and NaN
  // f16 weights are taken times 2^15 (as is their sum): small ones, of which a long context has many, keep their bits
  constexpr float UP = CT == VT_F16 ? 15.0f : 0.0f;
  typedef VRow<QF ? VT_F32 : CT> Q;
  struct Shared {
    float o[4][TM][LDR];
    float ml[4][TM][2];
    float w[4][TM][33];
    uint32_t seen[TM][RTQ_KV_TREE / 32];  // ancestors of each row's token
    uint16_t up[RTQ_KV_TREE];
    int dead[TM];
  };
  __shared__ Shared sh;
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, g = lane >> 4;
  const int group = a.nh / a.nkv, d = FULL ? D : a.d, ps = 1 << a.ps_shift;
  KvItem it;
  if (!kv_plan<TM>(a, blockIdx.x, it)) return;
  const int row_lo = it.tile * TM, rows = min((int)((int64_t)it.cnt * group - row_lo), TM);
  const int k_lo = it.split * it.C;
  // no row of the tile sees a new token after its own
  const int64_t last = (int64_t)it.held + (row_lo + rows - 1) / group + 1;
  const int k_hi = (int)min(min((int64_t)k_lo + it.C, (int64_t)it.total), last);
  const bool tree = a.parents != nullptr;
  if (it.split == 0 && threadIdx.x == 0) {
    int32_t* q = a.desc + 8 + 8 * it.qid;
    q[0] = it.slot, q[1] = it.splits, q[2] = it.row0, q[3] = row_lo, q[4] = rows, q[5] = it.hv;
  }
  // the rows' tokens (index among the sequence's new ones) of this lane's columns
  int tok[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) tok[n] = (row_lo + min(16 * n + li, rows - 1)) / group;
  // f32 rows over an f16 cache are scaled by a power of two that brings the row's largest element to [2^13, 2^14): its
  // planes then neither overflow nor lose bits below f16's range
  constexpr bool SCALED = QF && CT == VT_F16;
  u4v qf[NS][NQ][DC];
  float sc[NQ];
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    const int r = row_lo + min(16 * n + li, rows - 1);
    const int64_t at = (int64_t)(it.row0 + tok[n]) * a.ldq + (int64_t)(it.hv * group + r % group) * d;
    sc[n] = a.scale2;
    float x[QF ? DC : 1][8] = {};
#pragma unroll
    for (int c = 0; c < DC; c++) {
      const bool in = (FULL || 32 * c + 8 * g < d) && 16 * n + li < rows;
      if constexpr (QF) {
        if (in) {
          const u4v r1 = Q::load(a.q, at + 32 * c + 8 * g), r2 = Q::load(a.q, at + 32 * c + 8 * g + 4);
#pragma unroll
          for (int e = 0; e < 4; e++) x[c][e] = Q::get(r1, e), x[c][4 + e] = Q::get(r2, e);
        }
      } else {
        qf[0][n][c] = u4v{0, 0, 0, 0};
        if (in) qf[0][n][c] = Q::load(a.q, at + 32 * c + 8 * g);
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
        const int ex = (int)(__builtin_bit_cast(uint32_t, mx) >> 23);
        up = ex == 255 || ex == 0 ? 0 : min(max(140 - ex, -120), 120);
        sc[n] = ldexpf(a.scale2, -up);
      }
#pragma unroll
      for (int c = 0; c < DC; c++) {
        if constexpr (SCALED)
#pragma unroll
          for (int e = 0; e < 8; e++) x[c][e] = ldexpf(x[c][e], up);
        u4v pl[NS];
        kv_planes<CT, NS>(x[c], pl);
#pragma unroll
        for (int i = 0; i < NS; i++) qf[i][n][c] = pl[i];
      }
    }
  }
  const bool tail = k_hi > it.held;  // some of the item's keys are new tokens
  if (tree && tail) {
    const int words = (min(it.cnt, RTQ_KV_TREE) + 31) / 32;
    for (int i = threadIdx.x; i < TM * (RTQ_KV_TREE / 32); i += 256) (&sh.seen[0][0])[i] = 0;
    for (int i = threadIdx.x; i < min(it.cnt, RTQ_KV_TREE); i += 256) {  // 0: the cache, else the parent + 1; 65535: none
      const int p = a.parents[it.row0 + i];
      sh.up[i] = p < -1 || p >= i ? 65535 : p + 1;
    }
    __syncthreads();
    if (threadIdx.x < TM) {
      const int r = threadIdx.x;
      int node = r < rows ? (row_lo + r) / group : -1, dead = it.cnt > RTQ_KV_TREE;
      while (!dead && node >= 0) {
        sh.seen[r][node >> 5] |= 1u << (node & 31);
        const int p = sh.up[node];
        dead = p == 65535;
        node = p - 1;
      }
      sh.dead[r] = dead;
      if (dead)
        for (int w = 0; w < words; w++) sh.seen[r][w] = 0;
    }
    __syncthreads();
  }

  f4 acc[NQ][DT];
  float m[NQ], l[NQ];
  const int64_t head = (int64_t)d << a.ps_shift, pstride = head * a.nkv;
  const int32_t* table = a.s.table + (int64_t)it.seq * a.s.ldt;
  const auto page_of = [&](int k0) { return a.s.ldt > 0 ? table[min(k0 >> a.ps_shift, a.s.ldt - 1)] : -1; };
  const auto base_of = [&](int k0, int pg) { return ((unsigned)pg < (unsigned)a.n_pages ? pg : 0) * pstride + it.hv * head; };
  u4v kf[2][DC], vf[DT];
  const uint32_t k_at = (uint32_t)((8 * (li >> 2) + (li & 3)) * d + 8 * g) * 2, v_at = (uint32_t)((li << a.ps_shift) + 8 * g) * 2;
  const auto load_k = [&](int k0, int pg) {
    const char* base = reinterpret_cast<const char*>(a.k + base_of(k0, pg) + (int64_t)(k0 & (ps - 1)) * d);
#pragma unroll
    for (int t = 0; t < 2; t++)
#pragma unroll
      for (int c = 0; c < DC; c++) {
        kf[t][c] = u4v{0, 0, 0, 0};
        if (FULL || 32 * c + 8 * g < d) kf[t][c] = *reinterpret_cast<const u4v*>(base + k_at + (4 * t * d + 32 * c) * 2);
      }
  };
  const auto load_v = [&](int k0, int pg) {
    const char* base = reinterpret_cast<const char*>(a.v + base_of(k0, pg) + (k0 & (ps - 1)));
#pragma unroll
    for (int t = 0; t < DT; t++)
      if (FULL || 16 * t < d) vf[t] = *reinterpret_cast<const u4v*>(base + ((int64_t)(32 * t) << a.ps_shift) + v_at);
  };
  // A wave whose sums come out NaN takes its slots once more with care: keys and values that are not finite meet the
  // first plane of queries and weights alone (infinity times a lower plane, which may be 0 or of the other sign, is not
  // infinity times the whole)
  for (bool careful = false;; careful = true) {
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    m[n] = -INFINITY, l[n] = 0.0f;
#pragma unroll
    for (int t = 0; t < DT; t++) acc[n][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  int k0 = k_lo + 32 * wv;
  int pg = 0, pn = 0;
  if (k0 < k_hi) {
    pg = page_of(k0);
    pn = page_of(k0 + 128);
    load_k(k0, pg);
    load_v(k0, pg);
  }
  for (; k0 < k_hi; k0 += 128) {
    f4 s[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; n++)
#pragma unroll
      for (int t = 0; t < 2; t++) {
        s[n][t] = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int c = 0; c < DC; c++)
#pragma unroll
          for (int p = 0; p < NS; p++) s[n][t] = kv_mfma<CT>(kf[t][c], qf[p][n][c], s[n][t]);
        if constexpr (NS > 1)
          if (careful) {
            f4 hi = f4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int c = 0; c < DC; c++) hi = kv_mfma<CT>(kf[t][c], qf[0][n][c], hi);
#pragma unroll
            for (int r = 0; r < 4; r++) s[n][t][r] = s[n][t][r] != s[n][t][r] ? hi[r] : s[n][t][r];
          }
      }
    const int kn = k0 + 128 < k_hi ? k0 + 128 : k0;  // (the last step loads its own slots again)
    const int pgn = k0 + 128 < k_hi ? pn : pg;
    load_k(kn, pgn);
    pn = page_of(kn + 128);
    const bool there = (unsigned)pg < (unsigned)a.n_pages;
    const bool masked = k0 + 32 > it.held || k0 + 32 > k_hi || !there || careful;
    uint32_t bits[NQ];  // which of the lane's eight slots each row sees
    bool any_odd = false;  // values that are not finite, taken out of the product (masked steps)
    if (masked) {
#pragma unroll
      for (int n = 0; n < NQ; n++) {
        bits[n] = 0;
        const int r = 16 * n + li;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const int key = k0 + 8 * g + e, nw = key - it.held;
          bool v = there && key < k_hi && r < rows;
          if (nw >= 0) v = v && (tree ? (nw < RTQ_KV_TREE && (sh.seen[r][(nw & (RTQ_KV_TREE - 1)) >> 5] >> (nw & 31) & 1)) : nw <= tok[n]);
          bits[n] |= v ? 1u << e : 0u;
        }
#pragma unroll
        for (int e = 0; e < 8; e++)
          if (!(bits[n] >> e & 1)) s[n][e >> 2][e & 3] = -INFINITY;
      }
      // slots that no row may see hold anything: zeros in their place, so that nothing x 0 is not NaN; a value of a
      // new token that is not finite may be seen by some of the rows, and is added to those alone
#pragma unroll
      for (int t = 0; t < DT; t++)
        if (FULL || 16 * t < d) {
#pragma unroll
          for (int w = 0; w < 4; w++) {
            const int key = k0 + 8 * g + 2 * w;
            uint32_t x = vf[t][w];
            if (!there || key >= k_hi) x = 0;
            else if (key + 1 >= k_hi) x &= 0xffffu;
            uint32_t o = 0;
            if ((x & EXP) == EXP) o |= 0xffffu;
            if ((x >> 16 & EXP) == EXP) o |= 0xffff0000u;
            vf[t][w] = x & ~o;
            any_odd = any_odd || o;
          }
        }
      any_odd = __any(any_odd);
    }
    u4v pf[NQ][NP];
    float p[NQ][8];
#pragma unroll
    for (int n = 0; n < NQ; n++) {
      float mx = s[n][0][0];
#pragma unroll
      for (int e = 1; e < 8; e++) mx = fmaxf(mx, s[n][e >> 2][e & 3]);
      mx = fmaxf(mx, __shfl_xor(mx, 16));
      mx = fmaxf(mx, __shfl_xor(mx, 32));
      const float mn = fmaxf(m[n], mx * sc[n]), mu = mn == -INFINITY ? 0.0f : mn;
      const float al = __builtin_amdgcn_exp2f(m[n] - mu);
      m[n] = mn;
      float sum = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; e++) {
        p[n][e] = __builtin_amdgcn_exp2f(fmaf(s[n][e >> 2][e & 3], sc[n], UP - mu));
        sum += p[n][e];
      }
      l[n] = l[n] * al + sum;
      if (__any(al != 1.0f)) {
#pragma unroll
        for (int t = 0; t < DT; t++) acc[n][t] *= al;
      }
      kv_planes<CT, NP>(p[n], pf[n]);
    }
#pragma unroll
    for (int t = 0; t < DT; t++)
      if (FULL || 16 * t < d)
#pragma unroll
        for (int n = 0; n < NQ; n++)
#pragma unroll
          for (int q = 0; q < NP; q++) acc[n][t] = kv_mfma<CT>(vf[t], pf[n][q], acc[n][t]);
    if (masked && any_odd) {  // rare: those values are read again, one by one (sums and weights in LDS and the loops
                              // rolled, so that this path costs the others no registers)
#pragma unroll
      for (int n = 0; n < NQ; n++) {
#pragma unroll
        for (int e = 0; e < 8; e++) sh.w[wv][16 * n + li][8 * g + e] = bits[n] >> e & 1 ? p[n][e] : -1.0f;
#pragma unroll
        for (int t = 0; t < DT; t++) *reinterpret_cast<f4*>(&sh.o[wv][16 * n + li][16 * t + 4 * g]) = acc[n][t];
      }
      __builtin_amdgcn_wave_barrier();
      const uint16_t* base = a.v + base_of(k0, pg) + (k0 & (ps - 1));
#pragma unroll 1
      for (int e = 0; e < 32 && k0 + e < k_hi; e++)
#pragma unroll 1
        for (int c = 4 * g; c < d; c += (c & 3) < 3 ? 1 : 13) {
          const uint32_t x = base[((int64_t)c << a.ps_shift) + e];
          if ((x & EXP) == EXP)
#pragma unroll 1
            for (int r = li; r < TM; r += 16)
              if (sh.w[wv][r][e] != -1.0f) sh.o[wv][r][c] += sh.w[wv][r][e] * VRow<CT>::get(u4v{x, x, x, x}, 0);
        }
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int n = 0; n < NQ; n++)
#pragma unroll
        for (int t = 0; t < DT; t++) acc[n][t] = *reinterpret_cast<const f4*>(&sh.o[wv][16 * n + li][16 * t + 4 * g]);
    }
    load_v(kn, pgn);
    pg = pgn;
  }
  bool nan = false;
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    bool x = l[n] != l[n];
#pragma unroll
    for (int t = 0; t < DT; t++)
#pragma unroll
      for (int r = 0; r < 4; r++) x = x || acc[n][t][r] != acc[n][t][r];
    nan = nan || __any(x);
  }
  if (careful || !nan) break;
  }
  // the four waves' parts
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    l[n] += __shfl_xor(l[n], 16);
    l[n] += __shfl_xor(l[n], 32);
    if (g == 0) sh.ml[wv][16 * n + li][0] = m[n], sh.ml[wv][16 * n + li][1] = l[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < NQ; n++) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; w++) mx = fmaxf(mx, sh.ml[w][16 * n + li][0]);
    const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[n] - mx);
#pragma unroll
    for (int t = 0; t < DT; t++)
      if (FULL || 16 * t < d) *reinterpret_cast<f4*>(&sh.o[wv][16 * n + li][16 * t + 4 * g]) = acc[n][t] * f;
  }
  __syncthreads();
  const int vecs = d / 4;
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
    const bool dead = tree && tail && sh.dead[r];
    if (it.slot >= 0) {
      *reinterpret_cast<f4*>(a.part + ((int64_t)it.slot * TM + r) * D + c) = o;
      if (c == 0) a.ml[((int64_t)it.slot * TM + r) * 2] = mx, a.ml[((int64_t)it.slot * TM + r) * 2 + 1] = dead ? -1.0f : ls;
    } else {
      const int tk = (row_lo + r) / group;
      const int64_t at = (int64_t)(it.row0 + tk) * a.ldo + (int64_t)(it.hv * group + (row_lo + r) % group) * d + c;
      const float inv = 1.0f / ls;
#pragma unroll
      for (int e = 0; e < 4; e++) Q::put(a.o, at + e, dead || ls == 0.0f ? 0.0f : o[e] * inv);
    }
  }
}

// joins the parts of a tile's row: workgroup (tile, row)
template <int QT, int D>
__device__ __forceinline__ void kv_merge(const KvAttendArgs& a, int TM) {
  constexpr int V = D / 4, G = 256 / V;
  __shared__ float red[256];
  __shared__ f4 ro[256];
  if ((int)blockIdx.x >= a.desc[0]) return;
  const int32_t* q = a.desc + 8 + 8 * blockIdx.x;
  const int slot = q[0], ns = q[1], r = blockIdx.y;
  if (slot < 0 || r >= q[4]) return;
  const float* ml = a.ml + ((int64_t)slot * TM + r) * 2;
  const int tid = threadIdx.x;
  float mx = -INFINITY;
  int dead = 0;
  for (int i = tid; i < ns; i += 256) mx = fmaxf(mx, ml[(int64_t)i * TM * 2]), dead |= ml[(int64_t)i * TM * 2 + 1] == -1.0f;
  red[tid] = mx;
  dead = __syncthreads_or(dead);
  for (int s = 128; s > 0; s >>= 1) {
    if (tid < s) red[tid] = fmaxf(red[tid], red[tid + s]);
    __syncthreads();
  }
  mx = red[0];
  __syncthreads();
  const int c = tid % V * 4, gr = tid / V;
  float ls = 0.0f;
  f4 o = f4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = gr; i < ns; i += G) {
    const float f = mx == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(ml[(int64_t)i * TM * 2] - mx);
    ls += f * ml[(int64_t)i * TM * 2 + 1];
    if (c < a.d) o += f * *reinterpret_cast<const f4*>(a.part + ((int64_t)(slot + i) * TM + r) * D + c);
  }
  ro[tid] = o, red[tid] = ls;
  __syncthreads();
  if (gr == 0 && c < a.d) {
    for (int i = 1; i < G; i++) o += ro[i * V + tid], ls += red[i * V + tid];
    const int group = a.nh / a.nkv, row = q[3] + r;
    const int64_t at = (int64_t)(q[2] + row / group) * a.ldo + (int64_t)(q[5] * group + row % group) * a.d + c;
    const float inv = 1.0f / ls;
#pragma unroll
    for (int e = 0; e < 4; e++) VRow<QT>::put(a.o, at + e, dead || ls == 0.0f ? 0.0f : o[e] * inv);
  }
}

#define RTQ_KV_ATTEND(SUF, CT, QF, D, FULL, NQ) \
  extern "C" __global__ __launch_bounds__(256, D > 128 ? 1 : 2) void rtq_kv_attend##SUF(KvAttendArgs a) { kv_attend<CT, QF, D, FULL, NQ>(a); }
#define RTQ_KV_ATTENDS(SUF, CT, QF)             \
  RTQ_KV_ATTEND(16_64_##SUF, CT, QF, 64, true, 1)    \
  RTQ_KV_ATTEND(16_128_##SUF, CT, QF, 128, true, 1)  \
  RTQ_KV_ATTEND(16_128p_##SUF, CT, QF, 128, false, 1) \
  RTQ_KV_ATTEND(16_256p_##SUF, CT, QF, 256, false, 1) \
  RTQ_KV_ATTEND(32_64_##SUF, CT, QF, 64, true, 2)    \
  RTQ_KV_ATTEND(32_128_##SUF, CT, QF, 128, true, 2)  \
  RTQ_KV_ATTEND(32_128p_##SUF, CT, QF, 128, false, 2)
RTQ_KV_ATTENDS(f32_f16, VT_F16, true)
RTQ_KV_ATTENDS(f32_bf16, VT_BF16, true)
RTQ_KV_ATTENDS(f16, VT_F16, false)
RTQ_KV_ATTENDS(bf16, VT_BF16, false)

#define RTQ_KV_MERGE(NAME, QT, D) \
  extern "C" __global__ __launch_bounds__(256) void NAME(KvAttendArgs a) { kv_merge<QT, D>(a, a.tm); }
RTQ_KV_MERGE(rtq_kv_merge64_f32, VT_F32, 64)
RTQ_KV_MERGE(rtq_kv_merge128_f32, VT_F32, 128)
RTQ_KV_MERGE(rtq_kv_merge256_f32, VT_F32, 256)
RTQ_KV_MERGE(rtq_kv_merge64_f16, VT_F16, 64)
RTQ_KV_MERGE(rtq_kv_merge128_f16, VT_F16, 128)
RTQ_KV_MERGE(rtq_kv_merge256_f16, VT_F16, 256)
RTQ_KV_MERGE(rtq_kv_merge64_bf16, VT_BF16, 64)
RTQ_KV_MERGE(rtq_kv_merge128_bf16, VT_BF16, 128)
RTQ_KV_MERGE(rtq_kv_merge256_bf16, VT_BF16, 256)
