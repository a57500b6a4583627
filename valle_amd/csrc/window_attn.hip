// Prompt attention with a sliding window, first tokens that stay visible (sinks), a text prefix that every row sees, and grouped heads.
//
//   out_i = sum_j p_ij v_j,  p_i = softmax over the visible j of scale q_i . k_j
//   row i of a sequence sees key j  iff  j < text  or  (j <= i and (window <= 0 or i - j < window or j < sinks))
//
// One workgroup takes a run of query rows of one (sequence, head) and walks the key tiles that any of them sees: the tiles of the head
// (text, sinks), then those of the window; the tiles between are never loaded, so the work of a row is its window's, not its position's.
// Both products are computed transposed (S^T = K Q^T, O^T = V^T P^T): the weights leave the first in the operand layout of the second.
// The scores' running maximum, the row sums and both accumulators are fp32.  A lane holds the query column c = lane % 16 and of every 16-key
// score tile the keys 4 g + r, g = lane / 16.
//
// A key that a row does not see must not reach it, whatever it holds -- but a tile's product runs over all keys of the tile, and 0 * NaN is NaN.
// Rows whose result is not finite (a rarity: such a value, or sums past the largest number) are therefore computed once more, key by key over
// the visible ones alone (exact_row).
#include "common.h"
#include "kernels.h"

namespace vle {

namespace {

typedef __bf16 wa_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 wa_bf16x4 __attribute__((ext_vector_type(4)));
typedef short wa_s16x4 __attribute__((ext_vector_type(4)));
typedef short wa_s16x8 __attribute__((ext_vector_type(8)));
typedef float wa_f32x4 __attribute__((ext_vector_type(4)));
typedef float wa_f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned wa_u32x4 __attribute__((ext_vector_type(4)));

constexpr float WA_DEFER = 8.f;  // exp2-domain growth of a row's maximum below which its reference stays (weights up to 2^8)

// Where a workgroup works: sequence, head, first query row.  Work items are numbered group of heads by group (what one XCD holds of them, where 8 divides
// their number), sequence by sequence, run of rows by run (late ones, which see most without a window, first), head by head: neighbours read the same keys,
// and work shrinks from item to item (head by head instead: one sequence of 4000 rows without a window, 16 heads of 64, bf16 51 -> 66 us, fp32 303 -> 430).
// `seq` = -1: no sequence is left for this item and `rest` counts the runs of its head past the last one.
struct Place {
  int h, seq, off, len, text, q0, rest;
};
template <int QB>
__device__ inline Place place_of(const WindowAttnArgs& a) {
  const int lane = threadIdx.x & 63;
  const int per_head = gridDim.x / a.H;
  // workgroup L runs on XCD L % 8, each with its own L2: every XCD gets a contiguous run of the items
  const int nb = gridDim.x, q = nb / 8, rem = nb % 8, xcd = blockIdx.x % 8;
  int idx = blockIdx.x / 8;
  // ... and deals them out to its 32 CUs in turn: every other round backwards, so that the CUs with the longest item of one get the shortest of the next
  if ((idx & 32) && (idx | 31) < q + (xcd < rem)) idx ^= 31;
  const int item = (xcd < rem ? xcd * (q + 1) : rem * (q + 1) + (xcd - rem) * q) + idx;
  const int hg = a.H % 8 == 0 ? a.H / 8 : 1, group = item / (per_head * hg);
  Place p;
  int at = item - group * per_head * hg;
  auto rows_of = [&](int b, int& off) {  // clamped to the rows there are, whatever the offsets say
    off = (int)min((int64_t)max(a.seq_off[b], 0), a.rows);
    return (int)min((int64_t)max(a.seq_off[b + 1], off), a.rows) - off;
  };
  int lo = 0, hi = a.B;
  const int per = (a.B + 63) >> 6;
  if (per > 1) {  // many sequences: which lane's share of them holds the item
    int sum = 0, off;
    for (int b = lane * per; b < min((lane + 1) * per, a.B); ++b) sum += (rows_of(b, off) + QB - 1) / QB * hg;
    const int inc = wave_scan_i(sum);
    const unsigned long long past = __ballot(at < inc);
    if (past) {
      const int l = __builtin_ctzll(past);
      at -= __builtin_amdgcn_readlane(inc - sum, l);
      lo = l * per;
      hi = min(lo + per, a.B);
    } else {
      at -= __builtin_amdgcn_readlane(inc, 63);
      hi = 0;
    }
  }
  for (int b0 = lo; b0 < hi; b0 += 64) {
    const int b = b0 + lane;
    int off = 0, len = 0, text = 0;
    if (b < hi) {
      if (a.text_len) text = a.text_len[b];  // (with the offsets, not a round trip to memory later)
      len = rows_of(b, off);
    }
    const int inc = wave_scan_i((len + QB - 1) / QB * hg);
    const unsigned long long past = __ballot(at < inc);
    if (past) {
      const int l = __builtin_ctzll(past);
      p.off = __builtin_amdgcn_readlane(off, l);
      p.len = __builtin_amdgcn_readlane(len, l);
      p.text = min(max(__builtin_amdgcn_readlane(text, l), 0), p.len);
      const int left = __builtin_amdgcn_readlane(inc, l) - 1 - at, run = left / hg;
      p.h = group * hg + (left >= 0 ? left - run * hg : 0);
      p.q0 = run * QB;
      p.rest = 0x7fffffff;
      p.seq = (left >= 0) & (run < (p.len + QB - 1) / QB) ? b0 + l : -1;  // -1: offsets that go back and forth until the count of their runs overflows
      return p;
    }
    at -= __builtin_amdgcn_readlane(inc, 63);
  }
  p.seq = -1;
  p.off = p.len = p.text = p.q0 = 0;
  p.rest = at < 0 ? 0x7fffffff : at / hg;  // (< 0: the same)
  p.h = group * hg + (at < 0 ? 0 : at % hg);
  return p;
}

// The key tiles a run of rows i0 .. i1 sees (TK keys each): 0 .. th - 1 the head, then mf + (t - th).
struct Tiles {
  int th, mf, tt;
};
template <int TK>
__device__ inline Tiles tiles_of(int i0, int i1, int text, int window, int sinks) {
  Tiles r;
  const int hd = window > 0 ? max(text, min(sinks, i1 + 1)) : text;
  const int lo = window > 0 ? max(0, i0 - window + 1) : 0;
  r.th = (hd + TK - 1) / TK;
  r.mf = max(r.th, lo / TK);
  r.tt = r.th + max(0, (i1 + TK) / TK - r.mf);
  return r;
}

// What one row sees: keys j < hd, and lo <= j <= i.
struct Sight {
  int hd, lo, i;
  // (& and | on purpose: a select per key, no branches)
  __device__ bool sees(int j) const { return (j < hd) | ((j >= lo) & (j <= i)); }
};
__device__ inline Sight sight_of(int i, int text, int window, int sinks) {
  Sight s;
  s.hd = window > 0 ? max(text, min(sinks, i + 1)) : text;
  s.lo = window > 0 ? max(0, i - window + 1) : 0;
  s.i = i;
  return s;
}

// What the rows i0 .. i1 of a wave see of the keys j0 .. j0 + n - 1 (both ends of a row's sight grow with the row): scalar arithmetic.
struct Sights {
  Sight first, last;
  __device__ bool all(int j0, int n) const { return j0 + n <= first.hd || (j0 >= last.lo && j0 + n - 1 <= first.i); }
  __device__ bool none(int j0, int n) const { return j0 >= last.hd && (j0 > last.i || j0 + n - 1 < first.lo); }
};
__device__ inline Sights sights_of(int i0, int i1, int text, int window, int sinks) {
  return Sights{sight_of(i0, text, window, sinks), sight_of(i1, text, window, sinks)};
}

// One row over its visible keys alone, by one wave: 64 keys at a time, a lane the score of one, then two elements of the output as the average so far.
template <typename T>
__device__ inline void exact_row(const WindowAttnArgs& a, int h, int off, int i, int text, int len) {
#pragma clang fp contract(off)  // score - m must be the difference of two rounded scores: 0 for the largest, whatever its size
  constexpr int VE = Elem<T>::VEC;
  const int lane = threadIdx.x & 63, hk = h / (a.H / a.Hkv);
  const Sight see = sight_of(i, text, a.window, a.sinks);
  const T* q = (const T*)a.q + (int64_t)(off + i) * a.q_row + (int64_t)h * a.q_head;
  const T* k = (const T*)a.k + (int64_t)off * a.k_row + (int64_t)hk * a.k_head;
  const T* v = (const T*)a.v + (int64_t)off * a.v_row + (int64_t)hk * a.v_head;
  const bool in0 = lane < a.dh, in1 = lane + 64 < a.dh;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  bool bad = false;  // a score that is not a number, or none above -inf
  const int end = min(len, max(see.hd, i + 1));
  for (int j0 = 0; j0 < end && !bad; j0 += 64) {
    const int j = j0 + lane;
    const bool vis = (j < end) & see.sees(j);
    if (!__any(vis)) continue;
    float s = -INFINITY;
    if (vis) {
      float sum = 0.f;
      for (int e = 0; e < a.dh; e += VE) {
        float x[VE], y[VE];
        load_vec16(q + e, x);
        load_vec16(k + (int64_t)j * a.k_row + e, y);
#pragma unroll
        for (int u = 0; u < VE; ++u) sum = fmaf(x[u], y[u], sum);
      }
      s = sum * a.sl2;
    }
    bad = __any(s != s);
    const float mn = fmaxf(m, wave_max(s));
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float p = __builtin_amdgcn_exp2f(s - ref);
    const float was = l * __builtin_amdgcn_exp2f(m - ref), now = was + wave_sum(p);
    m = mn;
    l = now;
    if (now == 0.f) continue;  // nothing but -inf so far
    o0 *= was / now;
    o1 *= was / now;
    unsigned long long todo = __ballot(vis);
    while (todo) {
      const int t = __builtin_ctzll(todo);
      todo &= todo - 1;
      const float w = readlane_f32(p, t) / now;
      const T* row = v + (int64_t)(j0 + t) * a.v_row;
      if (in0) o0 = fmaf(w, Elem<T>::to_f32(row[lane]), o0);
      if (in1) o1 = fmaf(w, Elem<T>::to_f32(row[lane + 64]), o1);
    }
  }
  if (bad | (l == 0.f)) o0 = o1 = __builtin_nanf("");
  T* op = (T*)a.out + ((int64_t)(off + i) * a.H + h) * a.dh;
  if (in0) store_elem<T>(op + lane, o0);
  if (in1) store_elem<T>(op + lane + 64, o1);
}

// Rows that no sequence holds, `rest`-th run of them.
template <typename T, int QB>
__device__ inline void zero_rows(const WindowAttnArgs& a, int h, int rest) {
  const int first = a.B > 0 ? (int)min((int64_t)max(a.seq_off[0], 0), a.rows) : 0;
  const int64_t end = a.B > 0 ? min((int64_t)max(a.seq_off[a.B], first), a.rows) : 0;
  const int vpr = a.dh * (int)sizeof(T) / 16;
  for (int idx = threadIdx.x; idx < QB * vpr; idx += blockDim.x) {
    int64_t r = (int64_t)rest * QB + idx / vpr;
    if (r >= first) r += end - first;
    if (r >= a.rows) return;
    reinterpret_cast<wa_u32x4*>((T*)a.out + (r * a.H + h) * a.dh)[idx % vpr] = wa_u32x4{0u, 0u, 0u, 0u};
  }
}

// 16-byte slot swizzle of the LDS rows (NV slots each), applied to the address a DMA lane fetches from and to every read: rows land on
// different banks.  The key stays inside an aligned group of slots that divides NV.
template <int NV>
__device__ constexpr int wa_key(int row) {
  return NV % 16 == 0 ? (row & 15) : NV % 8 == 0 ? (row & 7) : ((row >> 1) & 3);
}

// The same for the V rows of the bf16 kernel: its transposing reads take 32 bytes (two slots) of 8 rows at a time, so these rows must differ in the pair of
// slots.  (With the key above a third of the LDS cycles were bank conflicts, now none are; the kernel's time is the same.)
template <int NV>
__device__ constexpr int wa_key_pairs(int row) {
  return NV % 16 == 0 ? (row & 7) << 1 : NV % 8 == 0 ? (row >> 1 & 3) << 1 : (row >> 2 & 1) << 1;
}

// 16 bytes per lane from base + off to LDS address dst + 16 * lane (base and dst wave-uniform).  Not the builtin: the compiler takes any later LDS
// read it cannot tell apart -- the transposing ones -- for a reader of what is in flight and waits for all of it, so that no tile is ever fetched ahead.
// The waits for these loads are the kernels' own, ahead of the barrier that hands a tile over.
__device__ inline void wa_dma(const void* base, unsigned off, unsigned dst) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(dst), "v"(off), "s"(base) : "memory", "m0");
}

// Stages tiles of TK rows (NV 16-byte vectors each) of K or V into LDS, by the whole workgroup.  Rows past the sequence repeat its last one and
// vectors past the head its first one: what they hold is never visible.  A lane's place in a tile is worked out once; a tile inside the sequence
// then costs scalar arithmetic alone.  (Byte offsets inside a tile are 32-bit: row strides are below 2^24 elements, checked at the entry.)
template <typename T, int TK, int NV, bool PAIRS = false>  // PAIRS: wa_key_pairs
struct Stager {
  static constexpr int VE = 16 / (int)sizeof(T), N = TK * NV / 256;
  const T* base;
  unsigned stride;  // bytes
  int len, wu;
  unsigned off[N];
  __device__ Stager(const T* b, int64_t row_stride, int l, int dh, int w_uniform) : base(b), stride((unsigned)row_stride * sizeof(T)), len(l), wu(w_uniform) {
#pragma unroll
    for (int i = 0; i < N; ++i) off[i] = row(i) * stride + vec(i, dh) * 16;
  }
  __device__ int row(int i) const { return ((i * 4 + wu) * 64 + (int)(threadIdx.x & 63)) / NV; }
  __device__ int vec(int i, int dh) const {
    const int v = (((i * 4 + wu) * 64 + (int)(threadIdx.x & 63)) % NV) ^ (PAIRS ? wa_key_pairs<NV>(row(i)) : wa_key<NV>(row(i)));
    return v * VE < dh ? v : 0;
  }
  __device__ void operator()(int kt0, int dh, const unsigned char* dst) const {
    const unsigned to = (unsigned)__builtin_amdgcn_readfirstlane((int)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)dst) + wu * 1024;
    const char* src = (const char*)base + (int64_t)kt0 * stride;
    if (kt0 + TK <= len) {
#pragma unroll
      for (int i = 0; i < N; ++i) wa_dma(src, off[i], to + i * 4096);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) wa_dma(src, min(row(i), len - 1 - kt0) * stride + vec(i, dh) * 16, to + i * 4096);
    }
  }
};

}  // namespace

// ---- bf16 --------------------------------------------------------------------------------------------------------------------------
// 4 waves, QW query fragments of 16 rows each; 64-key tiles of K and V go global -> LDS by DMA into one of two buffers while the other is
// multiplied (a third buffer changed nothing); V^T operands come from the row-major tile through the transposing LDS read.  The row sums ride on the
// matrix pipe (an all-ones row block of V^T), so numerator and denominator carry the same rounding of the weights to bf16: 2^-8 of each weight at most, which
// averages out over the keys.  It moves an output by 0.0003 (long rows) to 0.0006 of its size (a few keys), against the 0.0017 of the output's own rounding to
// bf16: in all 0.0017 - 0.0018 from the exact result, where weights of 32 bits give 0.0016 - 0.0017.  Weights of 16 bits, as the sum of two bf16 numbers, would take
// the second product twice, which is half of what the matrix pipe does here.
//
// Measured: one sequence of 12289 rows, 16 heads on 4 key-value heads of 128, window 2048: 211 - 216 us = 875 - 898 TFLOP/s of visible pairs, 73 % of what a large
// library product reaches here (1206).  The matrix pipe is busy 41 % of the cycles, the vector pipe 39 % (exponentials, masks, conversions), LDS 20 %; two
// waves a SIMD overlap them in part only.  32 sequences of 700 - 1100 rows, 16 heads of 64, window 256: 91 - 94 us (238 MB; a copy of it takes 49): vector pipe
// 51 %, matrix pipe 21 %, the rest waits -- a wave of 16 rows computes 460 keys a row for 340 visible ones, head size 64 has half the product per
// exponential, and walks of 8 tiles do not hide their start.  Two short sequences: 5.0 us, less than a launch costs the host.
template <int DHT, int QW>
__global__ __launch_bounds__(256) void window_attn_bf16_kernel(WindowAttnArgs a) {
  constexpr int QB = 64 * QW, TK = 64, NV = DHT / 8, ROW = DHT * 2, KS = DHT / 32, EB = DHT / 16;
  constexpr int HALF = TK * ROW, BUF = 2 * HALF;
  __shared__ __attribute__((aligned(16))) unsigned char smem[2 * BUF];
  const Place pl = place_of<QB>(a);
  if (pl.seq < 0) {
    if (a.zero_rest) zero_rows<bf16_t, QB>(a, pl.h, pl.rest);
    return;
  }
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
  const int wu = __builtin_amdgcn_readfirstlane(w);
  const int len = pl.len, q0 = pl.q0, dh = a.dh, hk = pl.h / (a.H / a.Hkv);
  const int text = pl.text;
  const Tiles ti = tiles_of<TK>(q0, min(q0 + QB, len) - 1, text, a.window, a.sinks);
  const bf16_t* kb = (const bf16_t*)a.k + (int64_t)pl.off * a.k_row + (int64_t)hk * a.k_head;
  const bf16_t* vb = (const bf16_t*)a.v + (int64_t)pl.off * a.v_row + (int64_t)hk * a.v_head;

  Sight see[QW];
  Sights group[QW];  // of the fragment's 16 rows
  bool valid[QW];
  wa_bf16x8 qf[QW][KS];
#pragma unroll
  for (int f = 0; f < QW; ++f) {
    const int i = q0 + (w * QW + f) * 16 + c;
    valid[f] = i < len;
    see[f] = sight_of(min(i, len - 1), text, a.window, a.sinks);
    const int i0 = q0 + (wu * QW + f) * 16;
    group[f] = sights_of(min(i0, len - 1), min(i0 + 15, len - 1), text, a.window, a.sinks);
    const bf16_t* qp = (const bf16_t*)a.q + (int64_t)(pl.off + min(i, len - 1)) * a.q_row + (int64_t)pl.h * a.q_head;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      wa_u32x4 x = {0u, 0u, 0u, 0u};
      if (ks * 32 + g * 8 < dh) x = *reinterpret_cast<const wa_u32x4*>(qp + ks * 32 + g * 8);
      qf[f][ks] = __builtin_bit_cast(wa_bf16x8, x);
    }
  }

  const float sl2 = a.sl2;
  float M[QW];  // reference of the row's scores, shared by its 4 lanes: their maximum when it was last moved; -inf: no key yet
  wa_f32x4 ol[QW], o[QW][EB];
#pragma unroll
  for (int f = 0; f < QW; ++f) {
    M[f] = -INFINITY;
    ol[f] = wa_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int eb = 0; eb < EB; ++eb) o[f][eb] = wa_f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const wa_bf16x8 ones = __builtin_bit_cast(wa_bf16x8, wa_s16x8{0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80, 0x3F80});
  auto key0 = [&](int t) { return (t < ti.th ? t : ti.mf + (t - ti.th)) * TK; };

  const Stager<bf16_t, TK, NV> stage_k(kb, a.k_row, len, dh, wu);
  const Stager<bf16_t, TK, NV, true> stage_v(vb, a.v_row, len, dh, wu);
  stage_k(key0(0), dh, smem);
  stage_v(key0(0), dh, smem + HALF);
  // the queries are waited for here, once: a wait at their first use would stand inside the loop and take the tiles in flight with it
#pragma unroll
  for (int f = 0; f < QW; ++f)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qf[f][ks]));
  for (int t = 0; t < ti.tt; ++t) {
    const int kt0 = key0(t);
    const unsigned char* Ks = smem + (t & 1) * BUF;
    const unsigned char* Vs = Ks + HALF;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's pieces of tile t have landed
    __syncthreads();                                  // everyone's have; everyone is done with tile t - 1
    if (t + 1 < ti.tt) {
      unsigned char* nb = smem + ((t + 1) & 1) * BUF;
      stage_k(key0(t + 1), dh, nb);
      stage_v(key0(t + 1), dh, nb + HALF);
    }
    bool none = true, unmasked = true;
#pragma unroll
    for (int f = 0; f < QW; ++f) {
      none = none && group[f].none(kt0, TK);
      unmasked = unmasked && group[f].all(kt0, TK);
    }
    if (none) continue;
    // (a masked tile's key that is not finite makes the row NaN: computed again at the end)

    // ---- S^T = K Q^T: the accumulators start from the mask (0 or -inf) ----
    wa_f32x4 s[QW][4];
    auto scores = [&]() {
      wa_bf16x8 ka[2][KS];  // the next 16 keys' fragments are read while these are multiplied
      auto read_k = [&](wa_bf16x8 (&d)[KS], int kb4) {
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
          d[ks] = *reinterpret_cast<const wa_bf16x8*>(Ks + (kb4 * 16 + c) * ROW + (((ks * 4 + g) ^ wa_key<NV>(c)) << 4));
      };
      read_k(ka[0], 0);
#pragma unroll
      for (int kb4 = 0; kb4 < 4; ++kb4) {
        if (kb4 < 3) read_k(ka[(kb4 + 1) & 1], kb4 + 1);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks)
#pragma unroll
          for (int f = 0; f < QW; ++f) s[f][kb4] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka[kb4 & 1][ks], qf[f][ks], s[f][kb4], 0, 0, 0);
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    if (unmasked) {
#pragma unroll
      for (int f = 0; f < QW; ++f)
#pragma unroll
        for (int kb4 = 0; kb4 < 4; ++kb4) s[f][kb4] = wa_f32x4{0.f, 0.f, 0.f, 0.f};
      scores();
    } else {
#pragma unroll
      for (int f = 0; f < QW; ++f) {
        // key number 16 kb4 + r of this lane is visible from lo to hi, or, in a tile of the head, below hd: compares with constants, as few as the tile needs
        // (a branch for every 16 keys, most of which are visible or hidden as a whole, is slower: 73 -> 86 us for 32 sequences of 900 rows, heads of 64)
        const int hi = see[f].i - kt0 - g * 4, lo = see[f].lo - kt0 - g * 4, hd = see[f].hd - kt0 - g * 4;
        auto mask = [&](auto hidden) {
#pragma unroll
          for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[f][kb4][r] = hidden(kb4 * 16 + r) ? -INFINITY : 0.f;
        };
        if (t < ti.th) mask([=](int k) { return (k >= hd) & ((k < lo) | (k > hi)); });
        else if (group[f].last.lo <= kt0) mask([=](int k) { return k > hi; });
        else if (group[f].first.i >= kt0 + TK - 1) mask([=](int k) { return k < lo; });
        else mask([=](int k) { return (k < lo) | (k > hi); });
      }
      scores();
    }
    // ---- online softmax: scores relative to the row's reference M, both in units of the exp2 argument ----
    wa_bf16x8 pf[QW][2];
#pragma unroll
    for (int f = 0; f < QW; ++f) {
      // s sl2 - M in one fma, of every tile against M as it is stored: the same rounding of M for the whole row, which cancels, so that equal scores get equal
      // weights whatever their size -- up to scores of 2^31, where it passes the exponent's range and the row is computed again
      wa_f32x4 x[4];
      auto relative = [&](float ref) {
#pragma unroll
        for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
          for (int r = 0; r < 4; ++r) x[kb4][r] = fmaf(s[f][kb4][r], sl2, ref == -INFINITY ? 0.f : -ref);
      };
      relative(M[f]);
      float mt = fmaxf(fmaxf(x[0][0], x[0][1]), fmaxf(x[0][2], x[0][3]));
#pragma unroll
      for (int kb4 = 1; kb4 < 4; ++kb4) mt = fmaxf(mt, fmaxf(fmaxf(x[kb4][0], x[kb4][1]), fmaxf(x[kb4][2], x[kb4][3])));
      // the reference stays while no score exceeds it by more than WA_DEFER: the result does not depend on it, O and the sum carry the same factor
      if (!__all((mt <= WA_DEFER) & (M[f] != -INFINITY))) {
        mt = rows4_max(mt);
        const bool begun = M[f] != -INFINITY;
        const float was = M[f];
        M[f] = begun ? was + fmaxf(mt, 0.f) : mt;
        const float alpha = begun ? __builtin_amdgcn_exp2f(was - M[f]) : 1.f;  // from the two as stored; a rounding of the difference is 2^-24 of it, of a weight 2^-difference
        relative(M[f]);  // not x less the step: x is rounded at the old reference's distance
        ol[f] *= alpha;
#pragma unroll
        for (int eb = 0; eb < EB; ++eb) o[f][eb] *= alpha;
      }
#pragma unroll
      for (int kb4 = 0; kb4 < 4; ++kb4)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[kb4][r] = __builtin_amdgcn_exp2f(x[kb4][r]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int tt = 0; tt < 8; ++tt) pf[f][j][tt] = (__bf16)x[2 * j + (tt >> 2)][tt & 3];
    }
    // ---- O^T += V^T P^T ----
    // the transposing read hands lane c the elements V[k0 .. k0 + 3][16 eb + c] of the rows whose addresses lanes c / 4 supply
    wa_s16x4 vr[2][2][2];  // [buffer][j][half]: the next 16 columns' fragments are read while these are multiplied
    auto read_v = [&](wa_s16x4 (&d)[2][2], int eb) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int key = j * 32 + g * 4 + (c >> 2);
        const unsigned char* va = Vs + key * ROW + (((eb * 2 + ((c & 3) >> 1)) ^ wa_key_pairs<NV>(key)) << 4) + ((c & 1) << 3);
        d[j][0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) wa_s16x4*)(va));
        d[j][1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) wa_s16x4*)(va + 16 * ROW));  // the swizzle has a period of 16 rows
      }
    };
    read_v(vr[0], 0);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int f = 0; f < QW; ++f) ol[f] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, pf[f][j], ol[f], 0, 0, 0);
#pragma unroll
    for (int eb = 0; eb < EB; ++eb) {
      if (eb + 1 < EB) read_v(vr[(eb + 1) & 1], eb + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const wa_s16x4 lo = vr[eb & 1][j][0], hi = vr[eb & 1][j][1];
        const wa_bf16x8 vf = __builtin_bit_cast(wa_bf16x8, wa_s16x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
#pragma unroll
        for (int f = 0; f < QW; ++f) o[f][eb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[f][j], o[f][eb], 0, 0, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }

#pragma unroll
  for (int f = 0; f < QW; ++f) {
    const float inv = 1.0f / ol[f][0];  // every row of the all-ones block holds the whole sum
    const int i = q0 + (w * QW + f) * 16 + c;
    bool odd = false;
    bf16_t* op = (bf16_t*)a.out + ((int64_t)(pl.off + i) * a.H + pl.h) * dh + g * 4;
#pragma unroll
    for (int eb = 0; eb < EB; ++eb) {
      if (eb * 16 + g * 4 >= dh) continue;
      wa_bf16x4 r4;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float x = o[f][eb][r] * inv;
        odd |= !(fabsf(x) < INFINITY);
        r4[r] = (__bf16)x;
      }
      if (valid[f]) *reinterpret_cast<wa_bf16x4*>(op + eb * 16) = r4;
    }
    unsigned long long again = __ballot(odd && valid[f]);
    if (again) {
      again = (again | (again >> 16) | (again >> 32) | (again >> 48)) & 0xffffull;
      while (again) {
        const int t = __builtin_ctzll(again);
        again &= again - 1;
        exact_row<bf16_t>(a, pl.h, pl.off, q0 + (wu * QW + f) * 16 + t, text, len);
      }
    }
  }
}

// ---- fp32 --------------------------------------------------------------------------------------------------------------------------
// The same walk on v_mfma_f32_16x16x4_f32 (exact fp32 products, 1/16 of the bf16 rate): 64 query rows, 32-key tiles.  A 16-byte fragment of
// K feeds four products (contraction slot g of product u is dim 16 t + 4 g + u); V^T needs no transpose: product j of key r takes V[4 g + r][dim(c, j)],
// with dim(c, j) the j-th of the up to 8 elements that lane c reads of a row.
// NG = 2: two groups of 4 waves share the rows and take every other tile each; their halves are joined at the end.
// Measured: two sequences of 700 - 1025 rows, 16 heads of 96, window 300: 57 us = 63 TFLOP/s of visible pairs (a large library product: 154); 1.75 workgroups
// a CU, so that most wait for those with two, and tiles on the window's edges bound it.  One sequence of 4000 rows, 16 heads of 64, window 1000: 162 us = 88 TFLOP/s.
template <int DHT, int NG>
__global__ __launch_bounds__(256 * NG) void window_attn_f32_kernel(WindowAttnArgs a) {
  constexpr int QB = 64, TK = 32, NV = DHT / 4, ROW = DHT * 4, KT = DHT / 16, DPL = DHT / 16;
  constexpr int HALF = TK * ROW, BUF = 2 * HALF;
  constexpr int A4 = DPL >= 4 ? 4 : 2;           // elements of a lane's first chunk of a V row, and of its second
  constexpr int B4 = DPL - A4;                   // (DHT 32: 2, 64: 4, 96: 4 + 2, 128: 4 + 4)
  // two groups: more than half of the LDS, so that a CU takes one workgroup at a time and the next goes to the first that is free (one sequence of 1300 rows,
  // 16 heads of 64: 70 -> 62 us)
  constexpr int LDS = NG == 2 && 2 * NG * BUF < (82 << 10) ? 82 << 10 : 2 * NG * BUF;
  __shared__ __attribute__((aligned(16))) unsigned char smem[LDS];
  const Place pl = place_of<QB>(a);
  if (pl.seq < 0) {
    if (a.zero_rest) zero_rows<float, QB>(a, pl.h, pl.rest);
    return;
  }
  const int lane = threadIdx.x & 63, g = lane >> 4, c = lane & 15;
  const int w8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), w = w8 & 3, group = NG == 2 ? w8 >> 2 : 0;
  unsigned char* const mine = smem + group * 2 * BUF;
  const int len = pl.len, q0 = pl.q0, dh = a.dh, hk = pl.h / (a.H / a.Hkv);
  const int text = pl.text;
  const Tiles ti = tiles_of<TK>(q0, min(q0 + QB, len) - 1, text, a.window, a.sinks);
  const float* kb = (const float*)a.k + (int64_t)pl.off * a.k_row + (int64_t)hk * a.k_head;
  const float* vb = (const float*)a.v + (int64_t)pl.off * a.v_row + (int64_t)hk * a.v_head;
  const int i = q0 + w * 16 + c;
  const bool valid = i < len;
  const Sight see = sight_of(min(i, len - 1), text, a.window, a.sinks);
  const Sights rows = sights_of(min(q0 + w * 16, len - 1), min(q0 + w * 16 + 15, len - 1), text, a.window, a.sinks);
  wa_f32x4 qf[KT];
  const float* qp = (const float*)a.q + (int64_t)(pl.off + min(i, len - 1)) * a.q_row + (int64_t)pl.h * a.q_head;
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    qf[t] = wa_f32x4{0.f, 0.f, 0.f, 0.f};
    if (t * 16 + g * 4 < dh) qf[t] = *reinterpret_cast<const wa_f32x4*>(qp + t * 16 + g * 4);
  }
  const float sl2 = a.sl2;
  float m = -INFINITY, l = 0.f;
  wa_f32x4 o[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) o[j] = wa_f32x4{0.f, 0.f, 0.f, 0.f};
  auto key0 = [&](int t) { return (t < ti.th ? t : ti.mf + (t - ti.th)) * TK; };

  const Stager<float, TK, NV> stage_k(kb, a.k_row, len, dh, w), stage_v(vb, a.v_row, len, dh, w);
  if (group < ti.tt) {
    stage_k(key0(group), dh, mine);
    stage_v(key0(group), dh, mine + HALF);
  }
#pragma unroll
  for (int t = 0; t < KT; ++t) asm volatile("" : "+v"(qf[t]));  // as in the bf16 kernel
  for (int t0 = 0; t0 < ti.tt; t0 += NG) {
    const int t = t0 + group;
    const unsigned char* Ks = mine + (t0 / NG & 1) * BUF;
    const unsigned char* Vs = Ks + HALF;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + NG < ti.tt) {
      unsigned char* nb = mine + (t0 / NG + 1 & 1) * BUF;
      stage_k(key0(t + NG), dh, nb);
      stage_v(key0(t + NG), dh, nb + HALF);
    }
    if (t >= ti.tt) continue;
    const int kt0 = key0(t);
    if (rows.none(kt0, TK)) continue;
    wa_f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
    wa_f32x4 ka[2][2];  // [buffer][16-key tile]: the next 16 dims' fragments are read while these are multiplied
    auto read_k = [&](wa_f32x4 (&d)[2], int t4) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) d[kt] = *reinterpret_cast<const wa_f32x4*>(Ks + (kt * 16 + c) * ROW + (((t4 * 4 + g) ^ wa_key<NV>(c)) << 4));
    };
    read_k(ka[0], 0);
#pragma unroll
    for (int t4 = 0; t4 < KT; ++t4) {
      if (t4 + 1 < KT) read_k(ka[(t4 + 1) & 1], t4 + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(ka[t4 & 1][kt][u], qf[t4][u], s[kt], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
    const bool unmasked = rows.all(kt0, TK);
    float mt = -INFINITY;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[kt][r] = unmasked | see.sees(kt0 + kt * 16 + g * 4 + r) ? s[kt][r] : -INFINITY;
        mt = fmaxf(mt, s[kt][r]);
      }
    mt = rows4_max(mt);
    const float mn = fmaxf(m, mt);
    const float ref = mn == -INFINITY ? 0.f : mn;
    const float alpha = __builtin_amdgcn_exp2f((m - ref) * sl2);
    m = mn;
    float sum = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        s[kt][r] = __builtin_amdgcn_exp2f((s[kt][r] - ref) * sl2);
        sum += s[kt][r];
      }
    l = fmaf(l, alpha, sum);
    if (!__all(alpha == 1.0f)) {
#pragma unroll
      for (int j = 0; j < DPL; ++j) o[j] *= alpha;
    }
    auto read_v = [&](float (&vv)[DPL], int n) {  // this lane's dims of key 4 g + n % 4 of score tile n / 4
      const int key = (n >> 2) * 16 + g * 4 + (n & 3);
      const unsigned char* row = Vs + key * ROW;
      if constexpr (A4 == 4) {
        const wa_f32x4 x = *reinterpret_cast<const wa_f32x4*>(row + ((c ^ wa_key<NV>(key)) << 4));
#pragma unroll
        for (int j = 0; j < 4; ++j) vv[j] = x[j];
        if constexpr (B4 == 4) {
          const wa_f32x4 y = *reinterpret_cast<const wa_f32x4*>(row + (((16 + c) ^ wa_key<NV>(key)) << 4));
#pragma unroll
          for (int j = 0; j < 4; ++j) vv[4 + j] = y[j];
        } else if constexpr (B4 == 2) {
          const wa_f32x2 y = *reinterpret_cast<const wa_f32x2*>(row + (((16 + (c >> 1)) ^ wa_key<NV>(key)) << 4) + ((c & 1) << 3));
          vv[4] = y[0];
          vv[5] = y[1];
        }
      } else {
        const wa_f32x2 x = *reinterpret_cast<const wa_f32x2*>(row + (((c >> 1) ^ wa_key<NV>(key)) << 4) + ((c & 1) << 3));
        vv[0] = x[0];
        vv[1] = x[1];
      }
    };
    float vv[2][DPL];  // the next key's elements are read while these are multiplied
    read_v(vv[0], 0);
#pragma unroll
    for (int n = 0; n < 8; ++n) {
      if (n < 7) read_v(vv[(n + 1) & 1], n + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < DPL; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vv[n & 1][j], s[n >> 2][n & 3], o[j], 0, 0, 0);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  l = rows4_sum(l);
  if constexpr (NG == 2) {  // lane by lane: both groups hold the same rows and elements in the same places
    __syncthreads();        // the tiles are done with
    float* part = reinterpret_cast<float*>(smem) + w * 64 + lane;
    constexpr int N = 4 * 64;
    if (group == 1) {
      part[0] = m;
      part[N] = l;
#pragma unroll
      for (int j = 0; j < DPL; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) part[(2 + 4 * j + r) * N] = o[j][r];
    }
    __syncthreads();
    if (group == 1) return;
    const float m1 = part[0], mn = fmaxf(m, m1), ref = mn == -INFINITY ? 0.f : mn;
    const float f0 = __builtin_amdgcn_exp2f((m - ref) * sl2), f1 = __builtin_amdgcn_exp2f((m1 - ref) * sl2);
    l = l * f0 + part[N] * f1;
#pragma unroll
    for (int j = 0; j < DPL; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[j][r] = o[j][r] * f0 + part[(2 + 4 * j + r) * N] * f1;
  }
  bool odd = false;
  float* op = (float*)a.out + ((int64_t)(pl.off + i) * a.H + pl.h) * dh;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int slot = 4 * g + r;
#pragma unroll
    for (int j = 0; j < DPL; j += 2) {
      const int e = j < A4 ? A4 * slot + j : 16 * A4 + B4 * slot + (j - A4);
      if (e >= dh) continue;
      const wa_f32x2 x = {o[j][r] / l, o[j + 1][r] / l};
      odd |= !(fabsf(x[0]) < INFINITY) || !(fabsf(x[1]) < INFINITY);
      if (valid) *reinterpret_cast<wa_f32x2*>(op + e) = x;
    }
  }
  unsigned long long again = __ballot(odd && valid);
  if (again) {
    again = (again | (again >> 16) | (again >> 32) | (again >> 48)) & 0xffffull;
    while (again) {
      const int t = __builtin_ctzll(again);
      again &= again - 1;
      exact_row<float>(a, pl.h, pl.off, q0 + w * 16 + t, text, len);
    }
  }
}

int launch_window_attention(hipStream_t st, int dtype, const WindowAttnArgs& a) {
  if (a.rows <= 0) return 0;
  const bool f32 = dtype == DT_F32;
  // items of a head: the rows' runs, one more for every sequence's ragged last one, one for the rows of no sequence
  auto items = [&](int qb) { return (a.rows + qb - 1) / qb + a.B + 1; };
  // bf16, head size above 96, two workgroups a CU or more: 128 rows each, so that a fragment read from LDS feeds two products (no window, 32 heads of 128, sequences
  // of 1000 rows, 64 rows an item / 128: 1 of them (320 items of 128) 20.1 / 27.5 us, 2 (608) 33.1 / 31.2, 4 (1184) 59.5 / 59.2, 8 110 / 103; one of 12289 rows, 16
  // heads: 714 / 599, window 1024 145 / 123; 8 of 1000, 16 heads of 120: 71.5 / 62.9).  Smaller heads win nothing by it (16 of 1000, 16 heads of 96: 88.2 / 89.1, window 256
  // 59.8 / 62.0; 32 of 900, 16 heads of 64: 106.9 / 108.9, window 256 72.7 / 75.8).
  const bool wide = !f32 && a.dh > 96 && items(128) * a.H >= 512;
  const int64_t n = items(wide ? 128 : 64) * a.H;
  // fp32, about one workgroup a CU (without a window, where the late rows' work is the longest and goes first, up to one and a half): a second group of waves
  // halves each one's walk.  16 heads of 96, one group / two: no window, one sequence of 1300 rows (368 items) 103.5 / 80.8 us, of 1600 (432) 131.9 / 97.0, but of 2000 (544)
  // 141.8 / 167.4; window 256, 1024 rows (288) 28.9 / 27.4, but 1152 (320) 33.4 / 35.8 and 1300 41.8 / 47.8, where a second workgroup a CU is worth more.  (16-key tiles, which
  // leave room for it, are slower from 300 rows to 16 sequences: 58 / 61, 302 / 336.)
  const bool pair = f32 && n <= (a.window > 0 ? 320 : 448);
  if (n > 0xffffff) return -1;  // 2^32 work items
  const dim3 grid((unsigned)n), block(256);
#define VLE_WA(DHT)                                                                             \
  do {                                                                                          \
    if (pair) hipLaunchKernelGGL((window_attn_f32_kernel<DHT, 2>), grid, dim3(512), 0, st, a);   \
    else if (f32) hipLaunchKernelGGL((window_attn_f32_kernel<DHT, 1>), grid, block, 0, st, a);   \
    else if (wide) hipLaunchKernelGGL((window_attn_bf16_kernel<128, 2>), grid, block, 0, st, a); \
    else hipLaunchKernelGGL((window_attn_bf16_kernel<DHT, 1>), grid, block, 0, st, a);          \
  } while (0)
  if (a.dh <= 32) VLE_WA(32);
  else if (a.dh <= 64) VLE_WA(64);
  else if (a.dh <= 96) VLE_WA(96);
  else VLE_WA(128);
#undef VLE_WA
  return 0;
}

}  // namespace vle
