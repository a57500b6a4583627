// Paged key-value cache: writing new tokens, one new query per sequence against the pages, eviction by accumulated weight.
//
//   k_pages / v_pages T [n_pages][Hkv][ps][dh]   ps keys of one head are contiguous (ps * dh * sizeof(T) bytes): a wave reads whole lines
//   mass          f32  [n_pages][Hkv][ps]        attention weight every key has received so far
//   page_table   int32 [B][W]                    key j of sequence b lives in page page_table[b][j / ps], slot j % ps
//
// A page id outside [0, n_pages) is never dereferenced: its keys count as absent (not read, not written).  Lengths are clamped to W * ps.
// Offsets of a page are 64-bit, offsets inside one 32-bit.
#include <algorithm>

#include "common.h"
#include "kernels.h"

namespace vle {

namespace {

typedef __bf16 pc_bf16x8 __attribute__((ext_vector_type(8)));
typedef float pc_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned pc_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned pc_u32x2 __attribute__((ext_vector_type(2)));

// Keys of one wave step: bf16 32 (two 16-key score tiles feed one product with 32 contraction slots), fp32 16 (64 registers for its keys and values).
template <typename T>
constexpr int pc_tile() { return sizeof(T) == 4 ? 16 : 32; }

// The keys the newest token of a sequence sees: j < n and (j < hd or j >= lo), as tiles of TK keys.  Tiles 0 .. th - 1 cover the head,
// tile t >= th starts at key (mf + t - th) * TK; tiles between the head and the window are never touched.
template <int TK>
struct Span {
  int n, hd, lo, th, mf, tt;
  __device__ int key0(int t) const { return (t < th ? t : mf + (t - th)) * TK; }
  // & and | on purpose, here and where a mask is applied.  Not for speed: with && and || (a branch inside a step that only some waves take) hipcc of ROCm 7.2 left element 0
  // of a vector of scores unmasked for keys in the gap ahead of the window.  A select for every key is compiled right, behind a wave-uniform branch too.
  __device__ bool sees(int j) const { return (j < n) & ((j < hd) | (j >= lo)); }
  __device__ bool sees_tile(int j0) const { return (j0 + TK <= n) & ((j0 + TK <= hd) | (j0 >= lo)); }
};

template <int TK>
__device__ inline Span<TK> span_of_row(const PagedDecodeArgs& a, int b) {
  Span<TK> s;
  s.n = min(max(a.lengths[b], 0), a.W << a.psl);  // W * ps < 2^30 (checked at the entry)
  if (a.window <= 0 || a.window >= s.n) {
    s.hd = s.lo = s.n;
  } else {
    s.hd = min(s.n, max(a.text_len ? a.text_len[b] : 0, a.sinks));
    s.lo = s.n - a.window;
  }
  s.th = (s.hd + TK - 1) / TK;
  s.mf = max(s.th, s.lo / TK);
  s.tt = s.th + max(0, (s.n + TK - 1) / TK - s.mf);
  return s;
}

// Tiles of one split: the sequence's own, in equal parts of PD_CHUNK tiles at least.
constexpr int PD_CHUNK = 8;
__device__ inline int split_tiles(int tt, int nsplit) { return nsplit == 1 ? max(tt, 1) : max(PD_CHUNK, (tt + nsplit - 1) / nsplit); }

}  // namespace

// ---- writing ---------------------------------------------------------------------------------------------------------------------
// One wave per new token and per half (K, V): Hkv * dh elements in 16-byte vectors, contiguous reads, one dh-segment per head out.
// HBM-bound copy: 64 prompts of 150 - 420 rows, 16 heads of 64 (151 MB) 34 us = 4.4 TB/s, a plain copy reaches 4.9; one row for each of 6 sequences 3.0 us.
template <typename T>
__global__ __launch_bounds__(256) void paged_write_kernel(PagedWriteArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= a.rows) return;
  int b, at;
  if (a.seq_off == nullptr) {
    b = (int)row;
    at = 0;
  } else {  // the sequence that holds this row: how many end at or before it
    int ended = 0;
    for (int i = lane; i < a.B; i += 64) ended += a.seq_off[i + 1] <= row;
    b = wave_sum_i(ended);
    if (b >= a.B || row < a.seq_off[b] || row >= a.seq_off[b + 1]) return;  // behind the last sequence or ahead of the first
    at = (int)row - a.seq_off[b];
  }
  const int64_t pos = (int64_t)a.start[b] + at;
  if (pos < 0 || pos >= ((int64_t)a.W << a.psl)) return;
  const int page = a.table[(int64_t)b * a.W + (pos >> a.psl)];
  if ((unsigned)page >= (unsigned)a.n_pages) return;
  const int ps = 1 << a.psl, slot = (int)(pos & (ps - 1));
  constexpr int VEC = Elem<T>::VEC;
  const int vpd = a.dh / VEC, nv = a.Hkv * vpd;
  const int64_t base = (int64_t)page * a.Hkv * ps * a.dh;
  const T* src = (const T*)(blockIdx.y ? a.v : a.k) + row * (blockIdx.y ? a.v_row : a.k_row);
  const int64_t hs = blockIdx.y ? a.v_head : a.k_head;
  T* dst = (T*)(blockIdx.y ? a.v_pages : a.k_pages) + base;
  for (int i = lane; i < nv; i += 64) {
    const int h = i / vpd, e = (i - h * vpd) * VEC;
    *reinterpret_cast<pc_u32x4*>(dst + (h * ps + slot) * a.dh + e) = *reinterpret_cast<const pc_u32x4*>(src + h * hs + e);
  }
  if (blockIdx.y == 0 && a.mass != nullptr)
    for (int h = lane; h < a.Hkv; h += 64) a.mass[((int64_t)page * a.Hkv + h) * ps + slot] = 0.f;
}

int launch_paged_write(hipStream_t st, int dtype, const PagedWriteArgs& a) {
  if (a.rows <= 0) return 0;
  const dim3 grid((unsigned)((a.rows + 3) / 4), 2), block(256);
  if (dtype == DT_F32) hipLaunchKernelGGL((paged_write_kernel<float>), grid, block, 0, st, a);
  else hipLaunchKernelGGL((paged_write_kernel<bf16_t>), grid, block, 0, st, a);
  return 0;
}

// ---- one new token against its pages ---------------------------------------------------------------------------------------------
// Both products are computed transposed on the matrix pipe, up to 16 heads of a group as the 16 columns: S^T[key][head] = K Q^T leaves
// the weights of keys 4 g + r of both 16-key tiles in lane (g, c) -- g = lane / 16, c = lane % 16 = head -- which is where the second product
// O^T[dim][head] = V^T P^T wants them, if its contraction runs over the keys in that order.  V^T comes straight from the row-major pages:
// lane (g, c) loads dims c * DPL .. + DPL - 1 of its group's 8 keys (four whole rows per instruction) and one byte-permute per packed pair turns
// them into the operands of DPL products, product j giving dims 4-lane-slot * DPL + j.  No LDS, no barrier in the loop; a group of one
// head leaves 15 columns empty, which the matrix pipe has room for (it needs 1/16 of the time the HBM takes for the same keys).
//
// HBM-bound.  Measured: 3 sequences of 40k - 60k keys, 32 heads on 8 of 128, bf16 (684 MB): 111 us = 6.2 TB/s, and 4.9 the join; 16 sequences, window 1500
// of 9k - 30k keys, 16 heads of 96, fp32 (312 MB): 60 us = 5.2 TB/s, and 4.9; 64 sequences of 330 - 1100 keys, 16 heads of 64, with mass (216 MB): 50 us = 4.3
// TB/s, bound by the longest sequences, whose workgroups run on alone; one sequence of 1025 keys: 9.8 us, the steps' latency one after another.
// A second tile of registers on its way is slower, also where workgroups are few (138 -> 141 us and 73 -> 87 for the first two, at the time; 10.2 -> 10.6
// for the last).

// NT: past the memory-side cache
template <bool NT, typename V>
__device__ inline V pd_load(const void* p) {
  if constexpr (NT) return __builtin_nontemporal_load((const V*)p);
  else return *(const V*)p;
}
template <bool NT, int N>
__device__ inline void pd_load_words(unsigned (&dst)[N], const void* src) {  // N = 2, 4 or 8 words of 32 bits, from 8 or 16 aligned bytes on
  if constexpr (N == 2) {
    const pc_u32x2 x = pd_load<NT, pc_u32x2>(src);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const pc_u32x4 x = pd_load<NT, pc_u32x4>((const pc_u32x4*)src + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[4 * i + j] = x[j];
    }
  }
}

// Element e of one head's output once more, by one wave (an element a lane): the running average of the visible values instead of their sum over a denominator.
// For results that are not finite, a rarity: a sum past the largest number, whose average need not be, and infinities, which the two parts of a bf16 weight
// (one of them may be negative) turn into NaN.  64 keys at a time, a lane the score of one; 8 values on their way.
// Done early where every element that is asked for is NaN already.
template <typename T, int TK>
__device__ inline float pd_exact(const PagedDecodeArgs& a, const Span<TK>& sp, int b, int h, int e, bool asked) {
#pragma clang fp contract(off)  // as for the scores of the kernel below
  constexpr int VE = Elem<T>::VEC;
  const int lane = threadIdx.x & 63, kvh = h / a.G, ps = 1 << a.psl;
  const int64_t page_elems = (int64_t)a.Hkv * ps * a.dh;
  const T* q = (const T*)a.q + (int64_t)b * a.q_b + (int64_t)h * a.q_h;
  const T* kbase = (const T*)a.k_pages + (int64_t)kvh * ps * a.dh;
  const T* vbase = (const T*)a.v_pages + (int64_t)kvh * ps * a.dh;
  e = min(e, a.dh - 1);
  float m = -INFINITY, l = 0.f, o = 0.f;
  for (int i0 = 0; i0 < sp.tt * TK; i0 += 64) {
    const int i = i0 + lane, j = sp.key0(i / TK) + i % TK;
    const bool in = (i < sp.tt * TK) & sp.sees(j);
    const int id = in ? a.table[(int64_t)b * a.W + (j >> a.psl)] : -1;
    const bool vis = (unsigned)id < (unsigned)a.n_pages;
    const int page = vis ? id : 0, at = vis ? (j & (ps - 1)) * a.dh : 0;  // what is not visible is not looked at: its loads go to the pool's first key
    if (!__any(vis)) continue;
    float s = -INFINITY;
    if (vis) {
      float sum = 0.f;
      for (int d = 0; d < a.dh; d += VE) {
        float x[VE], y[VE];
        load_vec16(q + d, x);
        load_vec16(kbase + (int64_t)page * page_elems + at + d, y);
#pragma unroll
        for (int u = 0; u < VE; ++u) sum = fmaf(x[u], y[u], sum);
      }
      s = sum * a.sl2;
    }
    if (__any(s != s)) return __builtin_nanf("");
    const float mn = fmaxf(m, wave_max(s)), ref = mn == -INFINITY ? 0.f : mn;
    const float p = __builtin_amdgcn_exp2f(s - ref), was = l * __builtin_amdgcn_exp2f(m - ref), now = was + wave_sum(p);
    m = mn;
    l = now;
    if (now == 0.f) continue;  // nothing but -inf so far
    o *= was / now;
    const float w = p / now;
    for (int t0 = 0; t0 < 64; t0 += 8) {
      float x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u)
        x[u] = Elem<T>::to_f32(vbase[(int64_t)__builtin_amdgcn_readlane(page, t0 + u) * page_elems + __builtin_amdgcn_readlane(at, t0 + u) + e]);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (__builtin_amdgcn_readlane((int)vis, t0 + u)) o = fmaf(readlane_f32(w, t0 + u), x[u], o);
    }
    if (!__any(asked & (o == o))) break;
  }
  return l == 0.f ? __builtin_nanf("") : o;
}

// WHOLE: dh == DHT, no lane is ever outside the head.  SPLIT: parts for the join; a kernel of its own, because what only a whole head needs (pd_exact, the weights)
// costs the walk scalar registers: 16 sequences, window 1500 (fp32, heads of 96): 65.9 -> 65.1 us
template <typename T, int DHT, int NW, bool WHOLE, bool NT, bool SPLIT>
__global__ __launch_bounds__(NW * 64, NW == 4 ? 3 : 1) void paged_decode_kernel(PagedDecodeArgs a) {
  constexpr bool BF = sizeof(T) == 2;
  constexpr int TK = pc_tile<T>(), ST = TK / 16;  // 16-key score tiles of a step
  constexpr int DPL = DHT / 16;                   // head elements per lane of a V row
  constexpr int KV = BF ? DHT / 32 : DHT / 16;    // 16-byte K vectors per lane and score tile
  constexpr int KE = BF ? 8 : 4;                  // elements per such vector
  constexpr int VW = DPL * (int)sizeof(T) / 4;    // 32-bit words per lane of a V row
  extern __shared__ float sm[];  // [NW][ng][DHT] outputs, [NW][16][2] (m, l), [16][2] (m, 1 / l), [ng][score_lds] scores

  const int split = SPLIT ? (int)blockIdx.x : 0, b = blockIdx.z;
  const int kvh = (int)blockIdx.y / a.GT, gt = (int)blockIdx.y - kvh * a.GT;
  const int h0 = kvh * a.G + gt * 16, ng = min(16, a.G - gt * 16);
  const Span<TK> sp = span_of_row<TK>(a, b);
  const int chunk = split_tiles(sp.tt, SPLIT ? a.nsplit : 1), t0 = split * chunk, t1 = min(t0 + chunk, sp.tt);
  const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4, c = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);  // wave-uniform, and with it everything about a step but the lanes' own places
  const int H = a.Hkv * a.G, ps = 1 << a.psl, dh = WHOLE ? DHT : a.dh;
  if (SPLIT && split > 0 && t0 >= sp.tt) return;  // nothing of this sequence is left for this split, and the join does not read it

  float* sm_ml = sm + NW * ng * DHT;
  float* sm_stat = sm_ml + NW * 32;
  float* sm_score = sm_stat + 32;
  const int32_t* tab = a.table + (int64_t)b * a.W;
  // page ids: lane i holds the page of key key0 + i of one step, fetched a step ahead of the keys; -1: not there
  auto load_ids = [&](int t) -> int {
    int id = -1;
    if (t < t1) {
      const int j = sp.key0(t) + (lane & (TK - 1));
      if (j < sp.n) id = tab[j >> a.psl];
    }
    return (unsigned)id < (unsigned)a.n_pages ? id : -1;
  };
  int ids = load_ids(t0 + w);

  pc_u32x4 qf[KV];
  {
    const T* qp = (const T*)a.q + (int64_t)b * a.q_b + (int64_t)(h0 + min(c, ng - 1)) * a.q_h + g * KE;
#pragma unroll
    for (int i = 0; i < KV; ++i) {
      qf[i] = pc_u32x4{0u, 0u, 0u, 0u};
      if (c < ng && (WHOLE || i * 4 * KE + g * KE < dh)) qf[i] = *reinterpret_cast<const pc_u32x4*>(qp + i * 4 * KE);
    }
  }
  const int64_t page_elems = (int64_t)a.Hkv * ps * dh;
  const T* kbase = (const T*)a.k_pages + (int64_t)kvh * ps * dh;
  const T* vbase = (const T*)a.v_pages + (int64_t)kvh * ps * dh;
  const int koff = c * dh + g * KE, voff = 4 * g * dh + c * DPL;
  const bool vin = WHOLE || c * DPL < dh;  // dh is a multiple of 8: a lane's elements are inside the head or outside it

  float m = -INFINITY, l = -0.0f;  // l stays -0 until a visible key was met: a row that sees nothing answers 0, not 0 / 0
  pc_f32x4 o[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) o[j] = pc_f32x4{0.f, 0.f, 0.f, 0.f};

  for (int t = t0 + w; t < t1; t += NW) {
    const int k0 = sp.key0(t);
    pc_u32x4 kf[ST][KV];
    unsigned vf[4 * ST][VW];
    int page[ST];  // page of keys 4 g + r of each score tile (four keys share one, ps >= 8)
    // all keys visible and every score tile on one page that is there: uniform bases, no predicates
    bool plain = (a.psl >= 4) & sp.sees_tile(k0);
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      page[st] = __shfl(ids, 16 * st + 4 * g, 64);
      plain = plain & (__builtin_amdgcn_readlane(ids, 16 * st) >= 0);
    }
    if (plain) {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int64_t at = (int64_t)__builtin_amdgcn_readlane(ids, 16 * st) * page_elems + ((k0 + 16 * st) & (ps - 1)) * dh;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          if (!WHOLE) kf[st][i] = pc_u32x4{0u, 0u, 0u, 0u};
          if (WHOLE || i * 4 * KE + g * KE < dh) kf[st][i] = pd_load<NT, pc_u32x4>(kbase + at + koff + i * 4 * KE);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          if (!WHOLE) {
#pragma unroll
            for (int i = 0; i < VW; ++i) vf[4 * st + r][i] = 0;
          }
          if (vin) pd_load_words<NT>(vf[4 * st + r], vbase + at + voff + r * dh);
        }
      }
    } else {
#pragma unroll
      for (int st = 0; st < ST; ++st) {
        const int id = __shfl(ids, 16 * st + c, 64), key = k0 + 16 * st + c;
        const T* p = kbase + (int64_t)max(id, 0) * page_elems + (key & (ps - 1)) * dh + g * KE;
#pragma unroll
        for (int i = 0; i < KV; ++i) {
          kf[st][i] = pc_u32x4{0u, 0u, 0u, 0u};
          if (id >= 0 && (WHOLE || i * 4 * KE + g * KE < dh)) kf[st][i] = *reinterpret_cast<const pc_u32x4*>(p + i * 4 * KE);
        }
        const int k4 = k0 + 16 * st + 4 * g;
        const T* pv = vbase + (int64_t)max(page[st], 0) * page_elems + (k4 & (ps - 1)) * dh + c * DPL;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int i = 0; i < VW; ++i) vf[4 * st + r][i] = 0;
          if ((page[st] >= 0) & vin & sp.sees(k4 + r)) pd_load_words<false>(vf[4 * st + r], pv + r * dh);  // what nobody sees may hold anything, NaN included
        }
      }
    }
    ids = load_ids(t + NW);
    // ---- scores, in units of the exp2 argument ----
    pc_f32x4 s[ST];
    bool any = plain;
#pragma unroll
    for (int st = 0; st < ST; ++st) {
      s[st] = pc_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        if constexpr (BF) {
          s[st] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pc_bf16x8, kf[st][i]), __builtin_bit_cast(pc_bf16x8, qf[i]), s[st], 0, 0, 0);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) s[st] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kf[st][i][u]), __uint_as_float(qf[i][u]), s[st], 0, 0, 0);
        }
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma clang fp contract(off)  // the rounded product: its difference to the maximum must be 0 for the largest, whatever its size
        if constexpr (BF) {
          s[st][r] = s[st][r] * a.sl2;
        } else {
          const bool vis = plain | ((page[st] >= 0) & sp.sees(k0 + 16 * st + 4 * g + r));
          any |= vis;
          const float x = s[st][r] * a.sl2;
          s[st][r] = vis ? x : -INFINITY;
        }
      }
    }
    if (BF && !plain) {  // behind a branch: one sequence of 1040 keys 10.4 -> 9.9 us in a graph, 64 sequences unchanged; fp32, whose steps have half the keys, is 2 % slower that way
#pragma unroll
      for (int st = 0; st < ST; ++st)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const bool vis = (page[st] >= 0) & sp.sees(k0 + 16 * st + 4 * g + r);
          any |= vis;
          s[st][r] = vis ? s[st][r] : -INFINITY;
        }
    }
    if (a.mass != nullptr && c < ng) {
      float* sc = !SPLIT && a.score_lds ? sm_score + c * a.score_lds + t * TK + 4 * g : a.scores + ((int64_t)b * H + h0 + c) * a.score_ld + (int64_t)t * TK + 4 * g;
#pragma unroll
      for (int st = 0; st < ST; ++st) *reinterpret_cast<pc_f32x4*>(sc + 16 * st) = s[st];
    }
    if (!__any(any)) continue;
    // ---- online softmax of column c ----
    float mt = fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3]));
    if constexpr (ST == 2) mt = fmaxf(mt, fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mt = rows4_max(mt);
    const float mn = fmaxf(m, mt);
    const float ref = mn == -INFINITY ? 0.f : mn;  // every score so far is -inf: their weights are 0, not exp(-inf + inf)
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    float p[4 * ST], sum = 0.f;
#pragma unroll
    for (int st = 0; st < ST; ++st)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        p[4 * st + r] = __builtin_amdgcn_exp2f(s[st][r] - ref);
        sum += p[4 * st + r];
      }
    l = fmaf(l, alpha, sum);
    if (!__all(alpha == 1.0f)) {
#pragma unroll
      for (int j = 0; j < DPL; ++j) o[j] *= alpha;
    }
    // ---- O^T += V^T P^T ----
    if constexpr (BF) {
      // the weights as the sum of two bf16 numbers (16 bits kept): the matrix pipe idles, and the output then carries one rounding, its own
      pc_bf16x8 hi, lo;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        hi[i] = (__bf16)p[i];
        lo[i] = (__bf16)(p[i] - (float)hi[i]);
      }
#pragma unroll
      for (int j = 0; j < DPL; ++j) {
        pc_u32x4 f;
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __builtin_amdgcn_perm(vf[2 * i + 1][j >> 1], vf[2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pc_bf16x8, f), hi, o[j], 0, 0, 0);
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pc_bf16x8, f), lo, o[j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4 * ST; ++i)
#pragma unroll
        for (int j = 0; j < DPL; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vf[i][j]), p[i], o[j], 0, 0, 0);
    }
  }

  // ---- the waves' parts meet in LDS ----
  l = rows4_sum(l);
  if (c < ng) {
    float* so = sm + (w * ng + c) * DHT;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < DPL; ++j) so[(4 * g + i) * DPL + j] = o[j][i];
    if (g == 0) {
      sm_ml[(w * 16 + c) * 2] = m;
      sm_ml[(w * 16 + c) * 2 + 1] = l;
    }
  }
  __syncthreads();
  if (tid < ng) {  // one head each: (m, l) over the waves; sm_ml[w][h][0] becomes wave w's factor
    float M = -INFINITY, L = -0.0f;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, sm_ml[(i * 16 + tid) * 2]);
    const float ref = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float f = __builtin_amdgcn_exp2f(sm_ml[(i * 16 + tid) * 2] - ref);
      L += sm_ml[(i * 16 + tid) * 2 + 1] * f;
      sm_ml[(i * 16 + tid) * 2] = f;
    }
    sm_stat[tid * 2] = ref;
    sm_stat[tid * 2 + 1] = __float_as_uint(L) == 0x80000000u ? 0.f : 1.0f / L;
    if (a.part_ml != nullptr) {
      float* ml = a.part_ml + (((int64_t)b * H + h0 + tid) * (SPLIT ? a.nsplit : 1) + split) * 2;
      ml[0] = M;
      ml[1] = L;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < ng * DHT; idx += NW * 64) {
    const int hh = idx / DHT, e = idx - hh * DHT;  // (a wave's lanes are in one head: 64 divides DHT)
    const bool in = WHOLE || e < dh;
    float O = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) O += sm[(i * ng + hh) * DHT + e] * sm_ml[(i * 16 + hh) * 2];
    if constexpr (!SPLIT) {
      float x = O * sm_stat[hh * 2 + 1];
      const bool odd = in & !(fabsf(x) < INFINITY);
      if (__builtin_expect(__any(odd), 0)) {
        const float again = pd_exact<T, TK>(a, sp, b, h0 + hh, e, odd);
        x = odd ? again : x;
      }
      if (in) store_elem<T>((T*)a.out + ((int64_t)b * H + h0 + hh) * dh + e, x);
    } else if (in) {
      a.part_o[(((int64_t)b * H + h0 + hh) * a.nsplit + split) * dh + e] = O;
    }
  }
  if (SPLIT || a.score_lds == 0) return;
  for (int idx = tid; idx < sp.tt * TK; idx += NW * 64) {  // the weights of this workgroup's keys and heads
    const int j = sp.key0(idx / TK) + idx % TK;
    if (!sp.sees(j)) continue;
    const int id = tab[j >> a.psl];
    if ((unsigned)id >= (unsigned)a.n_pages) continue;
    float sum = 0.f;
    for (int h = 0; h < ng; ++h) sum += __builtin_amdgcn_exp2f(sm_score[h * a.score_lds + idx] - sm_stat[h * 2]) * sm_stat[h * 2 + 1];
    // an atomic, because sequences may share the pages of a common prefix; without sharing there is one addend and one result
    unsafeAtomicAdd(a.mass + ((int64_t)id * a.Hkv + kvh) * ps + (j & (ps - 1)), sum);
  }
}

// Joins the splits and adds up the weights where a workgroup could not do it alone.  blockIdx.x < a.join_heads: one query head's output; behind them
// PD_JOIN_KEYS keys each of the weights.
constexpr int PD_JOIN_KEYS = 1024, PD_MAX_GROUP = 256, PD_MAX_SPLIT = 256;

template <typename T>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(PagedDecodeArgs a) {
  constexpr int TK = pc_tile<T>();
  __shared__ float sh_a[256], sh_b[256];
  __shared__ float sh_o[256 * 4];
  const int b = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int H = a.Hkv * a.G, ps = 1 << a.psl, dh = a.dh;
  const Span<TK> sp = span_of_row<TK>(a, b);
  const int chunk = split_tiles(sp.tt, a.nsplit), used = max(1, (sp.tt + chunk - 1) / chunk);
  // (reference, 1 / sum) of one head over its splits, by one wave
  auto stats = [&](const float* ml, float& ref, float& inv) {
    float M = -INFINITY, L = -0.0f;
    for (int s = lane; s < used; s += 64) M = fmaxf(M, ml[2 * s]);
    M = wave_max(M);
    ref = M == -INFINITY ? 0.f : M;
    for (int s = lane; s < used; s += 64) L += ml[2 * s + 1] * __builtin_amdgcn_exp2f(ml[2 * s] - ref);
    L = wave_sum(L);
    inv = __float_as_uint(L) == 0x80000000u ? 0.f : 1.0f / L;
  };
  if ((int)blockIdx.x < a.join_heads) {
    const int64_t hb = (int64_t)b * H + kvh * a.G + blockIdx.x;
    const float* ml = a.part_ml + hb * a.nsplit * 2;
    float ref, inv;
    stats(ml, ref, inv);
    if (tid < used) sh_a[tid] = __builtin_amdgcn_exp2f(ml[2 * tid] - ref);
    __syncthreads();
    // dh / 4 threads a row of partial outputs, 256 / (dh / 4) rows at a time
    const int vpr = dh / 4, rows = 256 / vpr, e = (tid % vpr) * 4, r0 = tid / vpr;
    pc_f32x4 O = {0.f, 0.f, 0.f, 0.f};
    if (r0 < rows)
      for (int s = r0; s < used; s += rows) O += *reinterpret_cast<const pc_f32x4*>(a.part_o + (hb * a.nsplit + s) * dh + e) * sh_a[s];
    *reinterpret_cast<pc_f32x4*>(sh_o + tid * 4) = O;
    __syncthreads();
    if (w * 64 >= dh) return;
    float x = 0.f;
    for (int r = 0; r < rows; ++r) x += sh_o[r * vpr * 4 + min(tid, dh - 1)];
    x *= inv;
    const bool odd = (tid < dh) & !(fabsf(x) < INFINITY);
    if (__builtin_expect(__any(odd), 0)) {
      const float again = pd_exact<T, TK>(a, sp, b, kvh * a.G + blockIdx.x, tid, odd);
      x = odd ? again : x;
    }
    if (tid < dh) store_elem<T>((T*)a.out + hb * dh + tid, x);
    return;
  }
  const int part = (int)blockIdx.x - a.join_heads;
  if (part * PD_JOIN_KEYS >= sp.tt * TK) return;
  for (int h = w; h < a.G; h += 4) {
    float ref, inv;
    stats(a.part_ml + ((int64_t)b * H + kvh * a.G + h) * a.nsplit * 2, ref, inv);
    if (lane == 0) {
      sh_a[h] = ref;
      sh_b[h] = inv;
    }
  }
  __syncthreads();
  for (int idx = part * PD_JOIN_KEYS + tid; idx < min((part + 1) * PD_JOIN_KEYS, sp.tt * TK); idx += 256) {
    const int j = sp.key0(idx / TK) + idx % TK;
    if (!sp.sees(j)) continue;
    const int page = a.table[(int64_t)b * a.W + (j >> a.psl)];
    if ((unsigned)page >= (unsigned)a.n_pages) continue;
    const float* sc = a.scores + ((int64_t)b * H + kvh * a.G) * a.score_ld + idx;
    float sum = 0.f;
    for (int h = 0; h < a.G; ++h) sum += __builtin_amdgcn_exp2f(sc[h * a.score_ld] - sh_a[h]) * sh_b[h];
    unsafeAtomicAdd(a.mass + ((int64_t)page * a.Hkv + kvh) * ps + (j & (ps - 1)), sum);
  }
}

static int pd_tiles_bound(int W, int ps, int window, int sinks, bool text, int tk) {  // tiles of a sequence, at most
  const int64_t n = (int64_t)W * ps;
  const int full = (int)((n + tk - 1) / tk);
  if (window <= 0 || window >= n || text) return full;
  return (int)std::min((int64_t)full, ((int64_t)sinks + tk - 1) / tk + ((int64_t)window + tk - 1) / tk + 1);
}

PagedDecodePlan paged_decode_plan(int dtype, int B, int Hkv, int G, int dh, int W, int ps, int window, int sinks, bool text, bool mass) {
  PagedDecodePlan p;
  const int tk = dtype == DT_F32 ? 16 : 32, ng = std::min(16, G);
  p.tiles = std::max(1, pd_tiles_bound(W, ps, window, sinks, text, tk));
  const int64_t groups = (int64_t)B * Hkv * ((G + 15) / 16), H = (int64_t)Hkv * G;
  // Workgroups of 4 waves that are resident at once: 256 CUs, 3 each (5 at head size 64).  One round of equal parts: 32 splits of three 40k - 60k
  // caches with 8 heads take 113 us, 43 (one third more than fit) 128, 64 (two rounds) 116, 128 (shorter parts, a longer join) 121.
  const int64_t slots = 256 * (dh <= 64 ? 5 : 3);
  p.nsplit = 1;
  // 8 waves where groups are few (their outputs fit 32 KB of LDS for up to 8 heads), 8 / 4 in a graph, 16 heads of 64: one sequence of 600 keys 6.6 / 8.9 us; 16 of 2000
  // 26.7 / 34.4; 24 of 1000 23.2 / 22.0; 32 of 2000 45.0 / 46.1; 64 sequences: no difference.  fp32: 12.3 / 16.6, 43.9 / 63.2, 42.0 / 39.5, 84.9 / 82.4
  p.nw = groups < 512 && ng <= 8 ? 8 : 4;
  // One workgroup a head takes 7 us per 1000 keys of 64 (a CU alone pulls about 40 GB/s), the join costs 3 us and a launch on the host.  16 heads of 64, unsplit / split:
  // one sequence of 1040 keys 10.0 / 14.4 us a call (9.1 / 8.8 in a graph), of 1300 10.8 / 15.0 (10.5 / 8.9), of 1500 11.6 / 14.8 (11.4 / 9.3), of 2040 14.7 / 14.8 (14.8 / 9.6);
  // fp32, whose tiles have half the keys, of 600 12.5 / 14.3 (12.3 / 9.3), of 1040 19.2 / 14.8.  A group for every CU needs no split yet at 2000 keys (16
  // sequences: 27.8 / 32.0 us, fp32 47.5 / 50.3), nor do two (32 of 2000: 47.8 / 52.2) or four (64 of 600: 29.3 / 29.3), for sequences of equal lengths.
  if (groups < 512 && p.tiles > (groups < 256 ? 5 : 16) * p.nw) {
    p.nw = 4;
    p.nsplit = (int)std::min((int64_t)std::min(PD_MAX_SPLIT, (p.tiles + PD_CHUNK - 1) / PD_CHUNK), std::max((int64_t)1, slots / groups));
  }
  // past the memory-side cache where the keys do not fit: 585 MB 114 -> 99 us, 250 MB 50.7 -> 46.2; 31 MB that would have stayed there 10.8 -> 14.1.  Head sizes 64 and 128
  // alone have a kernel for it: at 96 it made no difference (fp32, 750 MB 141.8 / 142.4; bf16, 375 MB 73.9 / 71.5)
  p.stream = (int64_t)p.tiles * tk * B * Hkv * dh * (dtype == DT_F32 ? 8 : 4) > (int64_t)128 << 20;
  // weights: by the workgroup that has all of a head's scores, where they fit beside its outputs; else by the join (64 sequences of 330 - 1100 keys,
  // 16 heads: 50 us, by the join 56)
  p.score_lds = mass && p.nsplit == 1 && G <= 16 && (int64_t)p.tiles * tk * ng <= 7168 ? p.tiles * tk : 0;
  const bool join_mass = mass && p.score_lds == 0;
  p.ml_floats = (p.nsplit > 1 || join_mass) ? (size_t)(B * H * p.nsplit * 2) : 0;
  p.o_floats = p.nsplit > 1 ? (size_t)(B * H * p.nsplit * dh) : 0;
  p.score_floats = join_mass ? (size_t)(B * H) * p.tiles * tk : 0;
  return p;
}

template <typename T, int DHT, int NW, bool SPLIT>
static void pd_launch_nw(hipStream_t st, const PagedDecodePlan& p, const PagedDecodeArgs& a, int B) {
  const int ng = std::min(16, a.G);
  const size_t lds = ((size_t)NW * ng * DHT + NW * 32 + 32 + (size_t)ng * p.score_lds) * sizeof(float);
  const dim3 grid(p.nsplit, a.Hkv * a.GT, B), block(NW * 64);
  if (a.dh != DHT) hipLaunchKernelGGL((paged_decode_kernel<T, DHT, NW, false, false, SPLIT>), grid, block, lds, st, a);
  else if (p.stream) hipLaunchKernelGGL((paged_decode_kernel<T, DHT, NW, true, true, SPLIT>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((paged_decode_kernel<T, DHT, NW, true, false, SPLIT>), grid, block, lds, st, a);
}

template <typename T, int DHT>
static int pd_launch(hipStream_t st, const PagedDecodePlan& p, PagedDecodeArgs& a, int B) {
  if (p.nsplit > 1) pd_launch_nw<T, DHT, 4, true>(st, p, a, B);
  else if (p.nw == 8) pd_launch_nw<T, DHT, 8, false>(st, p, a, B);
  else pd_launch_nw<T, DHT, 4, false>(st, p, a, B);
  a.join_heads = p.nsplit > 1 ? a.G : 0;
  const int parts = a.join_heads + (p.score_floats ? (p.tiles * pc_tile<T>() + PD_JOIN_KEYS - 1) / PD_JOIN_KEYS : 0);
  if (parts > 0) hipLaunchKernelGGL((paged_decode_join_kernel<T>), dim3(parts, a.Hkv, B), dim3(256), 0, st, a);
  return 0;
}

int launch_paged_decode(hipStream_t st, int dtype, const PagedDecodePlan& p, PagedDecodeArgs a, int B) {
  if (B <= 0) return 0;
  if (a.G > PD_MAX_GROUP) return -1;
  a.GT = (a.G + 15) / 16;
  a.nsplit = p.nsplit;
  a.score_lds = p.score_lds;
  a.score_ld = (int64_t)p.tiles * (dtype == DT_F32 ? 16 : 32);
  if (dtype == DT_F32) return a.dh <= 64 ? pd_launch<float, 64>(st, p, a, B) : pd_launch<float, 128>(st, p, a, B);
  return a.dh <= 64 ? pd_launch<bf16_t, 64>(st, p, a, B) : pd_launch<bf16_t, 128>(st, p, a, B);
}

// ---- eviction ----------------------------------------------------------------------------------------------------------------------
// Which keys stay: the first S and the last R of n, and of the n - S - R between them the M = budget - S - R with the most weight (of equal
// weights the earlier).  One workgroup per (sequence, head) finds the M-th largest weight by three counting passes over its order-preserving
// 32-bit key (11 + 11 + 10 bits, 2048 counters in LDS), then numbers the keys that stay in one more pass in the order of their positions.
// Bound by the passes' latency: 4 sequences of 900 - 1500 keys, 16 heads: 7.2 us; 32 sequences of 4.5k - 9k keys, 8 heads: 16 - 21 us.
constexpr int EV_T = 1024, EV_NW = EV_T / 64, EV_BINS = 2048;

__device__ inline uint32_t ev_key(float m) {  // larger weight, larger key; NaN above everything, -0 = +0
  if (m != m) return 0xffffffffu;
  return float_key(m == 0.f ? 0.f : m);
}

struct EvictRow {
  int n, S, R, M;
};
__device__ inline EvictRow evict_row(const EvictArgs& a, int b) {
  EvictRow r;
  r.n = min(max(a.lengths[b], 0), a.W << a.psl);
  r.S = min(min(r.n, a.budget), max(a.text_len ? a.text_len[b] : 0, a.sinks));
  r.S = max(r.S, 0);
  r.R = min(a.recent, a.budget - r.S);
  r.M = a.budget - r.S - r.R;
  return r;
}

// KPT > 0: the keys of up to EV_T * KPT candidates stay in registers; KPT = 0: any number, read again in every pass.
template <int KPT>
__global__ __launch_bounds__(EV_T) void kv_evict_select_kernel(EvictArgs a) {
  __shared__ int bins[3][EV_BINS];
  __shared__ int wsum[EV_NW], wsum2[EV_NW];
  __shared__ int cnt[2][(KPT > 0 ? KPT : 1) * EV_NW];
  __shared__ int sh_bin, sh_above;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, ps = 1 << a.psl;
  const EvictRow r = evict_row(a, b);
  int32_t* kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
  if (h == 0 && tid == 0) a.new_lengths[b] = min(r.n, a.budget);
  if (r.n <= a.budget) {
    for (int i = tid; i < a.budget; i += EV_T) kept[i] = i < r.n ? i : -1;
    return;
  }
  const int C = r.n - r.S - r.R;  // > M
  const int32_t* tab = a.table + (int64_t)b * a.W;
  auto weight = [&](int i) -> uint32_t {  // key of candidate i; the keys of a page that is not there have no weight
    const int j = r.S + i, page = tab[j >> a.psl];
    return (unsigned)page < (unsigned)a.n_pages ? ev_key(a.mass[((int64_t)page * a.Hkv + h) * ps + (j & (ps - 1))]) : ev_key(0.f);
  };
  uint32_t key[KPT > 0 ? KPT : 1];
#pragma unroll
  for (int u = 0; u < KPT; ++u) key[u] = u * EV_T + tid < C ? weight(u * EV_T + tid) : 0u;
  for (int i = tid; i < r.S; i += EV_T) kept[i] = i;
  for (int i = tid; i < r.R; i += EV_T) kept[r.S + r.M + i] = r.n - r.R + i;
  if (r.M == 0) return;
  for (int i = tid; i < 3 * EV_BINS; i += EV_T) (&bins[0][0])[i] = 0;
  __syncthreads();
  uint32_t prefix = 0, have = 0;  // the bits of the M-th largest key that are known, and their mask
  int need = r.M;                 // its rank among the keys that agree with them
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, nb = pass == 2 ? 1024 : 2048;
    int* bin = bins[pass];
    if constexpr (KPT > 0) {
#pragma unroll
      for (int u = 0; u < KPT; ++u)
        if (u * EV_T + tid < C && (key[u] & have) == prefix) atomicAdd(&bin[(key[u] >> shift) & (nb - 1)], 1);
    } else {
      for (int i = tid; i < C; i += EV_T) {
        const uint32_t k = weight(i);
        if ((k & have) == prefix) atomicAdd(&bin[(k >> shift) & (nb - 1)], 1);
      }
    }
    __syncthreads();
    // thread t counts bins 2047 - 2 t and 2046 - 2 t: an inclusive scan from the top finds the bin the need-th largest falls into
    const int hi = bin[EV_BINS - 1 - 2 * tid], lo = bin[EV_BINS - 2 - 2 * tid];
    const int inc = wave_scan_i(hi + lo);
    if (lane == 63) wsum[w] = inc;
    __syncthreads();
    int before = inc - hi - lo;
#pragma unroll
    for (int i = 0; i < EV_NW; ++i) before += i < w ? wsum[i] : 0;
    if (before < need && need <= before + hi) {
      sh_bin = EV_BINS - 1 - 2 * tid;
      sh_above = before;
    } else if (before + hi < need && need <= before + hi + lo) {
      sh_bin = EV_BINS - 2 - 2 * tid;
      sh_above = before + hi;
    }
    __syncthreads();
    prefix |= (uint32_t)sh_bin << shift;
    have |= (uint32_t)(nb - 1) << shift;
    need -= sh_above;
  }
  // every key above `prefix` stays, and of those equal to it the first `need`
  const unsigned long long below = (1ull << lane) - 1;
  auto keep = [&](int i, bool gt, bool eq, int gt_before, int eq_before) {
    const int at = gt_before + min(eq_before, need);
    if ((gt || (eq && eq_before < need)) && at < r.M) kept[r.S + at] = r.S + i;  // at < M always, unless the weights change during the call
  };
  if constexpr (KPT > 0) {
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const bool in = u * EV_T + tid < C;
      const unsigned long long beq = __ballot(in && key[u] == prefix), bgt = __ballot(in && key[u] > prefix);
      if (lane == 0) {
        cnt[0][u * EV_NW + w] = __popcll(bgt);
        cnt[1][u * EV_NW + w] = __popcll(beq);
      }
    }
    __syncthreads();
    if (w < 2) {  // exclusive scan of each list by one wave, in the order of the positions
      constexpr int PER = (KPT * EV_NW + 63) / 64;
      int v[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        v[i] = lane * PER + i < KPT * EV_NW ? cnt[w][lane * PER + i] : 0;
        sum += v[i];
      }
      int inc = wave_scan_i(sum) - sum;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        if (lane * PER + i < KPT * EV_NW) cnt[w][lane * PER + i] = inc;
        inc += v[i];
      }
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < KPT; ++u) {
      const int i = u * EV_T + tid;
      const bool eq = i < C && key[u] == prefix, gt = i < C && key[u] > prefix;
      const unsigned long long beq = __ballot(eq), bgt = __ballot(gt);
      keep(i, gt, eq, cnt[0][u * EV_NW + w] + __popcll(bgt & below), cnt[1][u * EV_NW + w] + __popcll(beq & below));
    }
  } else {
    int run = 0, run_eq = 0;
    for (int i0 = 0; i0 < C; i0 += EV_T) {
      const int i = i0 + tid;
      const uint32_t k = i < C ? weight(i) : 0u;
      const bool eq = i < C && k == prefix, gt = i < C && k > prefix;
      const unsigned long long beq = __ballot(eq), bgt = __ballot(gt);
      if (lane == 0) {
        wsum[w] = __popcll(beq);
        wsum2[w] = __popcll(bgt);
      }
      __syncthreads();
      int eq_before = run_eq + __popcll(beq & below), gt_before = run + __popcll(bgt & below);
#pragma unroll
      for (int q = 0; q < EV_NW; ++q) {
        eq_before += q < w ? wsum[q] : 0;
        gt_before += q < w ? wsum2[q] : 0;
        run_eq += wsum[q];
        run += wsum2[q];
      }
      keep(i, gt, eq, gt_before, eq_before);
      __syncthreads();
    }
  }
}

// The keys that stay move up in place: row i takes the place of kept[i] >= i.  Rows move in ascending chunks, all of a head's columns of one pool
// (or a slice of them) by ONE workgroup: a chunk's targets lie below every later chunk's sources, so the next chunk may be on its way while this
// one is stored, and only the rows of one chunk can overwrite each other's sources -- a barrier between its loads' return and its stores rules
// that out.  HBM-bound: two chunks of 32 KB in flight per workgroup.  1024 threads of 2 vectors a chunk: 32 sequences of 4.5k - 9k keys, 8 heads of 128,
// back to 4096, 211 us, and the selection 16 (1.09 GB in all: 4.8 TB/s, the rate of a large copy); with 256 threads of 8 vectors, whose chunk takes as
// many bytes but whose lanes walk it alone, both together, timed by events behind other work, 302 for 268.
constexpr int MV_T = 1024, MV_U = 2, MV_TAB = 4096;

template <bool CACHED, typename V>  // CACHED: the sequence's pages are in LDS
__device__ inline void evict_move(V* pool, const EvictArgs& a, const int32_t* kept, const int32_t* tab, const int32_t (&sh_tab)[MV_TAB], int h, int vpr,
                                  int e0, int width, int len) {
  const int tid = threadIdx.x, ps = 1 << a.psl, n = a.budget;
  const int64_t page_vecs = (int64_t)a.Hkv * ps * vpr;
  const int rows = MV_T / width, row0 = tid / width, e = e0 + tid % width;  // rows a pass, this thread's and its column
  const bool mine = row0 < rows;
  auto page_of = [&](int j) { return CACHED ? sh_tab[j >> a.psl] : tab[j >> a.psl]; };
  auto place = [&](int page, int j) { return pool + (int64_t)page * page_vecs + (int64_t)(h * ps + (j & (ps - 1))) * vpr + e; };
  // No branch around a load (rows past the end read the last one's, vectors that do not move the pool's first), so that the waits for a chunk can
  // leave the next one's loads in flight.
  int from[MV_U];
  auto load_kept = [&](int base) {
#pragma unroll
    for (int u = 0; u < MV_U; ++u) from[u] = kept[min(base + u * rows + row0, n - 1)];
  };
  auto load_rows = [&](int base, V (&x)[MV_U]) -> unsigned {  // bit u: vector u is to be stored
    unsigned moves = 0;
#pragma unroll
    for (int u = 0; u < MV_U; ++u) {
      const int row = base + u * rows + row0;
      const bool go = mine & (row < n) & (from[u] > row) & (from[u] < len);
      const int sp = page_of(go ? from[u] : 0), dp = page_of(go ? row : 0);
      const bool there = go & ((unsigned)sp < (unsigned)a.n_pages) & ((unsigned)dp < (unsigned)a.n_pages);
      x[u] = *(there ? place(sp, from[u]) : pool);
      moves |= there ? 1u << u : 0u;
    }
    return moves;
  };
  const int step = MV_U * rows;
  auto turn = [&](int base, V (&x)[MV_U], unsigned moves, V (&next)[MV_U]) -> unsigned {
    const unsigned m2 = load_rows(base + step, next);
    load_kept(base + 2 * step);
#pragma unroll
    for (int u = 0; u < MV_U; ++u) asm volatile("" : "+v"(x[u])::"memory");  // the chunk's loads have returned to this wave
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MV_U; ++u)
      if (moves >> u & 1) {
        const int row = base + u * rows + row0;
        *place(page_of(row), row) = x[u];
      }
    return m2;
  };
  V x[MV_U], y[MV_U];
  load_kept(0);
  unsigned mx = load_rows(0, x), my;
  load_kept(step);
  for (int base = 0; base < n; base += 2 * step) {
    my = turn(base, x, mx, y);
    mx = turn(base + step, y, my, x);  // past the end: nothing moves
  }
}

// blockIdx.z: the weights, then 2 * slices parts of the keys and values
__global__ __launch_bounds__(MV_T) void kv_evict_move_kernel(EvictArgs a, int vpr, int slices) {
  __shared__ int32_t sh_tab[MV_TAB];
  const int h = blockIdx.x, b = blockIdx.y, what = (int)blockIdx.z - 1;
  const EvictRow r = evict_row(a, b);
  if (r.n <= a.budget) return;
  const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
  const int32_t* tab = a.table + (int64_t)b * a.W;
  const int used = (r.n + (1 << a.psl) - 1) >> a.psl;  // pages of the sequence
  const int width = what < 0 ? 1 : vpr / slices, e0 = what < 0 ? 0 : (what % slices) * width;
  pc_u32x4* const pool = (pc_u32x4*)(what < slices ? a.k_pages : a.v_pages);
  if (used <= MV_TAB) {
    for (int i = threadIdx.x; i < used; i += MV_T) sh_tab[i] = tab[i];
    __syncthreads();
    if (what < 0) evict_move<true>(a.mass, a, kept, tab, sh_tab, h, 1, e0, width, r.n);
    else evict_move<true>(pool, a, kept, tab, sh_tab, h, vpr, e0, width, r.n);
  } else {
    if (what < 0) evict_move<false>(a.mass, a, kept, tab, sh_tab, h, 1, e0, width, r.n);
    else evict_move<false>(pool, a, kept, tab, sh_tab, h, vpr, e0, width, r.n);
  }
}

int launch_kv_evict(hipStream_t st, int dtype, const EvictArgs& a, int B, int dh) {
  if (B <= 0) return 0;
  const int64_t most = (int64_t)a.W << a.psl;
  const dim3 sgrid(a.Hkv, B);
  // candidates in registers where the table is short enough (4 sequences of 900 - 1500 keys, selection and move: 28 us, read again in every pass 30;
  // 32 of 4.5k - 9k: 267 / 279)
  if (most <= 4 * EV_T) hipLaunchKernelGGL((kv_evict_select_kernel<4>), sgrid, dim3(EV_T), 0, st, a);
  else if (most <= 16 * EV_T) hipLaunchKernelGGL((kv_evict_select_kernel<16>), sgrid, dim3(EV_T), 0, st, a);
  else hipLaunchKernelGGL((kv_evict_select_kernel<0>), sgrid, dim3(EV_T), 0, st, a);
  const int vpr = dh * (dtype == DT_F32 ? 4 : 2) / 16;
  // Slices of whole 128-byte lines.  (Half lines: 32 sequences, 8 heads of 128, 267 -> 370 us; 4 sequences, 16 heads of 64, where that doubles the 128
  // workgroups, 28 us both.)
  const int slices = vpr % 8 == 0 ? vpr / 8 : 1;
  hipLaunchKernelGGL(kv_evict_move_kernel, dim3(a.Hkv, B, 2 * slices + 1), dim3(MV_T), 0, st, a, vpr, slices);
  return 0;
}

}  // namespace vle
