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

constexpr int PC_TILE = 32;  // keys of one wave step: two 16-key score tiles feed one K = 32 MFMA of the weights

// The keys the newest token of a sequence sees: j < n and (j < hd or j >= lo), as tiles of 32 keys.  Tiles 0 .. th - 1 cover the head,
// tile t >= th starts at key (mf + t - th) * 32; tiles between the head and the window are never touched.
struct Span {
  int n, hd, lo, th, mf, tt;
  __device__ int key0(int t) const { return (t < th ? t : mf + (t - th)) * PC_TILE; }
  __device__ bool sees(int j) const { return j < n && (j < hd || j >= lo); }
};

__device__ inline Span span_of(int n, int text, int window, int sinks) {
  Span s;
  s.n = n;
  if (window <= 0 || window >= n) {
    s.hd = s.lo = n;
  } else {
    s.hd = min(n, max(text, sinks));
    s.lo = n - window;
  }
  s.th = (s.hd + PC_TILE - 1) / PC_TILE;
  s.mf = max(s.th, s.lo / PC_TILE);
  s.tt = s.th + max(0, (n + PC_TILE - 1) / PC_TILE - s.mf);
  return s;
}

__device__ inline Span span_of_row(const PagedDecodeArgs& a, int b) {
  const int n = min(max(a.lengths[b], 0), a.W << a.psl);  // W * ps < 2^31 (checked by the launcher)
  return span_of(n, a.text_len ? a.text_len[b] : 0, a.window, a.sinks);
}

}  // namespace

// ---- writing ---------------------------------------------------------------------------------------------------------------------
// One wave per new token and per half (K, V): Hkv * dh elements in 16-byte vectors, contiguous reads, one dh-segment per head out.  HBM-bound copy.
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
    if (b >= a.B || row < a.seq_off[b]) return;  // behind the last sequence or ahead of the first
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
template <int N>
__device__ inline void pd_load_words(unsigned (&dst)[N], const void* src) {  // N = 2, 4 or 8 words of 32 bits, from 8 or 16 aligned bytes on
  if constexpr (N == 2) {
    const pc_u32x2 x = *reinterpret_cast<const pc_u32x2*>(src);
    dst[0] = x[0];
    dst[1] = x[1];
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const pc_u32x4 x = reinterpret_cast<const pc_u32x4*>(src)[i];
#pragma unroll
      for (int j = 0; j < 4; ++j) dst[4 * i + j] = x[j];
    }
  }
}

template <int KV, int VW>
struct PdTile {  // 32 keys: K fragments of both 16-key tiles, and this lane's VW words of each of its 8 V rows
  pc_u32x4 k[2][KV];
  unsigned v[8][VW];
};

template <typename T, int DHT, int NW, bool MASS>
__global__ __launch_bounds__(NW * 64) void paged_decode_kernel(PagedDecodeArgs a) {
  constexpr bool BF = sizeof(T) == 2;
  constexpr int DPL = DHT / 16;           // head elements per lane of a V row
  constexpr int KV = BF ? DHT / 32 : DHT / 16;  // 16-byte K vectors per lane and 16-key tile
  constexpr int KE = BF ? 8 : 4;          // elements per such vector
  constexpr int VW = DPL * (int)sizeof(T) / 4;  // 32-bit words per lane of a V row
  using Tile = PdTile<KV, VW>;
  extern __shared__ float sm[];  // [NW][ng][DHT] partial outputs, then [NW][16][2] (m, l)

  const int split = blockIdx.x, b = blockIdx.z;
  const int kvh = (int)blockIdx.y / a.GT, gt = (int)blockIdx.y - kvh * a.GT;
  const int h0 = kvh * a.G + gt * 16, ng = min(16, a.G - gt * 16);
  const Span sp = span_of_row(a, b);
  const int t0 = split * a.chunk, t1 = min(t0 + a.chunk, sp.tt);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, g = lane >> 4, c = lane & 15;
  const int H = a.Hkv * a.G, ps = 1 << a.psl, dh = a.dh;
  if (split > 0 && t0 >= sp.tt) return;  // nothing of this sequence is left for this split, and the join does not read it

  pc_u32x4 qf[KV];
  {
    const T* qp = (const T*)a.q + (int64_t)b * a.q_b + (int64_t)(h0 + min(c, ng - 1)) * a.q_h;
#pragma unroll
    for (int i = 0; i < KV; ++i) {
      const int e = i * 4 * KE + g * KE;
      const bool in = c < ng && e < dh;
      qf[i] = pc_u32x4{0u, 0u, 0u, 0u};
      if (in) qf[i] = *reinterpret_cast<const pc_u32x4*>(qp + e);
    }
  }

  const int32_t* tab = a.table + (int64_t)b * a.W;
  const int64_t page_elems = (int64_t)a.Hkv * ps * dh;
  const T* kbase = (const T*)a.k_pages + (int64_t)kvh * ps * dh;
  const T* vbase = (const T*)a.v_pages + (int64_t)kvh * ps * dh;
  const bool vin = c * DPL < dh;  // dh is a multiple of 8 and DPL of 4: a lane's dims are inside the head or outside it (DPL 8: dh % 8 == 0)

  float m = -INFINITY, l = -0.0f;  // l stays -0 until a visible key was met: a row that sees nothing answers 0, not 0 / 0
  pc_f32x4 o[DPL];
#pragma unroll
  for (int j = 0; j < DPL; ++j) o[j] = pc_f32x4{0.f, 0.f, 0.f, 0.f};

  // page ids: lane i (0 .. 31) holds the page of key key0 + i of one tile, fetched a tile ahead of the keys
  auto load_ids = [&](int t) -> int {
    int id = -1;
    if (t < t1) {
      const int j = sp.key0(t) + (lane & 31);
      if (j < sp.n) id = tab[j >> a.psl];
    }
    return (unsigned)id < (unsigned)a.n_pages ? id : -1;
  };
  auto load_tile = [&](Tile& tl, int t, int ids) {
    const int k0 = sp.key0(t);
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int key = k0 + 16 * st + c;
      const int id = __shfl(ids, 16 * st + c, 64);
      const T* p = kbase + (int64_t)max(id, 0) * page_elems + (key & (ps - 1)) * dh;
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        const int e = i * 4 * KE + g * KE;
        tl.k[st][i] = pc_u32x4{0u, 0u, 0u, 0u};
        if (id >= 0 && e < dh) tl.k[st][i] = *reinterpret_cast<const pc_u32x4*>(p + e);
      }
    }
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      const int key = k0 + 16 * st + 4 * g;  // four keys of one page (ps >= 8)
      const int id = __shfl(ids, 16 * st + 4 * g, 64);
      const T* p = vbase + (int64_t)max(id, 0) * page_elems + (key & (ps - 1)) * dh + c * DPL;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma unroll
        for (int i = 0; i < VW; ++i) tl.v[4 * st + r][i] = 0;
        if (id >= 0 && vin && sp.sees(key + r)) pd_load_words(tl.v[4 * st + r], p + r * dh);  // what nobody sees may hold anything, NaN included
      }
    }
  };

  int ids = load_ids(t0 + w);
  for (int t = t0 + w; t < t1; t += NW) {
    Tile tl;
    load_tile(tl, t, ids);
    const int ids_next = load_ids(t + NW);
    const int k0 = sp.key0(t);
    const int page_a = __shfl(ids, 4 * g, 64), page_b = __shfl(ids, 16 + 4 * g, 64);
    ids = ids_next;
    // ---- scores, in units of the exp2 argument ----
    pc_f32x4 s[2];
    bool any = false;
#pragma unroll
    for (int st = 0; st < 2; ++st) {
      s[st] = pc_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < KV; ++i) {
        if constexpr (BF) {
          s[st] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pc_bf16x8, tl.k[st][i]), __builtin_bit_cast(pc_bf16x8, qf[i]), s[st], 0, 0, 0);
        } else {
#pragma unroll
          for (int u = 0; u < 4; ++u) s[st] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tl.k[st][i][u]), __uint_as_float(qf[i][u]), s[st], 0, 0, 0);
        }
      }
      const bool there = (st ? page_b : page_a) >= 0;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
#pragma clang fp contract(off)  // the rounded product: its difference to the maximum must be 0 for the largest, whatever its size
        const bool vis = there && sp.sees(k0 + 16 * st + 4 * g + r);
        any |= vis;
        s[st][r] = vis ? s[st][r] * a.sl2 : -INFINITY;
      }
    }
    if constexpr (MASS) {
      if (c < ng) {
        float* sc = a.scores + ((int64_t)b * H + h0 + c) * a.score_ld + (int64_t)t * PC_TILE + 4 * g;
        *reinterpret_cast<pc_f32x4*>(sc) = s[0];
        *reinterpret_cast<pc_f32x4*>(sc + 16) = s[1];
      }
    }
    if (!__any(any)) continue;
    // ---- online softmax of column c ----
    float mt = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
    mt = rows4_max(mt);
    const float mn = fmaxf(m, mt);
    const float ref = mn == -INFINITY ? 0.f : mn;  // every score so far is -inf: their weights are 0, not exp(-inf + inf)
    const float alpha = __builtin_amdgcn_exp2f(m - ref);
    m = mn;
    float p[8], sum = 0.f;
#pragma unroll
    for (int st = 0; st < 2; ++st)
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
        for (int i = 0; i < 4; ++i)
          f[i] = __builtin_amdgcn_perm(tl.v[2 * i + 1][j >> 1], tl.v[2 * i][j >> 1], (j & 1) ? 0x07060302u : 0x05040100u);
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pc_bf16x8, f), hi, o[j], 0, 0, 0);
        o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(pc_bf16x8, f), lo, o[j], 0, 0, 0);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < DPL; ++j) o[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(tl.v[i][j]), p[i], o[j], 0, 0, 0);
    }
  }

  // ---- the waves' parts meet in LDS ----
  l = rows4_sum(l);
  float* sm_ml = sm + NW * ng * DHT;
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
  for (int idx = tid; idx < ng * DHT; idx += NW * 64) {
    const int hh = idx / DHT, e = idx - hh * DHT;
    if (e >= dh) continue;
    float M = -INFINITY;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, sm_ml[(i * 16 + hh) * 2]);
    const float ref = M == -INFINITY ? 0.f : M;
    float L = -0.0f, O = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) {
      const float f = __builtin_amdgcn_exp2f(sm_ml[(i * 16 + hh) * 2] - ref);
      L += sm_ml[(i * 16 + hh) * 2 + 1] * f;
      O += sm[(i * ng + hh) * DHT + e] * f;
    }
    if (a.nsplit == 1) store_elem<T>((T*)a.out + ((int64_t)b * H + h0 + hh) * dh + e, __float_as_uint(L) == 0x80000000u ? 0.f : O / L);
    else a.part_o[(((int64_t)b * H + h0 + hh) * a.nsplit + split) * dh + e] = O;
    if (e == 0 && a.part_ml != nullptr) {
      float* ml = a.part_ml + (((int64_t)b * H + h0 + hh) * a.nsplit + split) * 2;
      ml[0] = M;
      ml[1] = L;
    }
  }
}

// Joins the splits (blockIdx.x == 0, when there are several) and adds every visible key's weight to `mass` (blockIdx.x >= 1, 1024 keys each).
constexpr int PD_JOIN_KEYS = 1024, PD_MAX_GROUP = 256;

template <typename T>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(PagedDecodeArgs a) {
  __shared__ float sh_m[PD_MAX_GROUP], sh_i[PD_MAX_GROUP];
  const int b = blockIdx.z, kvh = blockIdx.y, tid = threadIdx.x;
  const int H = a.Hkv * a.G, ps = 1 << a.psl;
  const Span sp = span_of_row(a, b);
  const int used = max(1, (sp.tt + a.chunk - 1) / a.chunk);
  const int part = (int)blockIdx.x - (a.nsplit > 1 ? 1 : 0);  // -1: the outputs
  if (part >= 0 && part * PD_JOIN_KEYS >= sp.tt * PC_TILE) return;
  for (int h = tid; h < a.G; h += 256) {  // the statistics of the group's heads over all splits
    const float* ml = a.part_ml + ((int64_t)b * H + kvh * a.G + h) * a.nsplit * 2;
    float M = -INFINITY, L = -0.0f;
    for (int s = 0; s < used; ++s) M = fmaxf(M, ml[2 * s]);
    const float ref = M == -INFINITY ? 0.f : M;
    for (int s = 0; s < used; ++s) L += ml[2 * s + 1] * __builtin_amdgcn_exp2f(ml[2 * s] - ref);
    sh_m[h] = ref;
    sh_i[h] = __float_as_uint(L) == 0x80000000u ? 0.f : 1.0f / L;
  }
  __syncthreads();
  if (part < 0) {
    for (int idx = tid; idx < a.G * a.dh; idx += 256) {
      const int h = idx / a.dh, e = idx - h * a.dh;
      const int64_t hb = (int64_t)b * H + kvh * a.G + h;
      float O = 0.f;
      for (int s = 0; s < used; ++s) O += a.part_o[(hb * a.nsplit + s) * a.dh + e] * __builtin_amdgcn_exp2f(a.part_ml[(hb * a.nsplit + s) * 2] - sh_m[h]);
      store_elem<T>((T*)a.out + hb * a.dh + e, O * sh_i[h]);
    }
    return;
  }
  for (int idx = part * PD_JOIN_KEYS + tid; idx < min((part + 1) * PD_JOIN_KEYS, sp.tt * PC_TILE); idx += 256) {
    const int j = sp.key0(idx / PC_TILE) + idx % PC_TILE;
    if (!sp.sees(j)) continue;
    const int page = a.table[(int64_t)b * a.W + (j >> a.psl)];
    if ((unsigned)page >= (unsigned)a.n_pages) continue;
    const float* sc = a.scores + ((int64_t)b * H + kvh * a.G) * a.score_ld + idx;
    float sum = 0.f;
    for (int h = 0; h < a.G; ++h) sum += __builtin_amdgcn_exp2f(sc[h * a.score_ld] - sh_m[h]) * sh_i[h];
    // an atomic, because sequences may share the pages of a common prefix; without sharing there is one addend and one result
    unsafeAtomicAdd(a.mass + ((int64_t)page * a.Hkv + kvh) * ps + (j & (ps - 1)), sum);
  }
}

static int pd_tiles_bound(int W, int ps, int window, int sinks, bool text) {  // tiles of a sequence, at most
  const int64_t n = (int64_t)W * ps;
  const int full = (int)((n + PC_TILE - 1) / PC_TILE);
  if (window <= 0 || window >= n || text) return full;
  return (int)std::min((int64_t)full, ((int64_t)sinks + PC_TILE - 1) / PC_TILE + ((int64_t)window + PC_TILE - 1) / PC_TILE + 1);
}

PagedDecodePlan paged_decode_plan(int B, int Hkv, int G, int dh, int W, int ps, int window, int sinks, bool text, bool mass) {
  PagedDecodePlan p;
  const int tiles = std::max(1, pd_tiles_bound(W, ps, window, sinks, text));
  const int64_t groups = (int64_t)B * Hkv * ((G + 15) / 16);
  p.tiles = tiles;
  p.nw = 4;
  p.chunk = tiles;
  p.nsplit = 1;
  if (groups < 512 && tiles > 16) {
    p.chunk = (int)std::max((int64_t)16, (tiles * groups + 1023) / 1024);
    p.nsplit = (tiles + p.chunk - 1) / p.chunk;
  }
  const int64_t H = (int64_t)Hkv * G;
  p.ml_floats = (p.nsplit > 1 || mass) ? (size_t)(B * H * p.nsplit * 2) : 0;
  p.o_floats = p.nsplit > 1 ? (size_t)(B * H * p.nsplit * dh) : 0;
  p.score_floats = mass ? (size_t)(B * H) * tiles * PC_TILE : 0;
  return p;
}

template <typename T, int DHT>
static int pd_launch(hipStream_t st, const PagedDecodePlan& p, const PagedDecodeArgs& a, int B) {
  const int ng = std::min(16, a.G);
  const size_t lds = ((size_t)p.nw * ng * DHT + p.nw * 32) * sizeof(float);
  const dim3 grid(p.nsplit, a.Hkv * a.GT, B), block(p.nw * 64);
  if (a.mass != nullptr) hipLaunchKernelGGL((paged_decode_kernel<T, DHT, 4, true>), grid, block, lds, st, a);
  else hipLaunchKernelGGL((paged_decode_kernel<T, DHT, 4, false>), grid, block, lds, st, a);
  const int parts = (p.nsplit > 1 ? 1 : 0) + (a.mass != nullptr ? (p.tiles * PC_TILE + PD_JOIN_KEYS - 1) / PD_JOIN_KEYS : 0);
  if (parts > 0) hipLaunchKernelGGL((paged_decode_join_kernel<T>), dim3(parts, a.Hkv, B), dim3(256), 0, st, a);
  return 0;
}

int launch_paged_decode(hipStream_t st, int dtype, const PagedDecodePlan& p, PagedDecodeArgs a, int B) {
  if (B <= 0) return 0;
  if (a.G > PD_MAX_GROUP) return -1;
  a.GT = (a.G + 15) / 16;
  a.chunk = p.chunk;
  a.nsplit = p.nsplit;
  a.score_ld = (int64_t)p.tiles * PC_TILE;
  if (dtype == DT_F32) return a.dh <= 64 ? pd_launch<float, 64>(st, p, a, B) : pd_launch<float, 128>(st, p, a, B);
  return a.dh <= 64 ? pd_launch<bf16_t, 64>(st, p, a, B) : pd_launch<bf16_t, 128>(st, p, a, B);
}

// ---- eviction ----------------------------------------------------------------------------------------------------------------------
// Which keys stay: the first S and the last R of n, and of the n - S - R between them the M = budget - S - R with the most weight (of equal
// weights the earlier).  One workgroup per (sequence, head) finds the M-th largest weight by three counting passes over its order-preserving
// 32-bit key (11 + 11 + 10 bits, 2048 counters in LDS), then numbers the keys that stay in one more pass in the order of their positions.
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

__global__ __launch_bounds__(EV_T) void kv_evict_select_kernel(EvictArgs a) {
  __shared__ int bins[EV_BINS];
  __shared__ int wsum[EV_NW], wsum2[EV_NW];
  __shared__ int sh_bin, sh_above;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 63, w = tid >> 6, ps = 1 << a.psl;
  const EvictRow r = evict_row(a, b);
  int32_t* kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
  if (h == 0 && tid == 0) a.new_lengths[b] = min(r.n, a.budget);
  if (r.n <= a.budget) {
    for (int i = tid; i < a.budget; i += EV_T) kept[i] = i < r.n ? i : -1;
    return;
  }
  for (int i = tid; i < r.S; i += EV_T) kept[i] = i;
  for (int i = tid; i < r.R; i += EV_T) kept[r.S + r.M + i] = r.n - r.R + i;
  if (r.M == 0) return;
  const int C = r.n - r.S - r.R;  // > M >= 1
  const int32_t* tab = a.table + (int64_t)b * a.W;
  auto weight = [&](int i) -> uint32_t {  // key of candidate i; the keys of a page that is not there have no weight
    const int j = r.S + i, page = tab[j >> a.psl];
    return (unsigned)page < (unsigned)a.n_pages ? ev_key(a.mass[((int64_t)page * a.Hkv + h) * ps + (j & (ps - 1))]) : ev_key(0.f);
  };
  uint32_t prefix = 0, have = 0;  // the bits of the M-th largest key that are known, and their mask
  int need = r.M;                 // its rank among the keys that agree with them
#pragma unroll 1
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, nb = pass == 2 ? 1024 : 2048;
    for (int i = tid; i < EV_BINS; i += EV_T) bins[i] = 0;
    __syncthreads();
    for (int i = tid; i < C; i += EV_T) {
      const uint32_t k = weight(i);
      if ((k & have) == prefix) atomicAdd(&bins[(k >> shift) & (nb - 1)], 1);
    }
    __syncthreads();
    // thread t counts bins 2047 - 2 t and 2046 - 2 t: an inclusive scan from the top finds the bin the need-th largest falls into
    const int hi = bins[EV_BINS - 1 - 2 * tid], lo = bins[EV_BINS - 2 - 2 * tid];
    int inc = hi + lo;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int t = __shfl_up(inc, o, 64);
      if (lane >= o) inc += t;
    }
    if (lane == 63) wsum[w] = inc;
    __syncthreads();
    int before = inc - hi - lo;
    for (int i = 0; i < w; ++i) before += wsum[i];
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
    __syncthreads();
  }
  // every key above `prefix` stays, and of those equal to it the first `need`
  int run = 0, run_eq = 0;
  for (int i0 = 0; i0 < C; i0 += EV_T) {
    const int i = i0 + tid;
    const uint32_t k = i < C ? weight(i) : 0u;
    const bool eq = i < C && k == prefix, gt = i < C && k > prefix;
    const unsigned long long beq = __ballot(eq), bgt = __ballot(gt), below = (1ull << lane) - 1;
    if (lane == 0) {
      wsum[w] = __popcll(beq);
      wsum2[w] = __popcll(bgt);
    }
    __syncthreads();
    int eq_before = run_eq + __popcll(beq & below), gt_before = run + __popcll(bgt & below), eq_all = 0, gt_all = 0;
#pragma unroll
    for (int q = 0; q < EV_NW; ++q) {
      eq_before += q < w ? wsum[q] : 0;
      gt_before += q < w ? wsum2[q] : 0;
      eq_all += wsum[q];
      gt_all += wsum2[q];
    }
    const int at = gt_before + min(eq_before, need);
    if ((gt || (eq && eq_before < need)) && at < r.M) kept[r.S + at] = r.S + i;  // at < M always, unless the weights change during the call
    run += gt_all;
    run_eq += eq_all;
    __syncthreads();
  }
}

// The keys that stay move up in place: row i takes the place of kept[i] >= i.  Rows are moved in ascending chunks by ONE workgroup per (sequence,
// head, K | V | weights): a chunk's targets lie below every later chunk's sources, so only the rows of one chunk can overwrite each other's
// sources, and a barrier between a chunk's loads and its stores rules that out.
constexpr int MV_T = 256, MV_U = 8;

template <typename V>
__device__ inline void evict_move(V* pool, const EvictArgs& a, const int32_t* kept, const int32_t* tab, int h, int vpr, int n, int len) {
  const int tid = threadIdx.x, ps = 1 << a.psl;
  const int64_t page_vecs = (int64_t)a.Hkv * ps * vpr;
  const int total = n * vpr;  // vectors
  for (int i0 = 0; i0 < total; i0 += MV_T * MV_U) {
    V x[MV_U];
    V* dst[MV_U];
#pragma unroll
    for (int u = 0; u < MV_U; ++u) {
      const int i = i0 + u * MV_T + tid;
      dst[u] = nullptr;
      if (i < total) {
        const int row = i / vpr, e = i - row * vpr, from = kept[row];
        if (from != row && (unsigned)from < (unsigned)len) {
          const int sp = tab[from >> a.psl], dp = tab[row >> a.psl];
          if ((unsigned)sp < (unsigned)a.n_pages && (unsigned)dp < (unsigned)a.n_pages) {
            x[u] = pool[(int64_t)sp * page_vecs + (int64_t)(h * ps + (from & (ps - 1))) * vpr + e];
            dst[u] = pool + (int64_t)dp * page_vecs + (int64_t)(h * ps + (row & (ps - 1))) * vpr + e;
          }
        }
      }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // this wave's loads of the chunk have returned
    __syncthreads();
#pragma unroll
    for (int u = 0; u < MV_U; ++u)
      if (dst[u] != nullptr) *dst[u] = x[u];
  }
}

__global__ __launch_bounds__(MV_T) void kv_evict_move_kernel(EvictArgs a, int vpr) {
  const int h = blockIdx.x, b = blockIdx.y, what = blockIdx.z;
  const EvictRow r = evict_row(a, b);
  if (r.n <= a.budget) return;
  const int32_t* kept = a.kept + ((int64_t)b * a.Hkv + h) * a.budget;
  const int32_t* tab = a.table + (int64_t)b * a.W;
  if (what == 2) evict_move<float>(a.mass, a, kept, tab, h, 1, a.budget, r.n);
  else evict_move<pc_u32x4>((pc_u32x4*)(what ? a.v_pages : a.k_pages), a, kept, tab, h, vpr, a.budget, r.n);
}

int launch_kv_evict(hipStream_t st, int dtype, const EvictArgs& a, int B, int dh) {
  if (B <= 0) return 0;
  hipLaunchKernelGGL(kv_evict_select_kernel, dim3(a.Hkv, B), dim3(EV_T), 0, st, a);
  hipLaunchKernelGGL(kv_evict_move_kernel, dim3(a.Hkv, B, 3), dim3(MV_T), 0, st, a, dh * (dtype == DT_F32 ? 4 : 2) / 16);
  return 0;
}

}  // namespace vle
