// Attention weights of the last S_q rows of a prompt, summed per key:
//   sums[b][g][j] = sum over the heads h of kv head g and the rows i of
//                   softmax_i(q_bhi . k_bg * scale)[j],
// row i at position S_k - S_q + i, keys up to its own position.  What a cache is
// cut by after a prefill.
//
// A weight needs its row's maximum and sum over all keys, a column sum needs
// the weights of all rows, so q.k is taken twice:
//   stats: a wave holds up to 64 rows of a head as the B operand and walks the
//     keys: S^T = K . Q^T, lane (lc, lr) gets row lc, keys 4 lr + i.  Each lane
//     keeps a running (m, l) of the keys it sees: no exchange until the end.
//   columns: a wave holds 64 keys of a kv head as the B operand and walks the
//     rows of all its heads: S = Q . K^T, lane (lc, lr) gets key lc, rows 4 lr +
//     i.  Each lane sums its keys' weights in registers.
// The walked rows go through LDS, 64 a tile, for the four waves of a workgroup
// (256 rows or keys); a stats item of fewer rows (see sums_plan) has its waves take
// different keys, and a window of rows with a kv head a head does its columns the
// same way (sums_window_kernel).
// Bound by the exponentials, two for each visible pair (a quarter-rate
// instruction), with a fused multiply-add and an add beside each, and the products,
// which hardly overlap with them: 16 heads (4 kv) x 16384 rows of 128 dims 1024 us,
// stats 574 and columns 551 by themselves, 1.07 PFLOP/s of both score products.  A
// window is bound by the keys, read twice: 32 heads x 64 rows of 131072 keys of 96
// dims 119 + 138 us, 6.3 TB/s.
// Sums are fp32 in two levels, in a fixed order.

#include <type_traits>

#include "msa_common.h"
#include "msa_kernels.h"
#include "msa_tile.h"

namespace msa {

#define INLINE __attribute__((always_inline))

namespace {

constexpr int kTileRows = 64;  // walked rows (keys) of a tile in LDS

template <int D>
struct SumsShape {
  static constexpr int NKS = D / 32;
  static constexpr int TILES = D <= 128 ? 4 : D == 256 ? 2 : 1;  // 16-row tiles a wave holds
  using Part = Tile<D, 16>;                                      // a wave's share of a tile
  static constexpr int STAGE = 4 * Part::BYTES;
};

// Descriptor of up to `rows` rows from `p` on, `left` of which exist: loads of
// the others return 0.
__device__ inline __amdgpu_buffer_rsrc_t rows_rsrc(const uint16_t* p, int left, int rows,
                                                   uint32_t stride, int D) {
  const uint32_t n = left > 0 ? uint32_t(min(left, rows) - 1) * stride + 2 * D : 0u;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), short(0), int(n), 0x00020000);
}

// A wave's walked keys, not kept in the caches where the call streams them.
template <typename Part>
__device__ INLINE inline void load_keys(const SumsParams& P, const Part& part, __amdgpu_buffer_rsrc_t rs,
                                        u32x4 (&x)[Part::NL]) {
  if (P.stream)
    part.template load<2>(rs, 0, x);
  else
    part.template load<0>(rs, 0, x);
}

// Operands of the 16 MT rows from `p` on (`left` exist, the others are 0),
// through this wave's 16 rows of LDS.
template <int D, int MT>
__device__ inline void hold_rows(const uint16_t* p, int left, int64_t stride, int lane,
                                 unsigned char* lds, u32x4 (&x)[MT][D / 32]) {
  using Part = Tile<D, 16>;
  const Part part(lane, uint32_t(stride) * 2u);
  u32x4 r[MT][Part::NL];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt)
    part.load_at(rows_rsrc(p + 16 * mt * stride, left - 16 * mt, 16, uint32_t(stride) * 2u, D), 0, r[mt]);
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    part.store(lds, r[mt]);
    wave_lds_fence();
#pragma unroll
    for (int ks = 0; ks < D / 32; ++ks)
      x[mt][ks] = Part::operand(lds, 0, lane & 15, lane >> 4, ks);
    wave_lds_fence();
  }
}

// SHARE: four waves of 16 MT rows each against the same keys; otherwise one set
// of rows, the waves on different keys.
template <typename T, int D, int MT, bool SHARE>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 256 ? 1 : SHARE && D <= 128 ? 3 : 2)))
void sums_stats_kernel(const SumsParams P) {
  using Shape = SumsShape<D>;
  using Part = typename Shape::Part;
  constexpr int NKS = Shape::NKS;
  __shared__ __align__(16) unsigned char lds[2 * Shape::STAGE];
  __shared__ float sm[4][16 * MT], sl[4][16 * MT];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane >> 4, lc = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // longest items (last rows) first
  int x = blockIdx.x;
  const int bh = x % (P.batch * P.heads);
  x /= P.batch * P.heads;
  const int split = x % P.n_split;
  const int rt = P.n_rt - 1 - x / P.n_split;
  const int b = bh / P.heads, h = bh - b * P.heads;
  const int wg_row0 = rt * 16 * MT * (SHARE ? 4 : 1);
  const int row0 = wg_row0 + (SHARE ? 16 * MT * w : 0);  // of this wave
  const int wg_rows = min(16 * MT * (SHARE ? 4 : 1), P.s_q - wg_row0);
  const int shift = P.s_k - P.s_q;
  const int j_begin = split * P.chunk;
  const int j_end = min(min(j_begin + P.chunk, P.s_k), shift + wg_row0 + wg_rows);
  const int n_tiles = j_end > j_begin ? (j_end - j_begin + kTileRows - 1) / kTileRows : 0;

  u32x4 qb[MT][NKS];
  hold_rows<D, MT>(reinterpret_cast<const uint16_t*>(P.q) + b * P.q_sb + int64_t(h) * P.q_sh +
                       int64_t(min(row0, P.s_q - 1)) * P.q_ss,
                   P.s_q - row0, P.q_ss, lane, lds + w * Part::BYTES, qb);

  const uint16_t* kbase = reinterpret_cast<const uint16_t*>(P.k) + b * P.k_sb +
                          int64_t(h / P.group) * P.k_sh;
  const uint32_t kss = uint32_t(P.k_ss) * 2u;
  const Part part(lane, kss);

  // of the keys this lane sees: what the exponentials are taken against (a
  // score of the row, at most 2^64 below the largest), and the sum in two
  // levels (small terms are not lost in a long sum)
  float mp[MT], l[MT], acc[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    mp[mt] = -__builtin_inff();
    l[mt] = acc[mt] = 0.0f;
  }
  const float c = P.scale_log2;
  auto scores = [&](const unsigned char* lp, f32x4 (&s)[MT][2]) INLINE {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = Part::operand(lp + u * Part::BYTES, 0, lc, lr, ks);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][u] = mfma_qk<T>(a, qb[mt][ks], s[mt][u]);
      }
    }
  };
  auto edge = [&](int j0) INLINE { return j0 + 31 > shift + row0 || j0 + 32 > j_end; };
  bool started = false;  // every lane has a reference
  // Hides what a row does not see, and starts the reference of a lane that has
  // none yet.
  auto prepare = [&](int j0, f32x4 (&s)[MT][2]) INLINE {
    if (edge(j0)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        const int last = min(shift + row0 + 16 * mt + lc, j_end - 1);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + 16 * u + 4 * lr + i > last) s[mt][u][i] = -__builtin_inff();
      }
    }
    bool none = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) none |= mp[mt] == -__builtin_inff();
    started = __ballot(none) == 0;
    if (!started) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (mp[mt] == -__builtin_inff()) mp[mt] = max8(s[mt][0], s[mt][1]) * c;
    }
  };
  auto weigh = [&](const f32x4 (&s)[2], float ref) INLINE {
    float e[8];
    const float z = ref == -__builtin_inff() ? 0.0f : ref;
#pragma unroll
    for (int j = 0; j < 8; ++j)
      e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], c, -z));
    return ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
  };
  // The sums of a block, taken again against a new reference where they ran
  // past 2^64 (the old sum moves to it).
  auto add = [&](const f32x4 (&s)[MT][2], float (&t)[MT]) INLINE {
    bool over = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) over |= t[mt] > 0x1p64f;
    if (__ballot(over) != 0) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        if (t[mt] > 0x1p64f) {
          const float mn = fmaxf(mp[mt], max8(s[mt][0], s[mt][1]) * c);
          const float al = __builtin_amdgcn_exp2f(mp[mt] - mn);
          l[mt] *= al;
          acc[mt] *= al;
          mp[mt] = mn;
          t[mt] = weigh(s[mt], mn);
        }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) acc[mt] += t[mt];
  };
  auto flush = [&]() INLINE {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      l[mt] += acc[mt];
      acc[mt] = 0.0f;
    }
  };

  u32x4 kr[Part::NL];
  auto key_rsrc = [&](int j0, int rows) INLINE {
    return rows_rsrc(kbase + int64_t(min(j0, P.s_k - 1)) * P.k_ss, P.s_k - j0, rows, kss, D);
  };
  auto block = [&](int j0, const unsigned char* lp) INLINE {
    f32x4 s[MT][2];
    float t[MT];
    scores(lp, s);
    if (!started || edge(j0)) prepare(j0, s);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) t[mt] = weigh(s[mt], mp[mt]);
    add(s, t);
  };
  if constexpr (SHARE) {
    // tile t in stage t & 1, the next one on its way through registers
    const bool active = row0 < P.s_q;
    auto load = [&](int tile) INLINE {
      part.load_at(key_rsrc(j_begin + kTileRows * tile + 16 * w, 16), 0, kr);
    };
    if (n_tiles > 0) {
      load(0);
      __syncthreads();  // the held rows have left LDS
      part.store(lds + w * Part::BYTES, kr);
      load(1);
      __syncthreads();
    }
    for (int tile = 0; tile < n_tiles; ++tile) {
      const unsigned char* cur = lds + (tile & 1) * Shape::STAGE;
      unsigned char* nxt = lds + ((tile + 1) & 1) * Shape::STAGE;
      const int j0 = j_begin + kTileRows * tile;
      if (active)
        for (int half = 0; half < 2; ++half)
          block(j0 + 32 * half, cur + 2 * half * Part::BYTES);
      part.store(nxt + w * Part::BYTES, kr);
      load(tile + 2);
      __syncthreads();
      if ((tile & 7) == 7) flush();
    }
  } else {
    // wave w takes 32-key blocks w, w + 4, ... through its own half stage
    unsigned char* mine = lds + w * 2 * Part::BYTES;
    u32x4 kr2[Part::NL];
    auto load = [&](int j0) INLINE {
      load_keys(P, part, key_rsrc(j0, 16), kr);
      load_keys(P, part, key_rsrc(j0 + 16, 16), kr2);
    };
    const int first = j_begin + 32 * w;
    __syncthreads();  // the held rows have left LDS
    load(first);
    for (int j0 = first, i = 0; j0 < j_end; j0 += 128, ++i) {
      part.store(mine, kr);
      part.store(mine + Part::BYTES, kr2);
      wave_lds_fence();
      load(j0 + 128);
      block(j0, mine);
      wave_lds_fence();
      if ((i & 15) == 15) flush();
    }
  }
  flush();

  // merge a row's lanes, then the waves
  float m[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = mp[mt];
#pragma unroll
    for (int off = 16; off <= 32; off <<= 1) {
      const float mo = __shfl_xor(m[mt], off, 64), lo = __shfl_xor(l[mt], off, 64);
      const float mn = fmaxf(m[mt], mo);
      const float z = mn == -__builtin_inff() ? 0.0f : mn;
      l[mt] = l[mt] * __builtin_amdgcn_exp2f(m[mt] - z) + lo * __builtin_amdgcn_exp2f(mo - z);
      m[mt] = mn;
    }
    if (lr == 0) {
      sm[w][16 * mt + lc] = m[mt];
      sl[w][16 * mt + lc] = l[mt];
    }
  }
  __syncthreads();
  constexpr int ROWS = 16 * MT * (SHARE ? 4 : 1);
  if (tid < ROWS) {
    float M, L;
    if constexpr (SHARE) {
      M = sm[tid / (16 * MT)][tid % (16 * MT)];
      L = sl[tid / (16 * MT)][tid % (16 * MT)];
    } else {
      M = -__builtin_inff();
      L = 0.0f;
#pragma unroll
      for (int v = 0; v < 4; ++v) M = fmaxf(M, sm[v][tid]);
#pragma unroll
      for (int v = 0; v < 4; ++v)
        if (sm[v][tid] != -__builtin_inff() || sl[v][tid] != 0.0f)
          L += __builtin_amdgcn_exp2f(sm[v][tid] - M) * sl[v][tid];
    }
    const int64_t row = int64_t(bh) * P.s_q_pad + wg_row0 + tid;
    if (wg_row0 + tid < P.s_q_pad) {
      if (P.n_split > 1) {
        float2* o = reinterpret_cast<float2*>(P.part) + int64_t(split) * P.batch * P.heads * P.s_q_pad;
        o[row] = make_float2(M, L);
      } else {
        P.stat_m[row] = M == -__builtin_inff() ? 0.0f : M;
        P.stat_r[row] = L == 0.0f ? 0.0f : 1.0f / L;
      }
    }
  }
}

// (m, 1 / l) of every row from its key splits: 16 rows a workgroup, 16 threads
// a row.
__global__ __launch_bounds__(256) void sums_merge_kernel(const SumsParams P) {
  const int64_t n = int64_t(P.batch) * P.heads * P.s_q_pad;
  const int64_t row = int64_t(blockIdx.x) * 16 + (threadIdx.x & 15);
  const int g = threadIdx.x >> 4;
  __shared__ float2 red[16][16];
  const float2* part = reinterpret_cast<const float2*>(P.part);
  float M = -__builtin_inff(), L = 0.0f;
  for (int s = g; s < P.n_split; s += 16) {
    const float2 y = part[s * n + row];
    if (y.x == -__builtin_inff()) continue;
    const float mn = fmaxf(M, y.x);
    L = L * __builtin_amdgcn_exp2f(M - mn) + y.y * __builtin_amdgcn_exp2f(y.x - mn);
    M = mn;
  }
  red[g][threadIdx.x & 15] = make_float2(M, L);
  __syncthreads();
  if (g != 0) return;
  for (int v = 0; v < 16; ++v) M = fmaxf(M, red[v][threadIdx.x].x);
  L = 0.0f;
  for (int v = 0; v < 16; ++v) {
    const float2 y = red[v][threadIdx.x];
    if (y.x != -__builtin_inff()) L += __builtin_amdgcn_exp2f(y.x - M) * y.y;
  }
  P.stat_m[row] = M == -__builtin_inff() ? 0.0f : M;
  P.stat_r[row] = L == 0.0f ? 0.0f : 1.0f / L;
}

template <typename T, int D>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 256 ? 1 : D > 128 ? 2 : 3)))
void sums_cols_kernel(const SumsParams P) {
  using Shape = SumsShape<D>;
  using Part = typename Shape::Part;
  constexpr int NKS = Shape::NKS, NT = Shape::TILES;
  constexpr int TK = 16 * NT;  // keys of a wave
  __shared__ __align__(16) unsigned char lds[2 * Shape::STAGE];
  __shared__ __align__(16) float stat[2][2][kTileRows];  // m and 1 / l of the tiles' rows
  const int tid = threadIdx.x, lane = tid & 63, lr = lane >> 4, lc = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // longest items (first keys) first
  int x = blockIdx.x;
  const int bkv = x % (P.batch * P.kv_heads);
  x /= P.batch * P.kv_heads;
  const int rsplit = x % P.n_rsplit;
  const int kt = x / P.n_rsplit;
  const int b = bkv / P.kv_heads, kvh = bkv - b * P.kv_heads;
  const int j0 = (4 * kt + w) * TK;
  const int shift = P.s_k - P.s_q;
  const float c = P.scale_log2;
  const bool active = j0 < P.s_k;

  // 64-row tiles from the first row that sees the item's first key (to 16), of
  // every head of the kv head
  const int rb = max(0, 4 * kt * TK - shift) / 16 * 16;
  const int nt = (P.s_q - rb + kTileRows - 1) / kTileRows;
  const int total = nt * P.group;
  const int t0 = int(int64_t(total) * rsplit / P.n_rsplit);
  const int t1 = int(int64_t(total) * (rsplit + 1) / P.n_rsplit);

  const uint32_t qss = uint32_t(P.q_ss) * 2u;
  const Part part(lane, qss);
  u32x4 qr[Part::NL];
  float st;  // lanes 0..15: m of this wave's rows of the tile, 16..31: 1 / l
  int lg = t0 / nt, lt = t0 - lg * nt;  // head and tile the next load takes
  auto load = [&]() INLINE {
    const int h = kvh * P.group + min(lg, P.group - 1), r = rb + kTileRows * lt + 16 * w;
    const int rc = min(r, P.s_q - 1);
    part.load_at(rows_rsrc(reinterpret_cast<const uint16_t*>(P.q) + b * P.q_sb + int64_t(h) * P.q_sh +
                               int64_t(rc) * P.q_ss,
                           P.s_q - r, 16, qss, D),
                 0, qr);
    if (lane < 32) {
      const float* src = lane < 16 ? P.stat_m : P.stat_r;
      st = src[(int64_t(b) * P.heads + h) * P.s_q_pad + min(r + lc, P.s_q - 1)];
    }
    if (++lt == nt) {
      lt = 0;
      ++lg;
    }
  };
  auto store = [&](int stage) INLINE {
    part.store(lds + stage * Shape::STAGE + w * Part::BYTES, qr);
    if (lane < 32) stat[stage][lane >> 4][16 * w + lc] = st;
  };

  if (t1 > t0) load();  // in flight under the held keys
  u32x4 kb[NT][NKS];
  hold_rows<D, NT>(reinterpret_cast<const uint16_t*>(P.k) + b * P.k_sb + int64_t(kvh) * P.k_sh +
                       int64_t(min(j0, P.s_k - 1)) * P.k_ss,
                   P.s_k - j0, P.k_ss, lane, lds + w * Part::BYTES, kb);

  float acc[NT], sum[NT];
#pragma unroll
  for (int n = 0; n < NT; ++n) acc[n] = sum[n] = 0.0f;
  auto scores = [&](const unsigned char* lp, f32x4 (&s)[NT][2]) INLINE {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int n = 0; n < NT; ++n) s[n][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = Part::operand(lp + u * Part::BYTES, 0, lc, lr, ks);
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][u] = mfma_qk<T>(a, kb[n][ks], s[n][u]);
      }
    }
  };
  // 32 rows from row r on, whose (m, 1 / l) are sp[.] and sp[kTileRows + .]
  auto weigh = [&](int r, bool edge, const float* sp, const f32x4 (&s)[NT][2]) INLINE {
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const f32x4 m = *reinterpret_cast<const f32x4*>(sp + 16 * u + 4 * lr);
      const f32x4 inv = *reinterpret_cast<const f32x4*>(sp + kTileRows + 16 * u + 4 * lr);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[n][u][i], c, -m[i])), f = inv[i];
          const int ri = r + 16 * u + 4 * lr + i;
          if (edge && (shift + ri < j0 + 16 * n + lc || ri >= P.s_q)) e = f = 0.0f;
          acc[n] = __builtin_fmaf(e, f, acc[n]);
        }
    }
  };
  auto flush = [&]() INLINE {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      sum[n] += acc[n];
      acc[n] = 0.0f;
    }
  };

  if (t1 > t0) {
    __syncthreads();  // the held keys have left LDS
    store(0);
    load();
    __syncthreads();
  }
  int ct = t0 % nt;
  for (int t = t0; t < t1; ++t) {
    const int cs = (t - t0) & 1;
    const float* sp = stat[cs][0];
    const int r = rb + kTileRows * ct;
    if (++ct == nt) ct = 0;
    if (active)
      for (int half = 0; half < 2; ++half) {
        const int rh = r + 32 * half;
        const bool edge = shift + rh < j0 + TK - 1 || rh + 32 > P.s_q;
        if (edge && shift + rh + 31 < j0) continue;  // before this wave's first key
        f32x4 s[NT][2];
        scores(lds + cs * Shape::STAGE + 2 * half * Part::BYTES, s);
        if (edge)
          weigh(rh, true, sp + 32 * half, s);
        else
          weigh(rh, false, sp + 32 * half, s);
      }
    store(1 - cs);  // the stage that all waves left before the last barrier
    load();
    __syncthreads();
    if ((t & 7) == 7) flush();
  }
  flush();
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    sum[n] += __shfl_xor(sum[n], 16, 64);
    sum[n] += __shfl_xor(sum[n], 32, 64);
  }
  // lane: key 16 lr + lc of the wave's (lr < NT)
  float r = sum[0];
#pragma unroll
  for (int n = 1; n < NT; ++n) r = lr == n ? sum[n] : r;
  const int j = j0 + 16 * lr + lc;
  if (lr >= NT || j >= P.s_k) return;
  if (P.n_rsplit > 1) {
    P.col_part[(int64_t(rsplit) * P.batch * P.kv_heads + bkv) * P.s_k + j] = r;
  } else {
    float* o = P.sums + b * P.s_sb + kvh * P.s_sh + j;
    *o = P.add ? *o + r : r;
  }
}

// Lane's share of the sums of v[0..7] over its row of 16 lanes: of v[4 b3 + 2 b2 +
// b1], b the bits of its place in the row.
__device__ INLINE inline float row_sums(const float (&v)[8], int lc) {
  const auto from = [](auto ctrl, float x) INLINE {
    return __builtin_bit_cast(
        float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl(), 0xf, 0xf, true));
  };
  const bool b3 = lc & 8, b2 = lc & 4, b1 = lc & 2;
  float a[4], b[2];
#pragma unroll
  for (int i = 0; i < 4; ++i)  // row_ror:8, lane ^ 8
    a[i] = (b3 ? v[4 + i] : v[i]) + from(std::integral_constant<int, 0x128>{}, b3 ? v[i] : v[4 + i]);
#pragma unroll
  for (int i = 0; i < 2; ++i)  // row_half_mirror, lane ^ 7
    b[i] = (b2 ? a[2 + i] : a[i]) + from(std::integral_constant<int, 0x141>{}, b2 ? a[i] : a[2 + i]);
  // quad_perm [2,3,0,1], lane ^ 2, then [1,0,3,2], lane ^ 1
  const float c = (b1 ? b[1] : b[0]) + from(std::integral_constant<int, 0x4e>{}, b1 ? b[0] : b[1]);
  return c + from(std::integral_constant<int, 0xb1>{}, c);
}

// Columns of one tile of rows against many keys (one head a kv head, S_q up to the
// rows a wave holds): the items of the stats pass, the rows held and the keys
// walked, so that the keys' loads run ahead of the work.
template <typename T, int D, int MT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 256 ? 1 : 2)))
void sums_window_kernel(const SumsParams P) {
  using Shape = SumsShape<D>;
  using Part = typename Shape::Part;
  constexpr int NKS = Shape::NKS;
  __shared__ __align__(16) unsigned char lds[2 * Shape::STAGE];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane >> 4, lc = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int bh = blockIdx.x % (P.batch * P.heads), split = blockIdx.x / (P.batch * P.heads);
  const int b = bh / P.heads, h = bh - b * P.heads;
  const int shift = P.s_k - P.s_q;
  const int j_begin = split * P.chunk, j_end = min(j_begin + P.chunk, P.s_k);
  const float c = P.scale_log2;

  const uint16_t* kbase = reinterpret_cast<const uint16_t*>(P.k) + b * P.k_sb + int64_t(h) * P.k_sh;
  const uint32_t kss = uint32_t(P.k_ss) * 2u;
  const Part part(lane, kss);
  u32x4 kr[2][Part::NL];
  auto load = [&](int j0) INLINE {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      load_keys(P, part, rows_rsrc(kbase + int64_t(min(j0 + 16 * u, P.s_k - 1)) * P.k_ss,
                                   P.s_k - j0 - 16 * u, 16, kss, D), kr[u]);
  };
  u32x4 qb[MT][NKS];
  hold_rows<D, MT>(reinterpret_cast<const uint16_t*>(P.q) + b * P.q_sb + int64_t(h) * P.q_sh, P.s_q,
                   P.q_ss, lane, lds + w * Part::BYTES, qb);
  float m[MT], inv[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = 16 * mt + lc;
    m[mt] = r < P.s_q ? P.stat_m[int64_t(bh) * P.s_q_pad + r] : 0.0f;
    inv[mt] = r < P.s_q ? P.stat_r[int64_t(bh) * P.s_q_pad + r] : 0.0f;
  }
  unsigned char* mine = lds + w * 2 * Part::BYTES;
  float* out = P.sums + b * P.s_sb + h * P.s_sh;
  const int place = 16 * (lc >> 3) + 4 * lr + 2 * ((lc >> 2) & 1) + ((lc >> 1) & 1);  // row_sums' key
  const int first = j_begin + 32 * w;
  __syncthreads();  // the held rows have left LDS
  load(first);
  for (int j0 = first; j0 < j_end; j0 += 128) {
#pragma unroll
    for (int u = 0; u < 2; ++u) part.store(mine + u * Part::BYTES, kr[u]);
    wave_lds_fence();
    load(j0 + 128);
    const int j = j0 + place;
    const bool stores = (lc & 1) == 0 && j < j_end;
    const float old = P.add && stores ? out[j] : 0.0f;
    f32x4 s[MT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) s[mt][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = Part::operand(mine + u * Part::BYTES, 0, lc, lr, ks);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) s[mt][u] = mfma_qk<T>(a, qb[mt][ks], s[mt][u]);
      }
    }
    float v[8];
    auto weigh = [&](bool edge) INLINE {
#pragma unroll
      for (int x = 0; x < 8; ++x) {
        v[x] = 0.0f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[mt][x >> 2][x & 3], c, -m[mt])), f = inv[mt];
          if (edge && j0 + 16 * (x >> 2) + 4 * lr + (x & 3) > shift + 16 * mt + lc) e = f = 0.0f;
          v[x] = __builtin_fmaf(e, f, v[x]);
        }
      }
    };
    if (j0 + 31 > shift)
      weigh(true);
    else
      weigh(false);
    wave_lds_fence();
    const float r = row_sums(v, lc);
    if (stores) out[j] = P.add ? old + r : r;
  }
}

// Column sums of the row splits, in order.
__global__ __launch_bounds__(256) void sums_reduce_kernel(const SumsParams P) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= P.s_k) return;
  const int bkv = blockIdx.y, b = bkv / P.kv_heads, kvh = bkv - b * P.kv_heads;
  float r = 0.0f;
  for (int s = 0; s < P.n_rsplit; ++s)
    r += P.col_part[(int64_t(s) * P.batch * P.kv_heads + bkv) * P.s_k + j];
  float* o = P.sums + b * P.s_sb + kvh * P.s_sh + j;
  *o = P.add ? *o + r : r;
}

template <typename T, int D>
hipError_t launch_sums_d(const SumsParams& p, hipStream_t st) {
  constexpr int NT = SumsShape<D>::TILES;
  const int64_t bh = int64_t(p.batch) * p.heads;
  const dim3 ga(uint32_t(bh * p.n_rt * p.n_split));
  if (p.share)
    hipLaunchKernelGGL((sums_stats_kernel<T, D, NT, true>), ga, dim3(256), 0, st, p);
  else if (p.stat_rows == 16)
    hipLaunchKernelGGL((sums_stats_kernel<T, D, 1, false>), ga, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((sums_stats_kernel<T, D, NT, false>), ga, dim3(256), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.n_split > 1) {
    hipLaunchKernelGGL(sums_merge_kernel, dim3(uint32_t(bh * p.s_q_pad / 16)), dim3(256), 0, st, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.window) {
    if (p.stat_rows == 16)
      hipLaunchKernelGGL((sums_window_kernel<T, D, 1>), ga, dim3(256), 0, st, p);
    else
      hipLaunchKernelGGL((sums_window_kernel<T, D, NT>), ga, dim3(256), 0, st, p);
    return hipGetLastError();
  }
  const uint32_t bkv = uint32_t(p.batch) * p.kv_heads;
  hipLaunchKernelGGL((sums_cols_kernel<T, D>), dim3(bkv * p.n_rsplit * p.n_kt), dim3(256), 0, st, p);
  e = hipGetLastError();
  if (e != hipSuccess || p.n_rsplit == 1) return e;
  hipLaunchKernelGGL(sums_reduce_kernel, dim3((p.s_k + 255) / 256, bkv), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_sums_t(const SumsParams& p, int D, hipStream_t st) {
  if (D == 64) return launch_sums_d<T, 64>(p, st);
  if (D == 96) return launch_sums_d<T, 96>(p, st);
  if (D == 128) return launch_sums_d<T, 128>(p, st);
  if (D == 256) return launch_sums_d<T, 256>(p, st);
  return launch_sums_d<T, 512>(p, st);
}

}  // namespace

int sums_tiles(int D) { return D <= 128 ? 4 : D == 256 ? 2 : 1; }

hipError_t launch_sums(const SumsParams& p, int dtype, int D, hipStream_t st) {
  return dtype == Bf16::id ? launch_sums_t<Bf16>(p, D, st) : launch_sums_t<F16>(p, D, st);
}

}  // namespace msa
