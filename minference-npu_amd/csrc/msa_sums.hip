// Attention weights of the last S_q rows of a prompt, summed per key:
//   sums[b][g][j] = sum over the heads h of kv head g and the rows i of
//                   softmax_i(q_bhi . k_bg * scale)[j],
// row i at position S_k - S_q + i, keys up to its own position.  What a cache is
// cut by after a prefill.
//
// A weight needs its row's maximum and sum over all keys, a column sum needs
// the weights of all rows, so q.k is taken twice:
//   stats: an item holds up to 64 rows of a head as the B operand and walks the
//     keys: S^T = K . Q^T, lane (lc, lr) gets row lc, keys 4 lr + i.  Each lane
//     keeps a running (m, l) of the keys it sees: no exchange until the end.
//   columns: an item holds 64 keys of a kv head as the B operand and walks the
//     rows of all its heads: S = Q . K^T, lane (lc, lr) gets key lc, rows 4 lr +
//     i, whose (m, 1 / l) are one 32-byte read.  Each lane sums its keys' weights
//     in registers.
// No LDS in the loops.  Bound by the exponentials, two for each visible pair (a
// quarter-rate instruction), with the products beside them: q.k costs a 16x16
// tile D / 32 MFMAs, its 256 weights a fused multiply-add, an exponential and
// an add a lane four times.
// Sums are fp32 in two levels (16 blocks of 16 rows, then those), in a fixed
// order.

#include "msa_common.h"
#include "msa_kernels.h"

namespace msa {

#define INLINE __attribute__((always_inline))

namespace {

template <int D>
struct SumsShape {
  static constexpr int NKS = D / 32;
  static constexpr int TILES = D <= 128 ? 4 : D == 256 ? 2 : 1;  // 16-row tiles held by an item
};

// Descriptor of up to `rows` rows from `p` on, `left` of which exist (at least
// one): loads of the others return 0.
__device__ inline __amdgpu_buffer_rsrc_t rows_rsrc(const uint16_t* p, int left, int rows,
                                                   uint32_t stride, int D) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(p), short(0),
                                           int(uint32_t(min(left, rows) - 1) * stride + 2 * D),
                                           0x00020000);
}

template <typename T, int D, int MT>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 256 ? 1 : 2)))
void sums_stats_kernel(const SumsParams P) {
  constexpr int NKS = SumsShape<D>::NKS;
  constexpr int KB = 32;  // keys of a block
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
  const int row0 = rt * 16 * MT;
  const int n_rows = min(16 * MT, P.s_q - row0);
  const int shift = P.s_k - P.s_q;
  const int j_begin = split * P.chunk;
  const int j_end = min(min(j_begin + P.chunk, P.s_k), shift + row0 + n_rows);

  u32x4 qb[MT][NKS];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const uint16_t* qrow = reinterpret_cast<const uint16_t*>(P.q) + b * P.q_sb + int64_t(h) * P.q_sh +
                           int64_t(row0 + min(16 * mt + lc, n_rows - 1)) * P.q_ss;
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qb[mt][ks] = load16(qrow + 32 * ks + 8 * lr);
  }
  const uint16_t* kbase = reinterpret_cast<const uint16_t*>(P.k) + b * P.k_sb +
                          int64_t(h / P.group) * P.k_sh;
  const uint32_t kss = uint32_t(P.k_ss) * 2u;
  const uint32_t koff = uint32_t(lc) * kss + 16u * lr;
  auto load_block = [&](int j0, u32x4 (&kr)[2][NKS]) INLINE {
    const __amdgpu_buffer_rsrc_t rs =
        rows_rsrc(kbase + int64_t(j0) * P.k_ss, P.s_k - j0, KB, kss, D);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        kr[u][ks] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, koff + 16u * u * kss + 64 * ks, 0, 0));
  };

  // of the keys this lane sees: running max, what the exponentials are taken
  // against, and the sum in two levels (small terms are not lost in a long sum)
  float m[MT], mp[MT], l[MT], part[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -__builtin_inff();
    mp[mt] = 0.0f;
    l[mt] = part[mt] = 0.0f;
  }
  const float c = P.scale_log2;
  auto block = [&](int j0, const u32x4 (&kr)[2][NKS]) INLINE {
    const bool edge = j0 + KB - 1 > shift + row0;  // some row does not see the whole block
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x4 s[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        s[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s[u] = mfma_qk<T>(kr[u][ks], qb[mt][ks], s[u]);
      }
      if (edge) {
        const int last = min(shift + row0 + 16 * mt + lc, j_end - 1);
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (j0 + 16 * u + 4 * lr + i > last) s[u][i] = -__builtin_inff();
      }
      const float bm = max8(s[0], s[1]) * c;
      if (__ballot(bm > m[mt] + 16.0f) != 0) {
        const float mn = fmaxf(m[mt], bm);
        mp[mt] = mn == -__builtin_inff() ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m[mt] - mp[mt]);
        l[mt] *= al;
        part[mt] *= al;
        m[mt] = mn;
      }
      float e[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        e[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], c, -mp[mt]));
      part[mt] += ((e[0] + e[1]) + (e[2] + e[3])) + ((e[4] + e[5]) + (e[6] + e[7]));
    }
  };
  auto flush = [&]() INLINE {
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      l[mt] += part[mt];
      part[mt] = 0.0f;
    }
  };
  const int first = j_begin + KB * w;
  const int nblk = j_end > first ? (j_end - first + 4 * KB - 1) / (4 * KB) : 0;
  auto jb = [&](int i) { return first + 4 * KB * min(i, nblk - 1); };
  if (nblk > 0) {
    u32x4 ka[2][NKS], kb[2][NKS];
    load_block(jb(0), ka);
    for (int i = 0; i < nblk; i += 2) {
      load_block(jb(i + 1), kb);
      block(jb(i), ka);
      if (i + 1 >= nblk) break;
      load_block(jb(i + 2), ka);
      block(jb(i + 1), kb);
      if ((i & 14) == 14) flush();
    }
    flush();
  }

  // merge a row's lanes, then the waves
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
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
  if (tid < 16 * MT) {
    float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
    for (int v = 0; v < 4; ++v) M = fmaxf(M, sm[v][tid]);
#pragma unroll
    for (int v = 0; v < 4; ++v)
      if (sm[v][tid] != -__builtin_inff()) L += __builtin_amdgcn_exp2f(sm[v][tid] - M) * sl[v][tid];
    const int64_t row = int64_t(bh) * P.s_q_pad + row0 + tid;
    if (row0 + tid < P.s_q_pad) {
      if (P.n_split > 1) {
        float2* part = reinterpret_cast<float2*>(P.part) +
                       int64_t(split) * P.batch * P.heads * P.s_q_pad;
        part[row] = make_float2(M, L);
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
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 256 ? 1 : 2)))
void sums_cols_kernel(const SumsParams P) {
  constexpr int NKS = SumsShape<D>::NKS, NT = SumsShape<D>::TILES;
  constexpr int TK = 16 * NT;  // keys of a wave
  __shared__ float red[4][TK];
  const int tid = threadIdx.x, lane = tid & 63, lr = lane >> 4, lc = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // longest items (first keys) first
  int x = blockIdx.x;
  const int bkv = x % (P.batch * P.kv_heads);
  x /= P.batch * P.kv_heads;
  const int rsplit = x % P.n_rsplit;
  const int kt = x / P.n_rsplit;
  const int b = bkv / P.kv_heads, kvh = bkv - b * P.kv_heads;
  const int j0 = P.wave_keys ? (4 * kt + w) * TK : kt * TK;
  const int shift = P.s_k - P.s_q;
  const float c = P.scale_log2;

  float acc[NT];
#pragma unroll
  for (int t = 0; t < NT; ++t) acc[t] = 0.0f;
  if (j0 < P.s_k) {
    const uint16_t* kbase = reinterpret_cast<const uint16_t*>(P.k) + b * P.k_sb + int64_t(kvh) * P.k_sh;
    u32x4 kb[NT][NKS];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint16_t* krow = kbase + int64_t(min(j0 + 16 * t + lc, P.s_k - 1)) * P.k_ss;
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) kb[t][ks] = load16(krow + 32 * ks + 8 * lr);
    }
    const uint32_t qss = uint32_t(P.q_ss) * 2u;
    const uint32_t qoff = uint32_t(lc) * qss + 16u * lr;
    // 16-row blocks from the first row that sees key j0, of every head
    const int rb0 = max(0, j0 - shift) / 16, nb = P.s_q_pad / 16 - rb0;
    const int total = nb * P.group;
    const int t0 = int(int64_t(total) * rsplit / P.n_rsplit);
    const int t1 = int(int64_t(total) * (rsplit + 1) / P.n_rsplit);
    const int step = P.wave_keys ? 1 : 4, first = t0 + (P.wave_keys ? 0 : w);

    auto load_block = [&](int t, u32x4 (&qr)[NKS], f32x4& sm, f32x4& sr) INLINE {
      const int g = t / nb, r0 = 16 * (rb0 + t - g * nb);
      const int h = kvh * P.group + g;
      const uint16_t* q0 = reinterpret_cast<const uint16_t*>(P.q) + b * P.q_sb + int64_t(h) * P.q_sh +
                           int64_t(r0) * P.q_ss;
      const __amdgpu_buffer_rsrc_t rs = rows_rsrc(q0, P.s_q - r0, 16, qss, D);
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks)
        qr[ks] = __builtin_bit_cast(
            u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, qoff + 64 * ks, 0, 0));
      const int64_t row = (int64_t(b) * P.heads + h) * P.s_q_pad + r0 + 4 * lr;
      sm = *reinterpret_cast<const f32x4*>(P.stat_m + row);
      sr = *reinterpret_cast<const f32x4*>(P.stat_r + row);
    };
    float part[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) part[t] = 0.0f;
    auto block = [&](int t, const u32x4 (&qr)[NKS], const f32x4& sm, const f32x4& sr) INLINE {
      const int row = 16 * (rb0 + t % nb);
      const bool edge = shift + row < j0 + TK - 1 || row + 16 > P.s_q;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        f32x4 s = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < NKS; ++ks) s = mfma_qk<T>(qr[ks], kb[n][ks], s);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float e = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -sm[i])), r = sr[i];
          const int ri = row + 4 * lr + i;
          if (edge && (shift + ri < j0 + 16 * n + lc || ri >= P.s_q)) e = r = 0.0f;
          part[n] = __builtin_fmaf(e, r, part[n]);
        }
      }
    };
    auto flush = [&]() INLINE {
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        acc[n] += part[n];
        part[n] = 0.0f;
      }
    };
    const int nblk = t1 > first ? (t1 - first + step - 1) / step : 0;
    auto tb = [&](int i) { return first + step * min(i, nblk - 1); };
    if (nblk > 0) {
      u32x4 qa[NKS], qc[NKS];
      f32x4 ma, ra, mc, rc;
      load_block(tb(0), qa, ma, ra);
      for (int i = 0; i < nblk; i += 2) {
        load_block(tb(i + 1), qc, mc, rc);
        block(tb(i), qa, ma, ra);
        if (i + 1 >= nblk) break;
        load_block(tb(i + 2), qa, ma, ra);
        block(tb(i + 1), qc, mc, rc);
        if ((i & 14) == 14) flush();
      }
      flush();
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      acc[n] += __shfl_xor(acc[n], 16, 64);
      acc[n] += __shfl_xor(acc[n], 32, 64);
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
    if (lr == 0) red[w][16 * n + lc] = acc[n];
  __syncthreads();
  const int nk = P.wave_keys ? 4 * TK : TK, jt = kt * nk;
  for (int y = tid; y < nk && jt + y < P.s_k; y += 256) {
    const float r = P.wave_keys ? red[y / TK][y % TK]
                                : (red[0][y] + red[1][y]) + (red[2][y] + red[3][y]);
    if (P.n_rsplit > 1) {
      P.col_part[(int64_t(rsplit) * P.batch * P.kv_heads + bkv) * P.s_k + jt + y] = r;
    } else {
      float* o = P.sums + b * P.s_sb + kvh * P.s_sh + jt + y;
      *o = P.add ? *o + r : r;
    }
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
  if (p.mt == 1)
    hipLaunchKernelGGL((sums_stats_kernel<T, D, 1>), ga, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL((sums_stats_kernel<T, D, NT>), ga, dim3(256), 0, st, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (p.n_split > 1) {
    hipLaunchKernelGGL(sums_merge_kernel, dim3(uint32_t(bh * p.s_q_pad / 16)), dim3(256), 0, st, p);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
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
