// Attention of a few query rows per kv head against long caches, split over
// the keys: a batch that shares a prefix, and decode that also leaves the
// attention weights.
//
// shared prefix: row i of sequence b sees every key of the prefix, one cache
// for all sequences, and its own sequence's keys up to its own position.  The
// query rows of all sequences and of the query heads of a kv head form one
// matrix against the prefix, so the prefix is read once per 64 rows instead of
// once per sequence.
// decode with accumulation: one query row per head against a cache of lens[b]
// keys; the raw scores go to the workspace and the second launch adds the
// normalised weights, summed over the heads of a kv head, to a score per key.
//
// A workgroup takes one item: rows of one kv head against one key range (of the
// prefix, or of one sequence's own cache).
//   S^T = K . Q^T on the 16-bit 16x16x32 MFMA (exact products, fp32 sums): A
//     = 16 keys from their rows, B = 16 query rows, held for the whole item.
//     Lane (lc, lr) gets query lc, keys 4 lr + i of the 16.
//   O^T += V^T . P^T on the same MFMA, 32 keys a step.  The order of the 32 is
//     free as long as V and P share it: slot 8 lr + j is key 4 lr + j of the
//     block's first 16 for j < 4, of the second 16 after that, which is where
//     P already lies.
// kOwn (up to 16 rows): wave w takes the 32-key blocks w, w + 4, ...; K goes
//   through LDS (each wave its own block, no barrier), V straight from its rows, a
//   lane holding E = D / 16 (8 from D = 128 on) dims of its 8 keys, and pairs of
//   keys are put together by byte permutes; MFMA e takes dim E lc + e of every lane.
//   Bound by memory: 16 rows on 8 x 1 M keys of 128 dims 6.7 TB/s; decode of 8 ragged
//   sequences on 8 x 65536 x 128 265 us, 5.5 TB/s, the raw scores' stores 20 of it.
// kTile (up to 64 MT rows): the waves share 64 keys in LDS and take 16 MT rows each.
//   Bound by the sum of the products (two of P where kTwoParts says so) and the
//   softmax, which hardly overlap: 128 rows a kv head on 8 x 65536 x 128, with 32 x
//   8 own caches of up to 1024 keys, 84 us (4.3 TB/s); 512 rows on 8 x 32768 x 128
//   fp16, with 128 x 8 caches of up to 512, 129 us (0.55 PFLOP/s).
// Softmax statistics and O are fp32; a row's running max moves only when a block
// exceeds it by 2^kSlack.  P is rounded to the inputs' type twice, P and what that
// rounding left, so the product's error stays below the output's own rounding
// (kTwoParts names the exception).
// Each item leaves O and (m, l) of its rows in the workspace; the second launch
// merges the items of a row (4 us for 128 rows, 10 for 1024, 13 for 4096).

#include "msa_common.h"
#include "msa_kernels.h"
#include "msa_tile.h"

namespace msa {

#define INLINE __attribute__((always_inline))

namespace {

typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x3 __attribute__((ext_vector_type(3)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr float kSlack = 8.0f;  // P up to 2^8: far inside fp16

template <typename T>
__device__ inline uint32_t pack2(float a, float b) {
  if constexpr (T::id == Bf16::id)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, f16x2));
}
template <typename T>
__device__ inline float lo_of(uint32_t x) { return T::to_float(uint16_t(x & 0xffffu)); }
template <typename T>
__device__ inline float hi_of(uint32_t x) { return T::to_float(uint16_t(x >> 16)); }

// Exponent all ones in either half of a packed pair.
template <typename T>
__device__ inline bool any_nonfinite(uint32_t x) {
  constexpr uint32_t e = T::id == Bf16::id ? 0x7f80u : 0x7c00u;
  return (x & e) == e || (x & (e << 16)) == (e << 16);
}

template <int W, int AUX>
__device__ inline void load_words(__amdgpu_buffer_rsrc_t rs, uint32_t off, uint32_t soff,
                                  uint32_t (&w)[W]) {
  if constexpr (W == 4) {
    const u32x4 x = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, off, soff, AUX));
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = x[i];
  } else if constexpr (W == 3) {
    const u32x3 x = __builtin_bit_cast(u32x3, __builtin_amdgcn_raw_buffer_load_b96(rs, off, soff, AUX));
#pragma unroll
    for (int i = 0; i < 3; ++i) w[i] = x[i];
  } else {
    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rs, off, soff, AUX));
#pragma unroll
    for (int i = 0; i < 2; ++i) w[i] = x[i];
  }
}

struct Item {
  const uint16_t* k;  // first key of the item's range
  const uint16_t* v;
  uint32_t kss, vss;  // row strides, bytes
  int n_keys;         // visible keys of the range (0 or less: none)
  int row0, n_rows;   // rows of the kv head in (sequence, head, position) order
  int seq_rows;       // rows of one sequence: group * s_q
  int kvh;
  int limit;          // CAUSAL: position i sees local keys j <= limit + i
  int64_t part_row;   // first row of part / ml
  float* raw;         // SCORES: raw score of (row 0, local key 0)
  int64_t raw_row;    // SCORES: floats between rows
};

// Row r of the kv head as an offset into q.
__device__ inline int64_t q_offset(const RowsParams& P, int kvh, int seq_rows, int r) {
  const int b = r / seq_rows, rr = r - b * seq_rows;
  const int g = rr / P.s_q, i = rr - g * P.s_q;
  return b * P.q_sb + int64_t(kvh * P.group + g) * P.q_sh + int64_t(i) * P.q_ss;
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

// V operand of 16 dims and 32 keys from LDS: 4 keys at p, 4 keys `far` bytes on.
__device__ inline u32x4 v_operand(const unsigned char* p, int far) {
  const u32x2 a = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(const_cast<unsigned char*>(p))));
  const u32x2 b = __builtin_bit_cast(
      u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)(const_cast<unsigned char*>(p + far))));
  return u32x4{a[0], a[1], b[0], b[1]};
}

// A packed pair with its Inf and NaN as 0.
template <typename T>
__device__ inline uint32_t finite_only(uint32_t x) {
  constexpr uint32_t e = T::id == Bf16::id ? 0x7f80u : 0x7c00u;
  if ((x & e) == e) x &= 0xffff0000u;
  if ((x & (e << 16)) == (e << 16)) x &= 0xffffu;
  return x;
}

// What the Inf and NaN values of V among the 32 keys from local key j0 add to
// the rows that see them, one key at a time (kTile's layout of O).
template <typename T, int MT, int ND>
__device__ INLINE inline void add_nonfinite(const Item& it, int j0, int lane,
                                                        const u32x4 (&ph)[MT], const u32x4 (&pl)[MT],
                                                        const int (&lim)[MT], f32x4 (&o)[MT][ND]) {
  const int lr = lane >> 4, lc = lane & 15;
  for (int kk = 0; kk < 32 && j0 + kk < it.n_keys; ++kk) {
    const uint16_t* vrow = it.v + int64_t(j0 + kk) * (it.vss / 2);
    const int slot = 4 * (kk >> 4) + (kk & 3);  // P's place in its lane
    const int src = lc + 16 * ((kk & 15) >> 2);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      uint32_t hw = 0, lw = 0;
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if ((slot >> 1) == x) {
          hw = ph[mt][x];
          lw = pl[mt][x];
        }
      const float pv = (slot & 1) ? hi_of<T>(hw) + hi_of<T>(lw) : lo_of<T>(hw) + lo_of<T>(lw);
      const float pk = __shfl(pv, src, 64);
      const bool sees = j0 + kk <= lim[mt];
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float x = T::to_float(vrow[16 * n + 4 * lr + i]);
          if (sees && !__builtin_isfinite(x)) o[mt][n][i] += pk * x;
        }
    }
  }
}

// Forms of an item (rows_forms): kOwn + MT: up to 16 MT rows, the four waves take
// different keys; kTile + MT: up to 64 MT rows, 16 MT a wave, the waves share the keys.
constexpr int kOwn = 0, kTile = 8;
constexpr int form_rows(int form) {
  return form >= kTile ? 64 * (form - kTile) : 16 * form;
}
constexpr int kTileKeys = 64;

// Bytes between V rows of a tile in LDS: 8 rows that a half wave reads 32 bytes
// of each lie in 8 different groups of 8 banks.
constexpr int v_row_bytes(int D) { return 2 * D + 32; }

template <int D, int FORMS>  // FORMS: 1 when a tile form is among them
struct RowsShared {
  static constexpr int LP = (D < 128 ? D : 128) + 4;  // padded row
  static constexpr int STAGE = FORMS ? kTileKeys * (2 * D + v_row_bytes(D)) : 16;
  union {
    __align__(16) unsigned char k[4][Tile<D, 32>::BYTES];  // kOwn: each wave's key block
    __align__(16) float om[4][16][LP];                      // kOwn: merge of the waves
    __align__(16) unsigned char kv[2][STAGE];               // kTile: K and V of two tiles
  };
  float sm[4][32], sl[4][32];
};

template <typename T, int D, int MT, bool CAUSAL, bool SCORES, typename Shared>
__device__ void rows_item(const RowsParams& P, const Item& it, Shared& sh) {
  constexpr int NKS = D / 32;
  constexpr int VG = (D + 127) / 128;       // groups of 128 dims of V
  constexpr int E = D < 128 ? D / 16 : 8;   // dims of a lane in a group
  constexpr int W = E / 2;
  constexpr int DG = 16 * E;                // dims of a group
  constexpr int AUX = 2;  // the item reads its keys alone, once: non-temporal loads
  auto& om = sh.om;
  auto& sm = sh.sm;
  auto& sl = sh.sl;

  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int lr = lane >> 4;
  const int lc = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  if (it.n_keys <= 0) {  // nothing visible: an empty split
    for (int r = tid; r < it.n_rows; r += 256) {
      P.ml[2 * (it.part_row + r)] = -__builtin_inff();
      P.ml[2 * (it.part_row + r) + 1] = 0.0f;
    }
    return;
  }

  // query rows as the QK B operand: lane (lc, lr) holds dims 32 ks + 8 lr .. +7
  // of row lc (rows past n_rows repeat the last one and are not stored)
  u32x4 qb[MT][NKS];
  int lim[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = it.row0 + min(16 * mt + lc, it.n_rows - 1);
    const uint16_t* qrow =
        reinterpret_cast<const uint16_t*>(P.q) + q_offset(P, it.kvh, it.seq_rows, r);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qb[mt][ks] = load16(qrow + 32 * ks + 8 * lr);
    lim[mt] = CAUSAL ? it.limit + r % P.s_q : 0;
  }

  // Buffer descriptors end with the last visible key, so rows behind it,
  // whatever they hold, read 0.
  const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(it.k), short(0), int(uint32_t(it.n_keys - 1) * it.kss + 2 * D), 0x00020000);
  const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(it.v), short(0), int(uint32_t(it.n_keys - 1) * it.vss + 2 * D), 0x00020000);
  using KTile = Tile<D, 32>;
  const KTile ktile(lane, it.kss);
  unsigned char* kl = sh.k[w];
  uint32_t voff[8];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    voff[j] = uint32_t(16 * (j >> 2) + 4 * lr + (j & 3)) * it.vss + 2u * E * lc;

  // The scalar offset names the block's first key, which is visible: the
  // range check compares the lane offset with the records left behind it.
  u32x4 kr[KTile::NL];  // the next key block on its way to LDS
  auto load_k = [&](int j0) INLINE { ktile.template load<AUX>(krs, uint32_t(j0) * it.kss, kr); };
  auto load_v = [&](int j0, uint32_t (&vr)[8][VG][W]) INLINE {
    const uint32_t vs0 = uint32_t(j0) * it.vss;
#pragma unroll
    for (int j = 0; j < 8; ++j)
#pragma unroll
      for (int g = 0; g < VG; ++g) load_words<W, AUX>(vrs, voff[j] + 256 * g, vs0, vr[j][g]);
  };

  // o[mt][g][e]: lane (lc, lr) holds row lc, dims 128 g + E (4 lr + j) + e
  f32x4 o[MT][VG][E];
  float m[MT], mp[MT], l[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -__builtin_inff();  // running max, raw scores times c, the same in a row's 4 lanes
    mp[mt] = 0.0f;              // what P is taken against: m, or 0 without a score above -inf
    l[mt] = 0.0f;               // this lane's share of the sum
#pragma unroll
    for (int g = 0; g < VG; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) o[mt][g][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float c = P.scale_log2;

  auto block = [&](int j0, int next, uint32_t (&vr)[8][VG][W]) INLINE {
    ktile.store(kl, kr);
    wave_lds_fence();
    load_k(next);
    f32x4 st[MT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) st[mt][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = KTile::operand(kl, u, lc, lr, ks);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) st[mt][u] = mfma_qk<T>(a, qb[mt][ks], st[mt][u]);
      }
    }
    wave_lds_fence();
    const bool edge = CAUSAL ? j0 + 31 > it.limit : j0 + 32 > it.n_keys;
    u32x4 ph[MT], pl[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x4(&s)[2] = st[mt];
      if (SCORES && lc < it.n_rows) {  // MT == 1; rows of raw end with a multiple of 32 keys
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *reinterpret_cast<f32x4*>(it.raw + lc * it.raw_row + j0 + 16 * u + 4 * lr) = s[u];
      }
      if (edge) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = j0 + 16 * u + 4 * lr + i;
            if (CAUSAL ? j > lim[mt] || j >= it.n_keys : j >= it.n_keys) s[u][i] = -__builtin_inff();
          }
      }
      // the lanes of a row compare their own keys; they only exchange to move it
      float bm = max8(s[0], s[1]) * c;
      if (__ballot(bm > m[mt] + kSlack) != 0) {
        bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
        bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
        const float mn = fmaxf(m[mt], bm);
        mp[mt] = mn == -__builtin_inff() ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m[mt] - mp[mt]);  // m = -inf at first: 0
        m[mt] = mn;
        l[mt] *= al;
#pragma unroll
        for (int g = 0; g < VG; ++g)
#pragma unroll
          for (int e = 0; e < E; ++e) o[mt][g][e] *= al;
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], c, -mp[mt]));
      l[mt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ph[mt][j] = pack2<T>(p[2 * j], p[2 * j + 1]);
        pl[mt][j] = pack2<T>(__builtin_fmaf(lo_of<T>(ph[mt][j]), -1.0f, p[2 * j]),
                             __builtin_fmaf(hi_of<T>(ph[mt][j]), -1.0f, p[2 * j + 1]));
      }
    }
    if (CAUSAL && edge) {
      // A key that some rows see and others do not: a zero P times an Inf or
      // NaN of its V would reach the others.  Such values leave the product
      // and are added one key at a time, to the rows that see it.
      bool bad = false;
#pragma unroll
      for (int j = 0; j < 8; ++j)
#pragma unroll
        for (int g = 0; g < VG; ++g)
#pragma unroll
          for (int x = 0; x < W; ++x) bad |= any_nonfinite<T>(vr[j][g][x]);
      if (__ballot(bad) != 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
          for (int g = 0; g < VG; ++g)
#pragma unroll
            for (int x = 0; x < W; ++x) {
              vr[j][g][x] = finite_only<T>(vr[j][g][x]);
            }
        for (int kk = 0; kk < 32 && j0 + kk < it.n_keys; ++kk) {
          const uint16_t* vrow = it.v + int64_t(j0 + kk) * (it.vss / 2);
          const int slot = 4 * (kk >> 4) + (kk & 3);  // P's place in its lane
          const int src = lc + 16 * ((kk & 15) >> 2);
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) {
            uint32_t hw = 0, lw = 0;
#pragma unroll
            for (int x = 0; x < 4; ++x)
              if ((slot >> 1) == x) {
                hw = ph[mt][x];
                lw = pl[mt][x];
              }
            const float pv = (slot & 1) ? hi_of<T>(hw) + hi_of<T>(lw) : lo_of<T>(hw) + lo_of<T>(lw);
            const float pk = __shfl(pv, src, 64);
            const bool sees = j0 + kk <= lim[mt];
#pragma unroll
            for (int g = 0; g < VG; ++g)
#pragma unroll
              for (int e = 0; e < E; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const float x = T::to_float(vrow[128 * g + E * (4 * lr + i) + e]);
                  if (sees && !__builtin_isfinite(x)) o[mt][g][e][i] += pk * x;
                }
          }
        }
      }
    }
#pragma unroll
    for (int g = 0; g < VG; ++g)
#pragma unroll
      for (int e = 0; e < E; ++e) {
        u32x4 a;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          a[j] = __builtin_amdgcn_perm(vr[2 * j + 1][g][e >> 1], vr[2 * j][g][e >> 1],
                                       e & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          o[mt][g][e] = mfma_qk<T>(a, ph[mt], o[mt][g][e]);
          o[mt][g][e] = mfma_qk<T>(a, pl[mt], o[mt][g][e]);
        }
      }
  };

  // Wave w takes blocks first + 128 i, i < nblk; a block's loads are in flight
  // under the block before.  Loads past the wave's last block repeat it, so
  // every load is unconditional.
  const int first = 32 * w;
  const int nblk = it.n_keys > first ? (it.n_keys - first + 127) / 128 : 0;
  auto jb = [&](int i) { return first + 128 * min(i, nblk - 1); };
  if (nblk > 0) {
    load_k(jb(0));
    if constexpr (D > 256) {  // one V set: q, O, K and V of a block fill the registers
      for (int i = 0; i < nblk; ++i) {
        uint32_t va[8][VG][W];
        load_v(jb(i), va);
        block(jb(i), jb(i + 1), va);
      }
    } else {
      uint32_t va[8][VG][W], vb[8][VG][W];
      load_v(jb(0), va);
      for (int i = 0; i < nblk; i += 2) {
        load_v(jb(i + 1), vb);
        block(jb(i), jb(i + 1), va);
        if (i + 1 >= nblk) break;
        load_v(jb(i + 2), va);
        block(jb(i + 1), jb(i + 2), vb);
      }
    }
  }

  // ---- merge the 4 waves, 16 rows and a group of dims at a time
  __syncthreads();  // om lies where the key blocks were
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] += __shfl_xor(l[mt], 16, 64);
    l[mt] += __shfl_xor(l[mt], 32, 64);
    if (lr == 0) {
      sm[w][16 * mt + lc] = m[mt];
      sl[w][16 * mt + lc] = l[mt];
    }
  }
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    if (16 * mt >= it.n_rows) break;
#pragma unroll
    for (int g = 0; g < VG; ++g) {
      if (mt + g > 0) __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < E; e += 2)
          *reinterpret_cast<float2*>(&om[w][lc][E * (4 * lr + i) + e]) =
              make_float2(o[mt][g][e][i], o[mt][g][e + 1][i]);
      __syncthreads();
      for (int x = tid; x < 16 * (DG / 4); x += 256) {
        const int row = x / (DG / 4), d = 4 * (x - row * (DG / 4));
        if (16 * mt + row >= it.n_rows) continue;
        float M = -__builtin_inff(), L = 0.0f;
#pragma unroll
        for (int v = 0; v < 4; ++v) M = fmaxf(M, sm[v][16 * mt + row]);
        float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int v = 0; v < 4; ++v) {
          const float mv = sm[v][16 * mt + row];
          if (mv == -__builtin_inff()) continue;
          const float f = __builtin_amdgcn_exp2f(mv - M);
          L += f * sl[v][16 * mt + row];
          const float4 y = *reinterpret_cast<const float4*>(&om[v][row][d]);
          acc.x = __builtin_fmaf(f, y.x, acc.x);
          acc.y = __builtin_fmaf(f, y.y, acc.y);
          acc.z = __builtin_fmaf(f, y.z, acc.z);
          acc.w = __builtin_fmaf(f, y.w, acc.w);
        }
        const int64_t pr = it.part_row + 16 * mt + row;
        *reinterpret_cast<float4*>(P.part + pr * D + 128 * g + d) = acc;
        if (g == 0 && d == 0) {
          P.ml[2 * pr] = M;
          P.ml[2 * pr + 1] = L;
        }
      }
    }
  }
}

// Whether a kTile item holds P in two parts.  In bf16 one part (8 bits) would
// round as coarsely as the output; in fp16 (11 bits, what the prefill kernels
// round P to) one is enough, and a third of the PV work: 128 sequences on 8 x
// 32768 x 128 take 128 us with two parts, 108 with one.
template <typename T>
constexpr bool kTwoParts = T::id == Bf16::id;

// kTile: 64 keys of K and V at a time in LDS for the four waves, the next tile
// on its way through registers.  V operands are transposing LDS reads: a group of
// 16 lanes takes 4 keys of 16 dims, which is the key order of P.
template <typename T, int D, int MT, bool CAUSAL, typename Shared>
__device__ void rows_tile_item(const RowsParams& P, const Item& it, Shared& sh) {
  constexpr int NKS = D / 32, ND = D / 16;
  constexpr int VS = v_row_bytes(D);
  const int tid = threadIdx.x;
  const int lane = tid & 63;
  const int lr = lane >> 4;
  const int lc = lane & 15;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  if (it.n_keys <= 0) {
    for (int r = tid; r < it.n_rows; r += 256) {
      P.ml[2 * (it.part_row + r)] = -__builtin_inff();
      P.ml[2 * (it.part_row + r) + 1] = 0.0f;
    }
    return;
  }
  const int wr0 = 16 * MT * w;  // first row of this wave in the item
  const bool active = wr0 < it.n_rows;

  u32x4 qb[MT][NKS];
  int lim[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    const int r = it.row0 + min(wr0 + 16 * mt + lc, it.n_rows - 1);
    const uint16_t* qrow =
        reinterpret_cast<const uint16_t*>(P.q) + q_offset(P, it.kvh, it.seq_rows, r);
#pragma unroll
    for (int ks = 0; ks < NKS; ++ks) qb[mt][ks] = load16(qrow + 32 * ks + 8 * lr);
    lim[mt] = CAUSAL ? it.limit + r % P.s_q : 0;
  }

  const __amdgpu_buffer_rsrc_t krs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(it.k), short(0), int(uint32_t(it.n_keys - 1) * it.kss + 2 * D), 0x00020000);
  const __amdgpu_buffer_rsrc_t vrs = __builtin_amdgcn_make_buffer_rsrc(
      const_cast<uint16_t*>(it.v), short(0), int(uint32_t(it.n_keys - 1) * it.vss + 2 * D), 0x00020000);
  // this wave stages 16 of the tile's 64 rows
  using Part = Tile<D, 16>;
  const Part kpart(lane, it.kss), vpart(lane, it.vss);
  u32x4 kr[Part::NL], vr[Part::NL];
  auto load_tile = [&](int j0) INLINE {
    kpart.load_at(krs, uint32_t(j0 + 16 * w) * it.kss, kr);
    vpart.load_at(vrs, uint32_t(j0 + 16 * w) * it.vss, vr);
  };
  auto store_tile = [&](unsigned char* stage) INLINE {
    kpart.store(stage + w * Part::BYTES, kr);
    unsigned char* vl = stage + 4 * Part::BYTES + 16 * w * VS;
#pragma unroll
    for (int i = 0; i < Part::NL; ++i) {
      const int f = 64 * i + lane, r = f / Part::NCH, c = f - r * Part::NCH;
      *reinterpret_cast<u32x4*>(vl + r * VS + 16 * c) = vr[i];
    }
  };

  // o[mt][n]: lane (lc, lr) holds row lc, dims 16 n + 4 lr + i
  f32x4 o[MT][ND];
  float m[MT], mp[MT], l[MT];
#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    m[mt] = -__builtin_inff();
    mp[mt] = 0.0f;
    l[mt] = 0.0f;
#pragma unroll
    for (int n = 0; n < ND; ++n) o[mt][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
  }
  const float c = P.scale_log2;

  // 32 keys of a tile: from local key j0, rows 32 h .. of the stage
  auto block = [&](int j0, const unsigned char* stage, int h) INLINE {
    const bool edge = CAUSAL ? j0 + 31 > it.limit : j0 + 32 > it.n_keys;
    f32x4 st[MT][2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) st[mt][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int ks = 0; ks < NKS; ++ks) {
        const u32x4 a = Part::operand(stage + (2 * h + u) * Part::BYTES, 0, lc, lr, ks);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) st[mt][u] = mfma_qk<T>(a, qb[mt][ks], st[mt][u]);
      }
    }
    u32x4 ph[MT], pl[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      f32x4(&s)[2] = st[mt];
      if (edge) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = j0 + 16 * u + 4 * lr + i;
            if ((CAUSAL && j > lim[mt]) || j >= it.n_keys) s[u][i] = -__builtin_inff();
          }
      }
      // the lanes of a row compare their own keys; they only exchange to move it
      float bm = max8(s[0], s[1]) * c;
      if (__ballot(bm > m[mt] + kSlack) != 0) {
        bm = fmaxf(bm, __shfl_xor(bm, 16, 64));
        bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
        const float mn = fmaxf(m[mt], bm);
        mp[mt] = mn == -__builtin_inff() ? 0.0f : mn;
        const float al = __builtin_amdgcn_exp2f(m[mt] - mp[mt]);
        m[mt] = mn;
        l[mt] *= al;
#pragma unroll
        for (int n = 0; n < ND; ++n) o[mt][n] *= al;
      }
      float p[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        p[j] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j >> 2][j & 3], c, -mp[mt]));
      l[mt] += ((p[0] + p[1]) + (p[2] + p[3])) + ((p[4] + p[5]) + (p[6] + p[7]));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        ph[mt][j] = pack2<T>(p[2 * j], p[2 * j + 1]);
        pl[mt][j] = 0;
        if constexpr (kTwoParts<T>)
          pl[mt][j] = pack2<T>(__builtin_fmaf(lo_of<T>(ph[mt][j]), -1.0f, p[2 * j]),
                               __builtin_fmaf(hi_of<T>(ph[mt][j]), -1.0f, p[2 * j + 1]));
      }
    }
    const unsigned char* vl = stage + 4 * Part::BYTES + (32 * h + 4 * lr + (lc >> 2)) * VS + 8 * (lc & 3);
    bool bad = false;
    if (CAUSAL && edge) {  // as in rows_item
#pragma unroll
      for (int n = 0; n < ND; ++n) {
        const u32x4 a = v_operand(vl + 32 * n, 16 * VS);
#pragma unroll
        for (int x = 0; x < 4; ++x) bad |= any_nonfinite<T>(a[x]);
      }
      bad = __ballot(bad) != 0;
      if (bad) add_nonfinite<T, MT, ND>(it, j0, lane, ph, pl, lim, o);
    }
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      u32x4 a = v_operand(vl + 32 * n, 16 * VS);
      if (CAUSAL && bad) {
#pragma unroll
        for (int x = 0; x < 4; ++x) a[x] = finite_only<T>(a[x]);
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        o[mt][n] = mfma_qk<T>(a, ph[mt], o[mt][n]);
        if constexpr (kTwoParts<T>) o[mt][n] = mfma_qk<T>(a, pl[mt], o[mt][n]);
      }
    }
  };

  const int nt = (it.n_keys + kTileKeys - 1) / kTileKeys;
  load_tile(0);
  store_tile(sh.kv[0]);
  __syncthreads();
  for (int t = 0; t < nt; ++t) {
    // rows behind the last tile read 0 and are not used
    load_tile(kTileKeys * (t + 1));
    if (active) {
      block(kTileKeys * t, sh.kv[t & 1], 0);
      if (kTileKeys * t + 32 < it.n_keys) block(kTileKeys * t + 32, sh.kv[t & 1], 1);
    }
    store_tile(sh.kv[(t + 1) & 1]);
    __syncthreads();
  }

#pragma unroll
  for (int mt = 0; mt < MT; ++mt) {
    l[mt] += __shfl_xor(l[mt], 16, 64);
    l[mt] += __shfl_xor(l[mt], 32, 64);
    const int row = wr0 + 16 * mt + lc;
    if (row >= it.n_rows) continue;
    const int64_t pr = it.part_row + row;
#pragma unroll
    for (int n = 0; n < ND; ++n)
      *reinterpret_cast<f32x4*>(P.part + pr * D + 16 * n + 4 * lr) = o[mt][n];
    if (lr == 0) {
      P.ml[2 * pr] = m[mt];
      P.ml[2 * pr + 1] = l[mt];
    }
  }
}

__device__ inline int clamped_len(const RowsParams& P, int b) {
  return P.lens ? max(0, min(P.lens[b], P.s_c)) : P.s_c;
}

constexpr int kUnit = 128;  // keys: one round of the four waves

struct OwnPlan {
  int total;  // units of all own caches
  int per;    // units of an item
};

__device__ inline int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Units of the sequences before each lane's, of b0 .. b0 + 63, and of all of these.
__device__ inline int own_scan(const RowsParams& P, int b0, int& chunk) {
  const int lane = threadIdx.x & 63, b = b0 + lane;
  const int mine = b < P.batch ? (clamped_len(P, b) + kUnit - 1) / kUnit * P.kv_heads * P.n_rto : 0;
  int incl = mine;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  chunk = __builtin_amdgcn_readlane(incl, 63);
  return incl - mine;
}

// The plan of a call; `write`: leaves it for the second launch, plan[0] = per,
// plan[1 + b] = units before sequence b.
__device__ inline OwnPlan own_plan(const RowsParams& P, bool write) {
  OwnPlan p;
  p.total = 0;
  for (int b0 = 0; b0 < P.batch; b0 += 64) {
    int chunk;
    const int before = own_scan(P, b0, chunk);
    if (write && threadIdx.x < 64 && b0 + int(threadIdx.x) < P.batch)
      P.plan[1 + b0 + threadIdx.x] = p.total + before;
    p.total += chunk;
  }
  p.per = uniform(max(1, (p.total + P.n_own - 1) / P.n_own));
  if (write && threadIdx.x == 0) P.plan[0] = p.per;
  return p;
}

// The sequence that unit u belongs to, and the units before it.
__device__ inline int own_find(const RowsParams& P, int u, int& before) {
  int base = 0;
  for (int b0 = 0;; b0 += 64) {
    int chunk;
    const int mine = base + own_scan(P, b0, chunk);
    if (u < base + chunk || b0 + 64 >= P.batch) {
      // the last sequence that starts at or before u is not empty: the next
      // one starts behind u
      const uint64_t at = __ballot(mine <= u && b0 + int(threadIdx.x & 63) < P.batch);
      const int last = 63 - __builtin_clzll(at);
      before = __builtin_amdgcn_readlane(mine, last);
      return b0 + last;
    }
    base += chunk;
  }
}

// First row in part / ml of what item x leaves of triple t (kv head, row tile)
// of sequence b: items and triples are in one order, so x + their number differ.
__device__ inline int64_t own_part_row(const RowsParams& P, int64_t x, int b, int t) {
  return P.own_row0 + (x + int64_t(b) * P.kv_heads * P.n_rto + t) * P.own_rows;
}

template <typename T, int D, int FORM, bool CAUSAL, bool SCORES, typename Shared>
__device__ inline void run_item(const RowsParams& P, const Item& it, Shared& sh) {
  if constexpr (FORM >= kTile)
    rows_tile_item<T, D, FORM - kTile, CAUSAL>(P, it, sh);
  else
    rows_item<T, D, FORM, CAUSAL, SCORES>(P, it, sh);
}

// Workgroups: n_own_wg (a multiple of 8) for the own caches, in form OF, which
// take longer to start; then the prefix items ((kv head, key range), row tile) in
// form PF (0: none).
template <typename T, int D, int PF, int OF, bool CAUSAL, bool SCORES>
__global__ __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(D > 128 ? 1 : 2)))
void rows_kernel(const RowsParams P) {
  __shared__ RowsShared<D, (PF >= kTile || OF >= kTile)> sh;
  Item it;
  it.seq_rows = P.group * P.s_q;
  it.raw = nullptr;
  it.raw_row = 0;
  int x = blockIdx.x;
  if (PF > 0 && x >= P.n_own_wg) {
    x -= P.n_own_wg;
    // The row tiles of one (kv head, key range) follow each other on one XCD
    // (workgroup i runs on XCD i % 8), so its L2 serves all but the first.
    const int y = x >> 3, rt = y % P.n_rt;
    const int unit = (y / P.n_rt) * 8 + (x & 7);
    if (unit >= P.kv_heads * P.n_sp) return;
    const int split = unit % P.n_sp;
    it.kvh = unit / P.n_sp;
    const int R = P.batch * it.seq_rows;
    const int j0 = split * P.chunk_p;
    it.k = reinterpret_cast<const uint16_t*>(P.kp) + it.kvh * P.kp_sh + int64_t(j0) * P.kp_ss;
    it.v = reinterpret_cast<const uint16_t*>(P.vp) + it.kvh * P.vp_sh + int64_t(j0) * P.vp_ss;
    it.kss = uint32_t(P.kp_ss) * 2u;
    it.vss = uint32_t(P.vp_ss) * 2u;
    it.n_keys = min(P.chunk_p, P.s_p - j0);
    it.limit = 0;
    it.row0 = rt * form_rows(PF);
    it.n_rows = min(form_rows(PF), R - it.row0);
    it.part_row = (int64_t(it.kvh) * P.n_sp + split) * R + it.row0;
    if constexpr (PF > 0) run_item<T, D, PF, false, false>(P, it, sh);
    return;
  }
  // Own caches: the units of 128 keys of all (sequence, kv head, row tile)
  // triples in a row, cut into equal ranges of P.n_own items, so lengths, known
  // on the device only, do not leave some workgroups with more than others.
  if (x >= P.n_own) return;
  const OwnPlan plan = own_plan(P, x == 0);
  const int per_seq = P.kv_heads * P.n_rto;
  int u = x * plan.per;
  const int u_end = min(u + plan.per, plan.total);
  if (u >= u_end) return;
  int before;
  int b = own_find(P, u, before);
  bool first = true;
  while (u < u_end) {
    const int len = uniform(clamped_len(P, b)), n = (len + kUnit - 1) / kUnit;
    if (u >= before + n * per_seq) {  // sequence b ends here
      before += n * per_seq;
      ++b;
      continue;
    }
    const int t = uniform((u - before) / n), k0 = u - before - t * n;
    const int n_here = min(n - k0, u_end - u);
    it.kvh = uniform(t / P.n_rto);
    const int r0 = (t - it.kvh * P.n_rto) * form_rows(OF);
    const int j0 = k0 * kUnit;
    it.k = reinterpret_cast<const uint16_t*>(P.k) + b * P.k_sb + it.kvh * P.k_sh + int64_t(j0) * P.k_ss;
    it.v = reinterpret_cast<const uint16_t*>(P.v) + b * P.v_sb + it.kvh * P.v_sh + int64_t(j0) * P.v_ss;
    it.kss = uint32_t(P.k_ss) * 2u;
    it.vss = uint32_t(P.v_ss) * 2u;
    it.n_keys = min(n_here * kUnit, len - j0);
    it.limit = len - P.s_q - j0;
    it.row0 = b * it.seq_rows + r0;
    it.n_rows = min(form_rows(OF), it.seq_rows - r0);
    it.part_row = own_part_row(P, x, b, t);
    if constexpr (SCORES) {  // s_q == 1: rows are the heads of the group
      it.raw_row = P.raw_row;
      it.raw = P.raw + (int64_t(b) * P.heads + it.kvh * P.group + r0) * P.raw_row + j0;
    }
    if (!first) __syncthreads();  // LDS of the range before
    first = false;
    run_item<T, D, OF, CAUSAL, SCORES>(P, it, sh);
    u += n_here;
  }
}

template <typename T, bool OUT_F32>
__device__ inline void store_one(void* o, int64_t off, float r) {
  if constexpr (OUT_F32) {
    reinterpret_cast<float*>(o)[off] = r;
  } else {
    reinterpret_cast<uint16_t*>(o)[off] = T::from_float(r);
  }
}

// Where the splits of row rr of (sequence b, kv head kvh) lie in part / ml:
// n_sp of the prefix, then n - n_sp of its own cache.
struct RowSplits {
  int n, n_sp;
  int64_t prefix, prefix_step, own, own_step;
  __device__ RowSplits(const RowsParams& P, int b, int kvh, int rr) {
    const int seq_rows = P.group * P.s_q;
    n = n_sp = P.n_sp;
    prefix_step = int64_t(P.batch) * seq_rows;
    prefix = int64_t(kvh) * P.n_sp * prefix_step + int64_t(b) * seq_rows + rr;
    own = 0;
    own_step = P.own_rows;
    const int units = P.n_own > 0 ? (clamped_len(P, b) + kUnit - 1) / kUnit : 0;
    if (units > 0) {
      const int rt = rr / P.own_rows, t = kvh * P.n_rto + rt;
      const int per = P.plan[0], u0 = P.plan[1 + b] + t * units;
      const int x0 = u0 / per, x1 = (u0 + units - 1) / per;
      n += x1 - x0 + 1;
      own = own_part_row(P, x0, b, t) + rr - rt * P.own_rows;
    }
  }
  __device__ int64_t at(int s) const {
    return s < n_sp ? prefix + s * prefix_step : own + (s - n_sp) * own_step;
  }
};

// Output row rr of (b, kvh): O = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s
// over its splits, by one workgroup.  Splits without a score above -inf leave
// no O.
template <typename T, bool OUT_F32, int D>
__device__ void combine_row(const RowsParams& P, int b, int kvh, int rr) {
  constexpr int TPR = D / 4;    // threads per split row, 4 elements each
  constexpr int G = 256 / TPR;  // split groups
  __shared__ float fs[kRowsMaxSplit];
  __shared__ float red[8];
  __shared__ __align__(16) float acc_g[G][D];
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const RowSplits sp(P, b, kvh, rr);
  const int ns = sp.n;
  float mx = -__builtin_inff();
  for (int s = tid; s < ns; s += 256) {
    const float ms = P.ml[2 * sp.at(s)];
    fs[s] = ms;
    mx = fmaxf(mx, ms);
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
  if (lane == 0) red[w] = mx;
  __syncthreads();
  const float M = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
  float L = 0.0f;
  for (int s = tid; s < ns; s += 256) {
    const float ms = fs[s];
    const float f = ms == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(ms - M);
    fs[s] = f;
    L += f * P.ml[2 * sp.at(s) + 1];
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) L += __shfl_xor(L, off, 64);
  if (lane == 0) red[4 + w] = L;
  __syncthreads();
  L = (red[4] + red[5]) + (red[6] + red[7]);

  const int g = tid / TPR, c = tid - g * TPR;
  if (g < G) {
    float a0 = 0.0f, a1 = 0.0f, a2 = 0.0f, a3 = 0.0f;
    for (int s = g; s < ns; s += G) {
      const float f = fs[s];
      if (f == 0.0f) continue;
      const float4 x = *reinterpret_cast<const float4*>(P.part + sp.at(s) * D + 4 * c);
      a0 = __builtin_fmaf(f, x.x, a0);
      a1 = __builtin_fmaf(f, x.y, a1);
      a2 = __builtin_fmaf(f, x.z, a2);
      a3 = __builtin_fmaf(f, x.w, a3);
    }
    *reinterpret_cast<float4*>(&acc_g[g][4 * c]) = float4{a0, a1, a2, a3};
  }
  __syncthreads();
  const int hg = rr / P.s_q, i = rr - hg * P.s_q;
  const int64_t off = b * P.o_sb + int64_t(kvh * P.group + hg) * P.o_sh + int64_t(i) * P.o_ss;
  for (int d = tid; d < D; d += 256) {
    float acc = 0.0f;
#pragma unroll
    for (int q = 0; q < G; ++q) acc += acc_g[q][d];
    // no score above -inf: 0; l = NaN (a NaN or +inf score) stays NaN
    store_one<T, OUT_F32>(P.o, off + d, L == 0.0f ? 0.0f : acc / L);
  }
}

template <typename T, bool OUT_F32, int D>
__global__ __launch_bounds__(256) void rows_combine_kernel(const RowsParams P) {
  const int seq_rows = P.group * P.s_q;
  int x = blockIdx.x;
  const int rr = x % seq_rows;
  x /= seq_rows;
  combine_row<T, OUT_F32, D>(P, x / P.kv_heads, x % P.kv_heads, rr);
}

constexpr int kWeightKeys = 1024;  // keys of a weight workgroup, 4 per thread

// Second launch of decode_accumulate, grid (key blocks + group, B * kv heads):
// the first key blocks add the weights of kWeightKeys keys, the others merge
// one head's output each.
template <typename T, bool OUT_F32, int D>
__global__ __launch_bounds__(256) void rows_weights_kernel(const RowsParams P, int n_kb) {
  __shared__ float sM[kMaxHeads], sR[kMaxHeads];
  const int b = blockIdx.y / P.kv_heads, kvh = blockIdx.y % P.kv_heads;
  if (int(blockIdx.x) >= n_kb) {
    combine_row<T, OUT_F32, D>(P, b, kvh, int(blockIdx.x) - n_kb);
    return;
  }
  const int len = clamped_len(P, b);
  const int j0 = int(blockIdx.x) * kWeightKeys;
  if (j0 >= len) return;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  for (int g = w; g < P.group; g += 4) {  // (M, 1 / L) of each head
    const RowSplits sp(P, b, kvh, g);
    float M = -__builtin_inff();
    for (int s = lane; s < sp.n; s += 64) M = fmaxf(M, P.ml[2 * sp.at(s)]);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) M = fmaxf(M, __shfl_xor(M, off, 64));
    float L = 0.0f;
    for (int s = lane; s < sp.n; s += 64) {
      const int64_t pr = sp.at(s);
      const float ms = P.ml[2 * pr];
      if (ms != -__builtin_inff()) L += __builtin_amdgcn_exp2f(ms - M) * P.ml[2 * pr + 1];
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) L += __shfl_xor(L, off, 64);
    if (lane == 0) {
      sM[g] = M == -__builtin_inff() ? 0.0f : M;
      sR[g] = L == 0.0f ? 0.0f : 1.0f / L;
    }
  }
  __syncthreads();
  const float* raw = P.raw + (int64_t(b) * P.heads + kvh * P.group) * P.raw_row;
  const float* in = P.w_in + b * P.wi_sb + kvh * P.wi_sh;
  float* out = P.w_out + b * P.wo_sb + kvh * P.wo_sh;
  const int j = j0 + 4 * tid;  // rows of raw are whole 16 bytes
  if (j >= len) return;
  float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
  for (int g = 0; g < P.group; ++g) {
    const f32x4 x = *reinterpret_cast<const f32x4*>(raw + g * P.raw_row + j);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[i] += sR[g] * __builtin_amdgcn_exp2f(__builtin_fmaf(x[i], P.scale_log2, -sM[g]));
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (j + i < len) out[j + i] = in[j + i] + acc[i];
}

template <typename T, int D, int PF, int OF, bool CAUSAL>
void launch_prefix_k(const RowsParams& p, hipStream_t st) {
  hipLaunchKernelGGL((rows_kernel<T, D, PF, OF, CAUSAL, false>), dim3(p.n_items), dim3(256), 0, st, p);
}

template <typename T, int D, bool CAUSAL>
void launch_prefix_f(const RowsParams& p, hipStream_t st) {
  if constexpr (D <= 128) {
    if (p.own_form == kTile + 2)
      return p.prefix_form == kTile + 2 ? launch_prefix_k<T, D, kTile + 2, kTile + 2, CAUSAL>(p, st)
                                        : launch_prefix_k<T, D, kTile + 1, kTile + 2, CAUSAL>(p, st);
    if (p.prefix_form == kTile + 2) return launch_prefix_k<T, D, kTile + 2, kOwn + 1, CAUSAL>(p, st);
    if (p.prefix_form == kTile + 1) return launch_prefix_k<T, D, kTile + 1, kOwn + 1, CAUSAL>(p, st);
  }
  launch_prefix_k<T, D, kOwn + 1, kOwn + 1, CAUSAL>(p, st);
}

template <typename T, bool OUT_F32, int D>
hipError_t launch_prefix_d(const RowsParams& p, hipStream_t st) {
  if (p.n_items > 0) {
    if (p.s_q == 1) launch_prefix_f<T, D, false>(p, st);
    else launch_prefix_f<T, D, true>(p, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL((rows_combine_kernel<T, OUT_F32, D>),
                     dim3(p.batch * p.heads * p.s_q), dim3(256), 0, st, p);
  return hipGetLastError();
}

template <typename T, bool OUT_F32, int D>
hipError_t launch_accumulate_d(const RowsParams& p, hipStream_t st) {
  if (p.n_items > 0) {
    hipLaunchKernelGGL((rows_kernel<T, D, 0, kOwn + 1, false, true>), dim3(p.n_items), dim3(256), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  const int n_kb = (p.s_c + kWeightKeys - 1) / kWeightKeys;
  hipLaunchKernelGGL((rows_weights_kernel<T, OUT_F32, D>),
                     dim3(n_kb + p.group, p.batch * p.kv_heads), dim3(256), 0, st, p, n_kb);
  return hipGetLastError();
}

template <typename T, bool OUT_F32>
hipError_t launch_rows_t(const RowsParams& p, bool accumulate, int D, hipStream_t st) {
#define MSA_ROWS_D(DD)                                                      \
  if (D == DD)                                                              \
    return accumulate ? launch_accumulate_d<T, OUT_F32, DD>(p, st)          \
                      : launch_prefix_d<T, OUT_F32, DD>(p, st);
  MSA_ROWS_D(64)
  MSA_ROWS_D(96)
  MSA_ROWS_D(128)
  MSA_ROWS_D(256)
  MSA_ROWS_D(512)
#undef MSA_ROWS_D
  return hipErrorInvalidValue;
}

}  // namespace

// us of a call, bf16, by form.
// Prefix 8 x 65536 x 128:   16 rows   24   32   48   64   96
//   kOwn + 1                54   61   61  106   96  182
//   kTile + 1               53   54   54   55   57   77
//   kTile + 2               55   55   55   58   60   65
// and 32 x 4096 x 96 with 4 rows: kOwn + 1 18.5, kTile + 1 19.1 (most waves of a
// kTile item of few rows only load).
// Own caches 8 x 8 x 4096 x 128 with 8 / 16 / 20 / 32 rows: kOwn + 1 36 / 40 / 59 /
// 62, kTile + 2 34 / 36 / 36 / 38; with 16 rows, 4 x 32 x 200 x 96 behind 1000 shared
// keys, 17 / 20.
// Above 128 dims O of a kTile item does not fit the registers; raw scores are kOwn's.
void rows_forms(RowsParams& p, int64_t rows, int64_t seq_rows, int D, bool scores) {
  const bool tiles = D <= 128 && !scores;
  p.own_form = tiles && seq_rows > 16 ? kTile + 2 : kOwn + 1;
  p.prefix_form = !tiles || rows <= 16 ? kOwn + 1 : rows <= 64 ? kTile + 1 : kTile + 2;
  p.prefix_rows = form_rows(p.prefix_form);
  p.own_rows = int(seq_rows < form_rows(p.own_form) ? seq_rows : form_rows(p.own_form));
}

hipError_t launch_rows(const RowsParams& p, bool accumulate, int dtype, int out_dtype, int D,
                       hipStream_t st) {
  const bool f32 = out_dtype == 3;
  if (dtype == Bf16::id)
    return f32 ? launch_rows_t<Bf16, true>(p, accumulate, D, st)
               : launch_rows_t<Bf16, false>(p, accumulate, D, st);
  return f32 ? launch_rows_t<F16, true>(p, accumulate, D, st)
             : launch_rows_t<F16, false>(p, accumulate, D, st);
}

}  // namespace msa
