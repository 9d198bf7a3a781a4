// Eviction from a cache: of the n keys of a sequence, the first `sinks`, the
// last `recent` and the best scored ones between them stay, `keep` in all, moved
// together in their order.
//
// The scores are taken as unsigned keys whose order is the scores' (NaN on top,
// -0 equal to 0); the largest key T that at least keep - sinks - recent of them
// reach is found digit by digit (11, 11 and 10 bits, a histogram in LDS); then all
// above T stay and, of those equal to T, the first ones.
// select: rows of up to 8192 scores, one workgroup each, the scores in registers.
// step 0 .. 3: longer rows in stretches, one workgroup each.  Step s takes digit
//   s - 1 from all the row's histograms of it (each workgroup for itself) and
//   counts digit s of its stretch; step 3 writes the positions, whose places
//   follow from how many keys of the earlier stretches stay, known from the
//   histograms.
// In both a wave has 64 contiguous keys at a time: ballots give the kept ones,
// lane i keeps the masks of the wave's i-th 64 keys, and one exchange between
// the waves gives the places.
//   Bound by latency, of the histograms' way from launch to launch and the scans:
//   8 x 8 heads x 65536 scores (17 MB) 8 + 13 + 12 + 20 us; select, 32 rows of 4113,
//   12 us.
// gather: the kept rows of K and V and their scores.  Bound by memory, each kept
//   row read and written once: 8 x 8 heads, 16384 of 65536 keys of 128 dims take
//   190 us for 1.07 GB (5.6 TB/s).

#include "msa_common.h"
#include "msa_kernels.h"

namespace msa {

#define INLINE __attribute__((always_inline))

namespace {

constexpr int kSelectThreads = 1024;

// Order of scores as unsigned integers: NaN above +inf, -0 as +0.
__device__ inline uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ INLINE inline int evict_len(const EvictParams& P, int b) {
  return P.lens ? max(0, min(P.lens[b], P.s)) : P.s;
}

constexpr int kWaves = kSelectThreads / 64;
constexpr int kBins = kEvictBins;

// x plus its value CTRL lanes away in the row of 16, 0 from outside it.  (Shuffles
// go through LDS, which 32 waves of a CU then wait for: with them the four steps of
// 64 rows x 65536 scores take 8 us more.)
template <int CTRL>
__device__ INLINE inline uint32_t add_from(uint32_t x) {
  return x + uint32_t(__builtin_amdgcn_update_dpp(0, int(x), CTRL, 0xf, 0xf, true));
}

// Sum over the wave, in every lane.
__device__ INLINE inline uint32_t wave_sum(uint32_t x) {
  x = add_from<0x128>(x);  // row_ror:8, 4, 2, 1
  x = add_from<0x124>(x);
  x = add_from<0x122>(x);
  x = add_from<0x121>(x);
  return (__builtin_amdgcn_readlane(x, 0) + __builtin_amdgcn_readlane(x, 16)) +
         (__builtin_amdgcn_readlane(x, 32) + __builtin_amdgcn_readlane(x, 48));
}

// Sum over the wave's lanes up to this one.
__device__ INLINE inline uint32_t wave_scan(uint32_t x) {
  const int row = (threadIdx.x >> 4) & 3;
  x = add_from<0x111>(x);  // row_shr:1, 2, 4, 8
  x = add_from<0x112>(x);
  x = add_from<0x114>(x);
  x = add_from<0x118>(x);
  const uint32_t a = __builtin_amdgcn_readlane(x, 15), b = a + __builtin_amdgcn_readlane(x, 31),
                 c = b + __builtin_amdgcn_readlane(x, 47);
  return x + (row == 0 ? 0u : row == 1 ? a : row == 2 ? b : c);
}

// Sum over the workgroup's threads before this one.
__device__ INLINE inline uint32_t scan_before(uint32_t x, uint32_t* wsum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const uint32_t incl = wave_scan(x);
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v)
    if (v < w) before += wsum[v];
  return before + incl - x;
}

// One key of each lane that has one into the histogram.  Scores crowd in few
// bins (a fifth may be 0): the first lane's bin is counted by ballot, the others
// by atomics.
__device__ INLINE inline void count(uint32_t* hist, bool has, uint32_t bin) {
  const uint64_t live = __ballot(has);
  if (live == 0) return;
  const int leader = __builtin_ctzll(live);
  const uint32_t lead = __builtin_amdgcn_readlane(bin, leader);
  const bool same = has && bin == lead;
  const uint64_t group = __ballot(same);
  if ((int(threadIdx.x) & 63) == leader) atomicAdd(&hist[lead], uint32_t(__builtin_popcountll(group)));
  if (has && !same) atomicAdd(&hist[bin], 1u);
}

// The candidates of row (b, h): keys [lo, hi) of n, `want` of which stay.
struct Row {
  int n, lo, hi;
  uint32_t want;
  const float* sc;
  __device__ INLINE Row(const EvictParams& P, int b, int h) {
    n = evict_len(P, b);
    lo = P.sinks;
    hi = n - P.recent;
    want = uint32_t(P.keep - P.sinks - P.recent);
    sc = P.scores + b * P.s_sb + h * P.s_sh;
  }
};

// Largest digit that `left` keys reach, from the counts of bins 2047 - 2 t (top)
// and 2046 - 2 t (next) of thread t; left: those of that digit still to be taken.
__device__ INLINE inline uint32_t take_digit(uint32_t top, uint32_t next, uint32_t* wsum,
                                             uint32_t* out, uint32_t& left) {
  const uint32_t above = scan_before(top + next, wsum);
  if (above < left && above + top + next >= left) {
    const bool second = above + top < left;
    out[0] = kBins - 1 - 2 * threadIdx.x - second;
    out[1] = left - above - (second ? top : 0u);
  }
  __syncthreads();
  left = out[1];
  return out[0];
}

__device__ INLINE inline int shift_of(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__device__ INLINE inline uint32_t digits_of(int d) { return d == 2 ? 1023u : 2047u; }
__device__ INLINE inline uint32_t known_of(int d) {
  return d == 0 ? 0u : d == 1 ? 0xffe00000u : 0xfffffc00u;
}

// The 64-key rows [r0, r1) of a wave (row r: keys 64 r .. 64 r + 63 of the score
// row), R of them in registers at a time.
template <int R>
struct Rows {
  const Row& row;
  int r0, r1, lane;
  uint32_t keys[R];

  __device__ INLINE Rows(const Row& row, int r0, int r1) : row(row), r0(r0), r1(r1) {
    lane = threadIdx.x & 63;
    load(r0);
  }
  __device__ INLINE void load(int c0) {
    float x[R];
#pragma unroll
    for (int i = 0; i < R; ++i) x[i] = row.sc[min(64 * (c0 + i) + lane, row.n - 1)];
#pragma unroll
    for (int i = 0; i < R; ++i) keys[i] = order_key(x[i]);
  }
  // Counts digit d of the candidates that share the known digits of prefix.
  __device__ INLINE void histogram(uint32_t* hist, int d, uint32_t prefix) {
    for (int c0 = r0; c0 < r1; c0 += R) {
      if (c0 > r0) load(c0);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int j = 64 * (c0 + i) + lane;
        count(hist, c0 + i < r1 && j >= row.lo && j < row.hi && (keys[i] & known_of(d)) == prefix,
              (keys[i] >> shift_of(d)) & digits_of(d));
      }
    }
    if (r1 - r0 > R) load(r0);
  }
  // Masks of the keys that stay in any case (sinks, recent ones, above T) and
  // of those equal to T, lane i for row c0 + i; at most 64 rows.
  __device__ INLINE void masks(int c0, uint32_t T, uint64_t& gt, uint64_t& eq) {
    gt = eq = 0;
#pragma unroll 1  // most waves take one turn, and fetching the code of eight cost 3 us
    for (int q = 0; q < 64 / R; ++q) {
      if (c0 + q * R >= r1) break;
      if (r1 - r0 > R) load(c0 + q * R);
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const int r = c0 + q * R + i, j = 64 * r + lane;
        const bool has = j >= row.lo && j < row.hi;
        const uint64_t g = __ballot(r < r1 && (has ? keys[i] > T : j < row.n));
        const uint64_t e = __ballot(r < r1 && has && keys[i] == T && row.want > 0);
        if (lane == q * R + i) {
          gt = g;
          eq = e;
        }
      }
    }
  }
  // Positions of the kept keys of the workgroup's waves: all above T and, of the
  // equal ones, the first `left` of the row; eq0, out: equal and kept keys of the
  // row before the workgroup's.
  __device__ INLINE void place(uint32_t T, uint32_t left, uint32_t eq0, uint32_t out, uint32_t* wgt,
                               uint32_t* weq, int32_t* pos) {
    const int w = threadIdx.x >> 6;
    uint64_t gt = 0, eq = 0;
    uint32_t n_gt = 0, n_eq = 0;
    for (int c0 = r0; c0 < r1; c0 += 64) {
      masks(c0, T, gt, eq);
      n_gt += wave_sum(__builtin_popcountll(gt));
      n_eq += wave_sum(__builtin_popcountll(eq));
    }
    if (lane == 0) {
      wgt[w] = n_gt;
      weq[w] = n_eq;
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < kWaves - 1; ++v) {
      const uint32_t g = wgt[v], e = weq[v];
      out += v < w ? g + min(e, left - min(left, eq0)) : 0u;
      eq0 += v < w ? e : 0u;
    }
    for (int c0 = r0; c0 < r1; c0 += 64) {
      if (r1 - r0 > 64) masks(c0, T, gt, eq);  // else still there
      uint32_t ne = __builtin_popcountll(eq), e_before = wave_scan(ne);
      const uint32_t e_total = __builtin_amdgcn_readlane(e_before, 63);
      e_before += eq0 - ne;
      const uint32_t take = min(ne, left - min(left, e_before));
      for (; ne > take; --ne) eq &= ~(uint64_t(1) << (63 - __builtin_clzll(eq)));
      const uint64_t m = gt | eq;
      const uint32_t k = __builtin_popcountll(m), k_before = wave_scan(k);
      const uint32_t at = out + k_before - k;
      for (int i = 0; i < min(64, r1 - c0); ++i) {
        const uint64_t mi = uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(m), i))) |
                            uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(m >> 32), i))) << 32;
        const uint32_t ai = __builtin_amdgcn_readlane(at, i);
        if ((mi >> lane) & 1)
          pos[ai + __builtin_popcountll(mi & ((uint64_t(1) << lane) - 1))] = 64 * (c0 + i) + lane;
      }
      out += __builtin_amdgcn_readlane(k_before, 63);
      eq0 += e_total;
    }
  }
};

// A row of at most keep keys keeps them all.
__device__ INLINE inline void keep_all(const EvictParams& P, int n, int32_t* pos) {
  for (int i = threadIdx.x; i < P.keep; i += kSelectThreads) pos[i] = i < n ? i : -1;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams P) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wsum[3][kWaves], wgt[kWaves], weq[kWaves], found[3][2];
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / P.kv_heads, h = blockIdx.x - b * P.kv_heads;
  const Row row(P, b, h);
  int32_t* pos = P.pos + int64_t(blockIdx.x) * P.keep;
  if (h == 0 && tid == 0) P.new_lens[b] = min(row.n, P.keep);
  if (row.n <= P.keep) return keep_all(P, row.n, pos);
  const int rows = (row.n + 63) / 64, per = (rows + kWaves - 1) / kWaves;
  Rows<8> mine(row, min(rows, w * per), min(rows, w * per + per));
  uint32_t T = 0xffffffffu, left = 0;  // want = 0: none is taken
  if (row.want > 0) {
    T = 0;
    left = row.want;
#pragma unroll
    for (int d = 0; d < 3; ++d) {
      hist[tid] = hist[tid + kSelectThreads] = 0;
      __syncthreads();
      mine.histogram(hist, d, T);
      __syncthreads();
      T |= take_digit(hist[kBins - 1 - 2 * tid], hist[kBins - 2 - 2 * tid], wsum[d], found[d], left)
           << shift_of(d);
    }
  }
  mine.place(T, left, 0, 0, wgt, weq, pos);
}

// grid (stretches, B * kv heads)
template <int STEP>
__global__ __launch_bounds__(kSelectThreads) __attribute__((amdgpu_waves_per_eu(8)))
void evict_step_kernel(const EvictParams P) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wsum[kWaves], wgt[kWaves], weq[kWaves], found[2];
  __shared__ uint32_t s_above[kEvictMaxStretch], s_eq[kEvictMaxStretch];
  const int tid = threadIdx.x;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int x = blockIdx.x, b = blockIdx.y / P.kv_heads, h = blockIdx.y - b * P.kv_heads;
  const Row row(P, b, h);
  int32_t* pos = P.pos + int64_t(blockIdx.y) * P.keep;
  if (STEP == 3 && x == 0 && h == 0 && tid == 0) P.new_lens[b] = min(row.n, P.keep);
  if (row.n <= P.keep) {
    if (STEP == 3 && x == 0) keep_all(P, row.n, pos);
    return;
  }
  if (STEP < 3 && row.want == 0) return;
  // of this score row: (T, left) after each digit; keys above it of each stretch
  uint32_t* state = P.state + int64_t(blockIdx.y) * (6 + 3 * kEvictMaxStretch);
  uint32_t* above = state + 6;
  uint32_t T = 0, left = row.want, above_before = 0;
  if (STEP > 1 && row.want > 0) {
    T = state[2 * (STEP - 2)];
    left = state[2 * (STEP - 2) + 1];
  }
  if (STEP == 3 && row.want > 0 && tid < x) above_before = above[tid] + above[kEvictMaxStretch + tid];
  const uint32_t* last = nullptr;  // the row's histograms of the digit before
  if (STEP > 0 && row.want > 0) {
    last = P.hist + (int64_t(STEP - 1) * gridDim.y + blockIdx.y) * P.n_stretch * kBins;
    if (tid < kEvictMaxStretch) s_above[tid] = 0;
    uint32_t top = 0, next = 0;
    uint2 part[kEvictMaxStretch];
#pragma unroll
    for (int y = 0; y < kEvictMaxStretch; ++y)
      part[y] = y < P.n_stretch ? *reinterpret_cast<const uint2*>(last + y * kBins + kBins - 2 - 2 * tid)
                                : make_uint2(0u, 0u);
#pragma unroll
    for (int y = 0; y < kEvictMaxStretch; ++y) {
      top += part[y].y;
      next += part[y].x;
    }
    const int digit = int(take_digit(top, next, wsum, found, left));
    T |= uint32_t(digit) << shift_of(STEP - 1);
    // keys above the digit: of every stretch before the last step, of this one
    // otherwise
    const bool t_above = kBins - 1 - 2 * tid > digit, n_above = kBins - 2 - 2 * tid > digit;
    const auto add_above = [&](int y, uint2 p) INLINE {
      const uint32_t sum = wave_sum((t_above ? p.y : 0u) + (n_above ? p.x : 0u));
      if ((tid & 63) == 0 && sum) atomicAdd(&s_above[y], sum);
    };
    if constexpr (STEP == 3) {
#pragma unroll
      for (int y = 0; y < kEvictMaxStretch; ++y)
        if (y < P.n_stretch) add_above(y, part[y]);
    } else {
      uint2 p = part[0];
#pragma unroll
      for (int y = 1; y < kEvictMaxStretch; ++y)
        if (y == x) p = part[y];
      add_above(x, p);
    }
    __syncthreads();
    if (STEP < 3 && tid == 0) above[(STEP - 1) * kEvictMaxStretch + x] = s_above[x];
    if (STEP < 3 && x == 0 && tid == 0) {
      state[2 * (STEP - 1)] = T;
      state[2 * (STEP - 1) + 1] = left;
    }
  }
  // this stretch's rows of 64 keys
  const int rows = (row.n + 63) / 64, s0 = min(rows, x * (P.stretch / 64));
  const int s1 = min(rows, s0 + P.stretch / 64), per = (s1 - s0 + kWaves - 1) / kWaves;
  Rows<8> mine(row, min(s1, s0 + w * per), min(s1, s0 + w * per + per));
  if constexpr (STEP < 3) {
    hist[tid] = hist[tid + kSelectThreads] = 0;
    __syncthreads();
    mine.histogram(hist, STEP, T);
    __syncthreads();
    uint2* o = reinterpret_cast<uint2*>(
        P.hist + ((int64_t(STEP) * gridDim.y + blockIdx.y) * P.n_stretch + x) * kBins);
    o[tid] = make_uint2(hist[2 * tid], hist[2 * tid + 1]);
  } else {
    const int j0 = 64 * s0;
    uint32_t eq0 = 0, out = min(j0, row.lo) + max(0, min(j0, row.n) - row.hi);
    if (row.want > 0) {
      if (tid < x) {
        s_eq[tid] = last[tid * kBins + (T & 1023u)];
        s_above[tid] += above_before;
      }
      __syncthreads();
#pragma unroll
      for (int y = 0; y < kEvictMaxStretch - 1; ++y) {
        const uint32_t a = s_above[y], e = s_eq[y];
        out += y < x ? a + min(e, left - min(left, eq0)) : 0u;
        eq0 += y < x ? e : 0u;
      }
    } else {
      T = 0xffffffffu;
      left = 0;
    }
    mine.place(T, left, eq0, out, wgt, weq, pos);
  }
}

// Units of U bytes of the kept rows, grid (units, B * kv heads).
template <typename U>
__global__ __launch_bounds__(256) void evict_gather_kernel(const EvictParams P) {
  const int b = blockIdx.y / P.kv_heads, h = blockIdx.y - b * P.kv_heads;
  const int64_t x = int64_t(blockIdx.x) * 256 + threadIdx.x;
  const int i = int(x / P.upr), u = int(x - int64_t(i) * P.upr);
  if (i >= P.keep) return;
  const int j = P.pos[int64_t(blockIdx.y) * P.keep + i];
  U kx{}, vx{};
  if (j >= 0) {
    kx = *(reinterpret_cast<const U*>(static_cast<const char*>(P.k) + b * P.k_sb + h * P.k_sh + j * P.k_ss) + u);
    vx = *(reinterpret_cast<const U*>(static_cast<const char*>(P.v) + b * P.v_sb + h * P.v_sh + j * P.v_ss) + u);
  }
  *(reinterpret_cast<U*>(static_cast<char*>(P.ko) + b * P.ko_sb + h * P.ko_sh + i * P.ko_ss) + u) = kx;
  *(reinterpret_cast<U*>(static_cast<char*>(P.vo) + b * P.vo_sb + h * P.vo_sh + i * P.vo_ss) + u) = vx;
  if (u == 0)
    P.scores_out[b * P.so_sb + h * P.so_sh + i] =
        j >= 0 ? P.scores[b * P.s_sb + h * P.s_sh + j] : 0.0f;
}

}  // namespace

hipError_t launch_evict(const EvictParams& p, hipStream_t st) {
  const uint32_t bh = uint32_t(p.batch) * p.kv_heads;
  const dim3 t(kSelectThreads), gs(p.n_stretch, bh);
  if (p.n_stretch == 0) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(bh), t, 0, st, p);
  } else {
    hipLaunchKernelGGL(evict_step_kernel<0>, gs, t, 0, st, p);
    hipLaunchKernelGGL(evict_step_kernel<1>, gs, t, 0, st, p);
    hipLaunchKernelGGL(evict_step_kernel<2>, gs, t, 0, st, p);
    hipLaunchKernelGGL(evict_step_kernel<3>, gs, t, 0, st, p);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const dim3 g(uint32_t((int64_t(p.keep) * p.upr + 255) / 256), bh);
  if (p.unit == 16)
    hipLaunchKernelGGL(evict_gather_kernel<u32x4>, g, dim3(256), 0, st, p);
  else
    hipLaunchKernelGGL(evict_gather_kernel<uint16_t>, g, dim3(256), 0, st, p);
  return hipGetLastError();
}

}  // namespace msa
