// Eviction from a cache: of the n keys of a sequence, the first `sinks`, the
// last `recent` and the best scored ones between them stay, `keep` in all, moved
// together in their order.
//
// select (one workgroup per (sequence, kv head)): the scores as unsigned keys
// whose order is the scores' (NaN on top, -0 equal to 0); the largest key T that
// at least keep - sinks - recent of them reach is found digit by digit (11, 11
// and 10 bits, a histogram in LDS); then all above T stay and, of those equal to
// T, the first ones.  Each of the 16 waves has a contiguous part of the keys, 64 at
// a time, so ballots give the order inside a wave and one exchange between the
// waves gives the rest.  Up to 65536 keys stay in registers over the passes (one
// read of the scores); longer rows are read again each pass.
// gather: the kept rows of K and V and their scores.  Bound by memory: each kept
// row is read and written once.

#include "msa_common.h"
#include "msa_kernels.h"

namespace msa {

namespace {

constexpr int kSelectThreads = 1024;

// Order of scores as unsigned integers: NaN above +inf, -0 as +0.
__device__ inline uint32_t order_key(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = __float_as_uint(f + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ inline int evict_len(const EvictParams& P, int b) {
  return P.lens ? max(0, min(P.lens[b], P.s)) : P.s;
}

constexpr int kWaves = kSelectThreads / 64;
constexpr int kBins = 2048;

// Sum over the workgroup's threads before this one.
__device__ inline uint32_t scan_before(uint32_t x, uint32_t* wsum) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
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
__device__ inline void count(uint32_t* hist, bool has, uint32_t bin) {
  const uint64_t live = __ballot(has);
  if (live == 0) return;
  const int leader = __builtin_ctzll(live);
  const uint32_t lead = __builtin_amdgcn_readlane(bin, leader);
  const bool same = has && bin == lead;
  const uint64_t group = __ballot(same);
  if ((int(threadIdx.x) & 63) == leader) atomicAdd(&hist[lead], uint32_t(__builtin_popcountll(group)));
  if (has && !same) atomicAdd(&hist[bin], 1u);
}

// R: keys of a thread, in registers (R * 1024 >= the cache's length); 0: any
// length, read again each pass.
template <int R>
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams P) {
  __shared__ uint32_t hist[kBins];
  __shared__ uint32_t wsum[3][kWaves], wgt[kWaves], weq[kWaves];
  __shared__ uint32_t s_digit[3], s_left[3];
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int b = blockIdx.x / P.kv_heads, h = blockIdx.x - b * P.kv_heads;
  const int n = evict_len(P, b);
  int32_t* pos = P.pos + int64_t(blockIdx.x) * P.keep;
  if (h == 0 && tid == 0) P.new_lens[b] = min(n, P.keep);
  if (n <= P.keep) {
    for (int i = tid; i < P.keep; i += kSelectThreads) pos[i] = i < n ? i : -1;
    return;
  }
  // candidates: keys [lo, hi); wave w has rows of 64 from lo + 64 rows w on
  const int lo = P.sinks, hi = n - P.recent;
  const float* sc = P.scores + b * P.s_sb + h * P.s_sh;
  const uint32_t want = uint32_t(P.keep - P.sinks - P.recent);
  for (int i = tid; i < P.sinks; i += kSelectThreads) pos[i] = i;
  for (int i = tid; i < P.recent; i += kSelectThreads) pos[P.keep - P.recent + i] = hi + i;
  if (want == 0) return;
  const int rows = (hi - lo + kSelectThreads - 1) / kSelectThreads;
  const int first = lo + 64 * rows * w + lane;
  uint32_t keys[R > 0 ? R : 1];
  if constexpr (R > 0) {
#pragma unroll
    for (int r = 0; r < R; ++r)
      keys[r] = r < rows && first + 64 * r < hi ? order_key(sc[first + 64 * r]) : 0u;
  }
  // f(key, whether there is one, its position) for this lane's keys in order, a
  // wave's rows at a time
  auto each = [&](auto f) __attribute__((always_inline)) {
    if constexpr (R > 0) {
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (r < rows) f(keys[r], first + 64 * r < hi, first + 64 * r);
    } else {
#pragma unroll 8
      for (int r = 0; r < rows; ++r) {
        const int j = first + 64 * r;
        f(j < hi ? order_key(sc[j]) : 0u, j < hi, j);
      }
    }
  };
  // the want-th largest key, digit by digit; left: how many of the keys that
  // share its leading digits are still to be taken
  uint32_t prefix = 0, left = want;
#pragma unroll
  for (int d = 0; d < 3; ++d) {
    const int shift = d == 0 ? 21 : d == 1 ? 10 : 0;
    const uint32_t mask = d == 0 ? 0u : d == 1 ? 0xffe00000u : 0xfffffc00u;
    const uint32_t digits = d == 2 ? 1023u : 2047u;
    hist[tid] = hist[tid + kSelectThreads] = 0;
    __syncthreads();
    each([&](uint32_t key, bool has, int) {
      count(hist, has && (key & mask) == prefix, (key >> shift) & digits);
    });
    __syncthreads();
    // thread t: bins 2047 - 2 t and 2046 - 2 t, from the largest down
    const uint32_t top = hist[kBins - 1 - 2 * tid], next = hist[kBins - 2 - 2 * tid];
    const uint32_t above = scan_before(top + next, wsum[d]);
    if (above < left && above + top + next >= left) {
      const bool second = above + top < left;
      s_digit[d] = kBins - 1 - 2 * tid - second;
      s_left[d] = left - above - (second ? top : 0u);
    }
    __syncthreads();
    prefix |= s_digit[d] << shift;
    left = s_left[d];
  }
  // keys above the threshold, and the first `left` equal to it, in order
  uint32_t n_gt = 0, n_eq = 0;
  each([&](uint32_t key, bool has, int) {
    n_gt += __builtin_popcountll(__ballot(has && key > prefix));
    n_eq += __builtin_popcountll(__ballot(has && key == prefix));
  });
  if (lane == 0) {
    wgt[w] = n_gt;
    weq[w] = n_eq;
  }
  __syncthreads();
  uint32_t eq = 0, out = P.sinks;  // equal ones and kept ones before this row
  for (int v = 0; v < w; ++v) {
    out += wgt[v] + min(weq[v], left - min(left, eq));
    eq += weq[v];
  }
  const uint64_t below = (uint64_t(1) << lane) - 1;
  each([&](uint32_t key, bool has, int j) {
    const uint64_t beq = __ballot(has && key == prefix);
    const bool in = has && (key > prefix ||
                            (key == prefix && eq + __builtin_popcountll(beq & below) < left));
    const uint64_t bin = __ballot(in);
    if (in) pos[out + __builtin_popcountll(bin & below)] = j;
    out += __builtin_popcountll(bin);
    eq += __builtin_popcountll(beq);
  });
}

// 16-byte units of the kept rows (or U bytes where rows are not aligned): grid
// (units, B * kv heads).
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
  if (p.s <= 8 * kSelectThreads)
    hipLaunchKernelGGL(evict_select_kernel<8>, dim3(bh), dim3(kSelectThreads), 0, st, p);
  else if (p.s <= 64 * kSelectThreads)
    hipLaunchKernelGGL(evict_select_kernel<64>, dim3(bh), dim3(kSelectThreads), 0, st, p);
  else
    hipLaunchKernelGGL(evict_select_kernel<0>, dim3(bh), dim3(kSelectThreads), 0, st, p);
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
