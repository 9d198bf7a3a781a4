// Eviction from a cache: of the n keys of a sequence, the first `sinks`, the
// last `recent` and the best scored ones between them stay, `keep` in all, moved
// together in their order.
//
// select (one workgroup per (sequence, kv head)): the scores as unsigned keys
// whose order is the scores' (NaN on top, -0 equal to 0); the largest key T that
// at least `free` = keep - sinks - recent of them reach is found digit by digit
// (8 bits a pass, a histogram in LDS); then all above T stay and, of those equal
// to T, the first ones.  Positions are written in ascending order from a scan
// over the workgroup.
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

// Sum over the workgroup's threads before this one, and the total.
__device__ inline uint32_t scan_before(uint32_t x, uint32_t* wsum, uint32_t& total) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  uint32_t incl = x;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const uint32_t y = __shfl_up(incl, off, 64);
    if (lane >= off) incl += y;
  }
  __syncthreads();  // wsum of an earlier call has been read
  if (lane == 63) wsum[w] = incl;
  __syncthreads();
  uint32_t before = 0;
  total = 0;
#pragma unroll
  for (int v = 0; v < kSelectThreads / 64; ++v) {
    if (v < w) before += wsum[v];
    total += wsum[v];
  }
  return before + incl - x;
}

__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(const EvictParams P) {
  __shared__ uint32_t hist[256];
  __shared__ uint32_t wsum[kSelectThreads / 64];
  __shared__ uint32_t s_digit, s_left;
  const int tid = threadIdx.x;
  const int b = blockIdx.x / P.kv_heads, h = blockIdx.x - b * P.kv_heads;
  const int n = evict_len(P, b);
  int32_t* pos = P.pos + int64_t(blockIdx.x) * P.keep;
  if (h == 0 && tid == 0) P.new_lens[b] = min(n, P.keep);
  if (n <= P.keep) {
    for (int i = tid; i < P.keep; i += kSelectThreads) pos[i] = i < n ? i : -1;
    return;
  }
  // candidates: keys [lo, hi)
  const int lo = P.sinks, hi = n - P.recent;
  const float* sc = P.scores + b * P.s_sb + h * P.s_sh;
  const uint32_t want = uint32_t(P.keep - P.sinks - P.recent);
  for (int i = tid; i < P.sinks; i += kSelectThreads) pos[i] = i;
  for (int i = tid; i < P.recent; i += kSelectThreads) pos[P.keep - P.recent + i] = hi + i;
  if (want == 0) return;
  // the want-th largest key, digit by digit; left: how many of the keys that
  // share its leading digits are still to be taken
  uint32_t prefix = 0, left = want;
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    const uint32_t mask = shift == 24 ? 0u : 0xffffffffu << (shift + 8);
    for (int j = lo + tid; j < hi; j += kSelectThreads) {
      const uint32_t key = order_key(sc[j]);
      if ((key & mask) == prefix) atomicAdd(&hist[(key >> shift) & 255u], 1u);
    }
    __syncthreads();
    // thread d: keys with a digit above 255 - d
    const uint32_t mine = tid < 256 ? hist[255 - tid] : 0;
    uint32_t total;
    const uint32_t above = scan_before(mine, wsum, total);
    if (tid < 256 && above < left && above + mine >= left) {
      s_digit = 255 - tid;
      s_left = left - above;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    left = s_left;
  }
  // keys above the threshold, and the first `left` equal to it, in order
  int out = P.sinks;
  uint32_t ties = 0;
  for (int j0 = lo; j0 < hi; j0 += kSelectThreads) {
    const int j = j0 + tid;
    const uint32_t key = j < hi ? order_key(sc[j]) : 0;
    const bool eq = j < hi && key == prefix, gt = j < hi && key > prefix;
    uint32_t n_eq, n_in;
    const uint32_t eq_before = scan_before(eq, wsum, n_eq);
    const bool in = gt || (eq && ties + eq_before < left);
    const uint32_t before = scan_before(in, wsum, n_in);
    if (in) pos[out + before] = j;
    out += n_in;
    ties += n_eq;
  }
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
  hipLaunchKernelGGL(evict_select_kernel, dim3(bh), dim3(kSelectThreads), 0, st, p);
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
