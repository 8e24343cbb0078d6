// Beam search's choice: of the beams x vocabulary continuations of each
// request the `keep` with the largest score_b + log softmax(logits_b)[v],
// the first `beams` of them that do not end, and their token histories.
//
// One pass over the logits. Each row (request, beam) is cut into slices, one
// CTA each, that keep a running maximum and sum of exponentials per thread
// and a short buffer of the elements above the slice's keep-th best so far; a
// second kernel (one CTA per request) joins the slices' sums, scores their
// sorted lists and merges them. Bound: HBM for many rows, latency for few.
//
// Order: by score in 64 bits, equal scores by logit, then by beam and token
// (lowest first). Within a row the score grows with the logit, so a slice
// only needs the logit and the token. Exponentials are 32-bit and their sums
// 64-bit: the scores of different beams are then right to about 1e-8, which
// keeps near ties in order.
#include <cuda_runtime.h>

#include "paged.h"

namespace rai {

namespace {

constexpr int kThreads = 256;
constexpr int kBufCap = 2 * kThreads * 8;  // most elements of a step, twice

// A float's bits in the order of its value (-0 as +0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t b = __float_as_uint(x + 0.f);
  return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t o) {
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ uint64_t key_of(float x, int token) {
  return ((uint64_t)ordered(x) << 32) | (0xffffffffu - (uint32_t)token);
}

// e^(x - m), where x = m also counts when both are infinite: a row with
// infinite logits shares its mass among them, a row of -inf among all.
__device__ __forceinline__ float weight(float x, float m) { return x == m ? 1.f : expf(x - m); }

template <int DT>
__device__ __forceinline__ float to_f32(uint32_t w, int half) {
  if constexpr (DT == kF16) return __half2float(__ushort_as_half((uint16_t)(w >> (16 * half))));
  else return __uint_as_float(half ? w & 0xffff0000u : w << 16);
}

struct Slice {
  float max;
  int pad;
  double sum;
};

__host__ __device__ inline size_t slice_bytes(int keep) { return sizeof(Slice) + (size_t)keep * 8; }

// Sorts n = 2^k keys, largest first.
__device__ __forceinline__ void bitonic(uint64_t* a, int n) {
  for (int size = 2; size <= n; size <<= 1)
    for (int step = size >> 1; step; step >>= 1) {
      __syncthreads();
      for (int i = threadIdx.x; i < n / 2; i += kThreads) {
        const int lo = 2 * step * (i / step) + i % step, hi = lo + step;
        const bool down = (lo & size) == 0;
        const uint64_t x = a[lo], y = a[hi];
        if ((x < y) == down) a[lo] = y, a[hi] = x;
      }
    }
  __syncthreads();
}

// The `keep` largest of buf[0 .. n), sorted, in front; keys are unique.
__device__ __forceinline__ void prune(uint64_t* buf, int n, int keep) {
  int size = 64;
  while (size < n) size <<= 1;
  for (int i = n + threadIdx.x; i < size; i += kThreads) buf[i] = 0;
  bitonic(buf, size);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) beam_slice_kernel(BeamArgs a, int slices, int len) {
  constexpr int V = DT == kF32 ? 4 : 8;  // elements of 16 bytes
  constexpr int kU = 8 / V;              // vectors of a step
  constexpr int kE = DT == kF32 ? 4 : 2;
  __shared__ uint64_t buf[kBufCap];
  __shared__ uint64_t tops[kThreads];
  __shared__ int count;
  __shared__ float wm[kThreads / 32];
  __shared__ double wsum[kThreads / 32];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int row = blockIdx.y, slice = blockIdx.x;
  const int begin = slice * len, end = min(a.vocab, begin + len);
  const char* src = static_cast<const char*>(a.logits) + (long long)row * a.row * kE;
  // Vector slots from the 16-byte boundary at or before the slice's start.
  const int off = (int)((reinterpret_cast<uintptr_t>(src + (long long)begin * kE) & 15) / kE);
  const int base = begin - off;
  if (threadIdx.x == 0) count = 0;
  float m = -INFINITY;
  double sum = 0.0;
  uint64_t bar = 0;  // keys at or above it are kept
  __syncthreads();
  for (int at = base; at < end; at += kThreads * V * kU) {
    float x[V * kU];
    bool whole[kU];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      const int e0 = at + (u * kThreads + threadIdx.x) * V;
      whole[u] = e0 >= begin && e0 + V <= end;
      if (whole[u]) {
        const uint4 w = __ldcs(reinterpret_cast<const uint4*>(src + (long long)e0 * kE));
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < V; ++i) {
          if constexpr (DT == kF32) x[u * V + i] = __uint_as_float(ws[i]);
          else x[u * V + i] = to_f32<DT>(ws[i / 2], i & 1);
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          x[u * V + i] = -INFINITY;
          if (e0 + i >= begin && e0 + i < end) {
            if constexpr (DT == kF32) x[u * V + i] = reinterpret_cast<const float*>(src)[e0 + i];
            else x[u * V + i] = to_f32<DT>(reinterpret_cast<const uint16_t*>(src)[e0 + i], 0);
          }
        }
      }
    }
    float top = -INFINITY;
    int there = 0;
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < V * kU; ++i) {
      const int e = at + (i / V * kThreads + threadIdx.x) * V + i % V;
      if (!(x[i] == x[i])) x[i] = -INFINITY;  // a NaN is not chosen
      if (e >= begin && e < end) {
        top = fmaxf(top, x[i]);
        ++there;
      }
    }
    if (there) {
      if (top > m) {
        sum *= (double)expf(m - top);
        m = top;
      }
      float part = 0.f;
#pragma unroll
      for (int i = 0; i < V * kU; ++i) {
        const int e = at + (i / V * kThreads + threadIdx.x) * V + i % V;
        if (e >= begin && e < end) part += weight(x[i], m);
      }
      sum += (double)part;
    }
    if (at == base) {
      // The keep-th largest of the threads' best is no larger than the
      // keep-th largest element: a first bar.
#pragma unroll
      for (int i = 0; i < V * kU; ++i) {
        const int e = at + (i / V * kThreads + threadIdx.x) * V + i % V;
        if (e >= begin && e < end) best = max(best, key_of(x[i], e));
      }
      tops[threadIdx.x] = best;
      bitonic(tops, kThreads);
      bar = tops[a.keep - 1];
    }
    const float bar_x = bar ? unordered((uint32_t)(bar >> 32)) : -INFINITY;
    if (there && top >= bar_x) {
#pragma unroll
      for (int i = 0; i < V * kU; ++i) {
        const int e = at + (i / V * kThreads + threadIdx.x) * V + i % V;
        if (e >= begin && e < end && x[i] >= bar_x) {
          const uint64_t k = key_of(x[i], e);
          if (k >= bar) buf[atomicAdd(&count, 1)] = k;
        }
      }
    }
    __syncthreads();
    const int n = count;
    if (n > kBufCap - kThreads * V * kU || n > 4 * a.keep + 64) {
      prune(buf, n, a.keep);
      bar = buf[a.keep - 1];
      if (threadIdx.x == 0) count = min(n, a.keep);
    }
    __syncthreads();
  }
  const int n = count;
  prune(buf, n, a.keep);
  // Join the threads' sums.
  float top = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if ((threadIdx.x & 31) == 0) wm[threadIdx.x >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, wm[w]);
  double s = sum == 0.0 ? 0.0 : sum * (double)weight(m, top);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if ((threadIdx.x & 31) == 0) wsum[threadIdx.x >> 5] = s;
  __syncthreads();
  char* out = static_cast<char*>(a.ws) + ((long long)row * slices + slice) * slice_bytes(a.keep);
  if (threadIdx.x == 0) {
    Slice r = {top, 0, 0.0};
    for (int w = 0; w < kThreads / 32; ++w) r.sum += wsum[w];
    *reinterpret_cast<Slice*>(out) = r;
  }
  for (int i = threadIdx.x; i < a.keep; i += kThreads)
    reinterpret_cast<uint64_t*>(out + sizeof(Slice))[i] = i < n ? buf[i] : 0;
}

struct Cand {
  double score;
  float logit;
  int flat;  // beam * vocab + token, -1: none
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) {
  if (a.flat < 0 || b.flat < 0) return b.flat < 0 && a.flat >= 0;
  if (a.score != b.score) return a.score > b.score;
  if (a.logit != b.logit) return a.logit > b.logit;
  return a.flat < b.flat;
}
__device__ __forceinline__ Cand shuffled(const Cand& c, int o) {
  Cand r;
  r.score = __shfl_xor_sync(~0u, c.score, o);
  r.logit = __shfl_xor_sync(~0u, c.logit, o);
  r.flat = __shfl_xor_sync(~0u, c.flat, o);
  return r;
}

constexpr int kMaxSlices = 16;

// One CTA per request, one thread per (beam, slice) list; each round takes
// the best of the lists' heads.
__global__ void __launch_bounds__(kMaxBeams * kMaxSlices) beam_merge_kernel(BeamArgs a, int slices) {
  __shared__ double lse[kMaxBeams];  // log of the sum beside the maximum
  __shared__ float tops[kMaxBeams];
  __shared__ Cand warp_best[kMaxBeams * kMaxSlices / 32];
  __shared__ Cand chosen[kMaxKeep];
  __shared__ int next[kMaxBeams];
  pdl_wait_prior();
  pdl_launch_dependents();
  const int req = blockIdx.x, lists = a.beams * slices, warps = blockDim.x >> 5;
  const size_t sb = slice_bytes(a.keep);
  const char* ws = static_cast<const char*>(a.ws) + (long long)req * lists * sb;
  if (threadIdx.x < a.beams) {
    const char* mine = ws + (long long)threadIdx.x * slices * sb;
    float top = -INFINITY;
    for (int i = 0; i < slices; ++i) top = fmaxf(top, reinterpret_cast<const Slice*>(mine + i * sb)->max);
    double sum = 0.0;
    for (int i = 0; i < slices; ++i) {
      const Slice s = *reinterpret_cast<const Slice*>(mine + i * sb);
      sum += s.sum * (s.max == top ? 1.0 : exp((double)s.max - (double)top));
    }
    tops[threadIdx.x] = top;
    lse[threadIdx.x] = log(sum);
  }
  __syncthreads();
  const int beam = threadIdx.x / slices;
  const bool real = (int)threadIdx.x < lists;
  const uint64_t* list = reinterpret_cast<const uint64_t*>(ws + (long long)threadIdx.x * sb + sizeof(Slice));
  float score = 0.f;
  if (real) {
    score = a.scores[req * a.beams + beam];
    if (!(score == score)) score = -INFINITY;
  }
  int at = 0;
  auto head = [&]() {
    Cand c = {0.0, 0.f, -1};
    if (!real || at >= a.keep) return c;
    const uint64_t k = list[at];
    if (!k) return c;
    c.logit = unordered((uint32_t)(k >> 32));
    c.flat = beam * a.vocab + (int)(0xffffffffu - (uint32_t)k);
    const double d = c.logit == tops[beam] ? 0.0 : (double)c.logit - (double)tops[beam];
    c.score = (double)score + (d - lse[beam]);
    return c;
  };
  Cand mine = head();
  for (int r = 0; r < a.keep; ++r) {
    Cand best = mine;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const Cand c = shuffled(best, o);
      if (before(c, best)) best = c;
    }
    if (warps > 1) {
      if ((threadIdx.x & 31) == 0) warp_best[threadIdx.x >> 5] = best;
      __syncthreads();
      for (int w = 0; w < warps; ++w)
        if (before(warp_best[w], best)) best = warp_best[w];
      __syncthreads();
    }
    if (threadIdx.x == 0) chosen[r] = best;
    if (best.flat >= 0 && best.flat == mine.flat) {
      ++at;
      mine = head();
    }
  }
  __syncthreads();
  for (int r = threadIdx.x; r < a.keep; r += blockDim.x) {
    const Cand c = chosen[r];
    const long long o = (long long)req * a.keep + r;
    const int b = c.flat < 0 ? -1 : c.flat / a.vocab;
    a.cand_score[o] = c.flat < 0 ? -INFINITY : (float)c.score;
    a.cand_beam[o] = b;
    a.cand_token[o] = c.flat < 0 ? -1 : c.flat - b * a.vocab;
  }
  if (threadIdx.x == 0) {
    int n = 0;
    for (int r = 0; r < a.keep && n < a.beams; ++r)
      if (chosen[r].flat >= 0 && chosen[r].flat % a.vocab != a.eos) next[n++] = r;
    for (; n < a.beams; ++n) next[n] = -1;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.beams; i += blockDim.x) {
    const long long o = (long long)req * a.beams + i;
    const bool some = next[i] >= 0;
    const Cand c = some ? chosen[next[i]] : Cand{};
    const int b = some ? c.flat / a.vocab : 0;
    a.score[o] = some ? (float)c.score : -INFINITY;
    a.parent[o] = some ? req * a.beams + b : -1;
    a.token[o] = some ? c.flat - b * a.vocab : -1;
  }
  if (!a.history) return;
  for (int i = 0; i < a.beams; ++i) {
    const long long o = (long long)req * a.beams + i;
    if (next[i] < 0) {
      if (threadIdx.x == 0) a.out_len[o] = 0;
      continue;
    }
    const Cand c = chosen[next[i]];
    const int b = c.flat / a.vocab;
    const long long p = (long long)req * a.beams + b;
    int n = a.hist_len[p];
    const bool fits = n >= 0 && n < a.hist_cap;
    if (!fits) n = min(max(n, 0), a.hist_cap);
    for (int x = threadIdx.x; x < n; x += blockDim.x) a.out_history[o * a.out_stride + x] = a.history[p * a.hist_stride + x];
    if (threadIdx.x == 0) {
      if (fits) a.out_history[o * a.out_stride + n] = c.flat - b * a.vocab;
      else atomicOr(a.err, kErrBadInput);
      a.out_len[o] = fits ? n + 1 : n;
    }
  }
}

int slices_of(int batch, int beams, int vocab) {
  // Enough CTAs for four on each SM, none with less than 2048 elements.
  const long long rows = (long long)batch * beams;
  long long n = (4ll * device_sm_count() + rows - 1) / rows;
  const long long most = (vocab + 2047) / 2048;
  n = n < most ? n : most;
  n = n < kMaxSlices ? n : kMaxSlices;
  return n < 1 ? 1 : (int)n;
}

}  // namespace

size_t beam_workspace(int batch, int beams, int vocab, int keep) {
  return (size_t)batch * beams * slices_of(batch, beams, vocab) * slice_bytes(keep);
}

cudaError_t beam_select(const BeamArgs& a, cudaStream_t s) {
  const int slices = slices_of(a.batch, a.beams, a.vocab);
  int len = (a.vocab + slices - 1) / slices;
  len = (len + 7) / 8 * 8;
  const dim3 grid(slices, a.batch * a.beams);
  cudaError_t e = a.dtype == kF32   ? launch_pdl(beam_slice_kernel<kF32>, grid, dim3(kThreads), 0, s, a, slices, len)
                  : a.dtype == kF16 ? launch_pdl(beam_slice_kernel<kF16>, grid, dim3(kThreads), 0, s, a, slices, len)
                                    : launch_pdl(beam_slice_kernel<kBF16>, grid, dim3(kThreads), 0, s, a, slices, len);
  if (e != cudaSuccess) return e;
  const int lists = a.beams * slices;
  return launch_pdl(beam_merge_kernel, dim3(a.batch), dim3((lists + 31) / 32 * 32), 0, s, a, slices);
}

}  // namespace rai
