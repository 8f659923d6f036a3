// Draws from rows of float32 logits with temperature, top-k, top-p and min-p, from given uniform numbers; several draws may take the
// same row.  With x the row, m its largest logit, T the temperature and e_i = exp((x_i - m) / T):
//   * T <= 0: the lowest index of m;
//   * top-k keeps x_i >= the k-th largest logit; top-p then keeps x_i >= t for the largest t at which the kept mass reaches
//     top_p times the mass that top-k left; min-p keeps e_i >= min_p (both beside the largest logit, which always stays).  Equal
//     logits are kept or left out together;
//   * the token is the first index at which the running kept mass exceeds u times the kept mass.
// The log-probability is x_token - m - ln sum_i exp(x_i - m), at temperature 1 and over the whole row.  NaN is no logit (as
// -infinity); a row without any finite or infinite logit gives token 0 with a log-probability of -infinity.
//
// Masses are sums of 64-bit numbers: with 200,000 tokens of like probability the borders between tokens lie 5e-6 of the mass apart and
// sums in 32 bits are 1e-6 off, so that every few draws would name a neighbour.  Sums are taken in a fixed order.
#include "common.cuh"

namespace ftk {

constexpr int kDrawThreads = 1024;

struct DrawParams {
  const float* logits;
  long long stride;
  int n_rows, vocab;
  const int32_t* rows;
  const float* temperature;
  const int32_t* top_k;
  const float* top_p;
  const float* min_p;
  const float* u;
  int32_t* out;
  float* logprobs;
};

// Logits in an order-preserving integer form: key 0 stands for NaN and -infinity.
__device__ __forceinline__ float clean(float x) { return x != x ? -INFINITY : x + 0.f; }  // (-0 is 0)
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x == -INFINITY) return 0u;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  if (k == 0u) return -INFINITY;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ double block_sum64(double v, double* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = scratch[threadIdx.x & 31];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
  return t;
}

__global__ void __launch_bounds__(kDrawThreads) draw_kernel(DrawParams p) {
  pdl_wait();
  pdl_trigger();
  __shared__ double scratch[32];
  __shared__ double prefix[kDrawThreads];
  __shared__ uint32_t best;
  __shared__ int first, last;
  const int r = blockIdx.x, V = p.vocab, tid = threadIdx.x;
  const int row = p.rows ? p.rows[r] : r;
  if (row < 0 || row >= p.n_rows) {
    if (tid == 0) {
      p.out[r] = -1;
      if (p.logprobs) p.logprobs[r] = -INFINITY;
    }
    return;
  }
  const float* x = p.logits + (size_t)row * p.stride;
  if (tid == 0) {
    best = 0u;
    first = V;
    last = -1;
  }
  __syncthreads();
  uint32_t mine = 0u;
  for (int i = tid; i < V; i += kDrawThreads) mine = max(mine, order_key(clean(x[i])));
  atomicMax(&best, mine);
  __syncthreads();
  const uint32_t top_key = best;
  const float top = of_key(top_key);
  const float t = p.temperature[r];
  int token = 0;
  if (top_key != 0u) {
    const double inv_t = t > 0.f ? 1.0 / (double)t : 1.0;
    auto mass_of = [&](float v) -> double { return v == top ? 1.0 : exp(((double)v - (double)top) * inv_t); };
    // mass and number of logits whose keys reach `from`
    auto count = [&](uint32_t from) -> double {
      double c = 0.0;
      for (int i = tid; i < V; i += kDrawThreads) c += order_key(clean(x[i])) >= from ? 1.0 : 0.0;
      return block_sum64(c, scratch);
    };
    auto mass = [&](uint32_t from) -> double {
      double c = 0.0;
      for (int i = tid; i < V; i += kDrawThreads) {
        const float v = clean(x[i]);
        if (order_key(v) >= from) c += mass_of(v);
      }
      return block_sum64(c, scratch);
    };
    if (!(t > 0.f)) {
      for (int i = tid; i < V; i += kDrawThreads)
        if (order_key(clean(x[i])) == top_key) {
          atomicMin(&first, i);
          break;
        }
      __syncthreads();
      token = first;
    } else {
      uint32_t limit = 1u;  // (key 0 is never drawn)
      const int k = p.top_k[r];
      if (k > 0 && k < V) {
        uint32_t lo = 0u, hi = top_key;
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo + 1u) / 2u;
          if (count(mid) >= (double)k) lo = mid; else hi = mid - 1u;
        }
        limit = max(limit, lo);
      }
      const float tp = p.top_p[r];
      if (tp < 1.f) {
        const double need = (double)tp * mass(limit);
        uint32_t lo = limit, hi = top_key;
        while (lo < hi) {
          const uint32_t mid = lo + (hi - lo + 1u) / 2u;
          if (mass(mid) >= need) lo = mid; else hi = mid - 1u;
        }
        limit = lo;
      }
      const float mp = p.min_p[r];
      const double least = mp > 0.f ? fmin(log((double)mp), 0.0) : -INFINITY;
      auto kept = [&](float v) -> double {
        if (order_key(v) < limit) return 0.0;
        if (v != top && !(((double)v - (double)top) * inv_t >= least)) return 0.0;
        return mass_of(v);
      };
      // a run of indices per thread, and the running mass in front of it
      const int per = (V + kDrawThreads - 1) / kDrawThreads, i0 = min(V, tid * per), i1 = min(V, i0 + per);
      double c = 0.0;
      int newest = -1;
      for (int i = i0; i < i1; ++i) {
        const double e = kept(clean(x[i]));
        c += e;
        if (e > 0.0) newest = i;
      }
      if (newest >= 0) atomicMax(&last, newest);
      prefix[tid] = c;
      __syncthreads();
      if (tid == 0) {
        double run = 0.0;
        for (int i = 0; i < kDrawThreads; ++i) {
          const double s = prefix[i];
          prefix[i] = run;
          run += s;
        }
        scratch[0] = run;
      }
      __syncthreads();
      const double target = (double)p.u[r] * scratch[0];
      double run = prefix[tid];
      if (run + c > target) {
        for (int i = i0; i < i1; ++i) {
          run += kept(clean(x[i]));
          if (run > target) {
            atomicMin(&first, i);
            break;
          }
        }
      }
      __syncthreads();
      token = first < V ? first : last;  // (u of one and more: the last kept one)
    }
  }
  if (p.logprobs) {
    double c = 0.0;
    if (top_key != 0u)
      for (int i = tid; i < V; i += kDrawThreads) {
        const float v = clean(x[i]);
        if (v != -INFINITY) c += v == top ? 1.0 : exp((double)v - (double)top);
      }
    c = block_sum64(c, scratch);
    const float v = clean(x[token]);
    if (tid == 0) p.logprobs[r] = top_key == 0u ? -INFINITY : (float)((v == top ? 0.0 : (double)v - (double)top) - log(c));
  }
  if (tid == 0) p.out[r] = token;
}

}  // namespace ftk

using namespace ftk;

extern "C" int ftk_sample_draws(const float* logits, long long row_stride, int n_rows, int vocab, const int32_t* rows, int n_draws,
                                const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p, const float* u,
                                int32_t* out, float* logprobs, void* stream) {
  FTK_REQUIRE(n_rows >= 0 && n_draws >= 0 && vocab >= 1 && vocab <= (1 << 24) && row_stride >= vocab, "sample_draws: bad sizes rows=%d draws=%d vocab=%d", n_rows, n_draws, vocab);
  if (n_draws == 0) return 0;
  FTK_REQUIRE(n_rows >= 1 && logits && temperature && top_k && top_p && min_p && u && out, "sample_draws: null pointer");
  FTK_REQUIRE(rows || n_draws <= n_rows, "sample_draws: %d draws from %d rows", n_draws, n_rows);
  DrawParams p{logits, row_stride, n_rows, vocab, rows, temperature, top_k, top_p, min_p, u, out, logprobs};
  note_variant("draws: one block each");
  FTK_LAUNCH(draw_kernel, n_draws, kDrawThreads, 0, (cudaStream_t)stream, p);
  FTK_LAUNCH_CHECK("sample_draws");
  return 0;
}
