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
//
// A cluster of up to eight CTAs takes a draw: a thread has a run of neighbouring logits, kept in shared memory from the one pass over
// memory.  A threshold is searched for by the number or the mass of the logits above it, with three candidates a pass; a logit's
// exponential is taken only where it lies between the last candidates, and when at most kListed logits do, each of them is tried.
// What bounds it: for one draw the passes one after the other (a barrier of the cluster and a trip through its shared memory each, about
// a microsecond); for many the exponentials in 64 bits (13 operations each at 64 an SM and cycle).
#include "common.cuh"

namespace ftk {

constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32;
constexpr int kListed = 256;      // logits that are tried one by one
constexpr int kMostRun = 105;     // logits of a thread's run that shared memory has room for

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
  int cluster, run;  // CTAs a draw; logits of a thread's run (odd: neighbouring threads' runs begin in different banks)
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

// 2^(j / 32)
__device__ const double kPowers[32] = {
    1.00000000000000000e+00, 1.02189714865411663e+00, 1.04427378242741375e+00, 1.06714040067682370e+00,
    1.09050773266525769e+00, 1.11438674259589243e+00, 1.13878863475669156e+00, 1.16372485877757748e+00,
    1.18920711500272103e+00, 1.21524735998046896e+00, 1.24185781207348400e+00, 1.26905095719173322e+00,
    1.29683955465100964e+00, 1.32523664315974132e+00, 1.35425554693689265e+00, 1.38390988196383202e+00,
    1.41421356237309515e+00, 1.44518080697704665e+00, 1.47682614593949935e+00, 1.50916442759342284e+00,
    1.54221082540794074e+00, 1.57598084510788650e+00, 1.61049033194925428e+00, 1.64575547815396495e+00,
    1.68179283050742900e+00, 1.71861929812247793e+00, 1.75625216037329945e+00, 1.79470907500310717e+00,
    1.83400808640934243e+00, 1.87416763411029996e+00, 1.91520656139714740e+00, 1.95714412417540018e+00,
};
// e^x for x <= 0: x = k ln 2 / 32 + r with k = 32 n + j the nearest, e^x = 2^n 2^(j / 32) e^r, |r| <= ln 2 / 64, where the series up to r^5 is
// within 2.3e-15; ln 2 / 32 in two parts, of which k times the first (36 bits) is exact.  Below e^-700: zero.
__device__ __forceinline__ double exp_down(double x, const double* powers) {
  if (!(x > -700.0)) return x != x ? x : 0.0;
  double k = fma(x, 4.61662413084468283841e+01, 6755399441055744.0);
  const int n = __double2loint(k);
  k -= 6755399441055744.0;
  double r = fma(k, -2.16608493924468348268e-02, x);
  r = fma(k, -5.14560924465533821524e-14, r);
  double q = fma(r, 1.0 / 120.0, 1.0 / 24.0);
  q = fma(q, r, 1.0 / 6.0);
  q = fma(q, r, 0.5);
  q = fma(q * r, r, r);
  const double t = powers[n & 31], y = fma(t, q, t);
  return __hiloint2double(__double2hiint(y) + ((n >> 5) << 20), __double2loint(y));
}

__device__ __forceinline__ uint32_t draw_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t draw_remote(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(draw_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ double remote_f64(uint32_t at) {
  double v;
  asm volatile("ld.shared::cluster.f64 %0, [%1];" : "=d"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t remote_u32(uint32_t at) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(at));
  return v;
}
__device__ __forceinline__ void draw_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

constexpr int kSums = 8;
struct DrawShared {
  double powers[32];
  double parts[kDrawWarps][kSums];  // the warps' sums
  double sums[2][kSums];            // the CTA's, for the cluster: in turns, so that one barrier a pass is enough
  double listed_mass[kListed];
  uint32_t listed[kListed];
  double result[kSums];             // the cluster's
  uint32_t own_key[2];              // the CTA's largest and smallest key
  int own_index[2];
  uint32_t keys[kDrawWarps], low_keys[kDrawWarps];
  int found, first;
};

template <int N>
struct SumCount {
  static constexpr int value = N;
};
using Sums1 = SumCount<1>;
using Sums8 = SumCount<8>;

template <bool STAGED>
__global__ void __launch_bounds__(kDrawThreads, 2) draw_kernel(const __grid_constant__ DrawParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) uint32_t staged[];  // the chunk's logits as keys
  __shared__ DrawShared sh;
  const int C = p.cluster, rank = blockIdx.x % C, draw = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, V = p.vocab;
  const int row = p.rows ? p.rows[draw] : draw;
  if (row < 0 || row >= p.n_rows) {  // (every CTA of the cluster)
    if (rank == 0 && tid == 0) {
      p.out[draw] = -1;
      if (p.logprobs) p.logprobs[draw] = -INFINITY;
    }
    return;
  }
  const int chunk = p.run * kDrawThreads, c0 = min(V, rank * chunk), n_here = min(V - c0, chunk);  // (rank * chunk < 2^31: the host checks)
  const float* x = p.logits + (size_t)row * p.stride + c0;
  if (tid < 32) sh.powers[tid] = kPowers[tid];
  if (tid == 0) {
    sh.found = 0x7fffffff;
    sh.first = 0x7fffffff;
  }
  // ---- the chunk comes in; its largest logit
  uint32_t top_key = 0u, low_key = 0xffffffffu;  // the largest logit, and the smallest above -infinity
  {
    auto note = [&](float v) -> uint32_t {
      const uint32_t k = order_key(clean(v));
      top_key = max(top_key, k);
      low_key = min(low_key, k - 1u);  // (0 wraps)
      return k;
    };
    if ((((uintptr_t)x) & 15) == 0) {
      const float4* x4 = reinterpret_cast<const float4*>(x);
      const int n4 = n_here >> 2;
      for (int i0 = 0; i0 < n4; i0 += 4 * kDrawThreads) {
        float4 v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + e * kDrawThreads + tid;
          if (i < n4) v[e] = __ldg(x4 + i);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = i0 + e * kDrawThreads + tid;
          if (i < n4) {
            if (STAGED) *reinterpret_cast<uint4*>(staged + 4 * i) = make_uint4(note(v[e].x), note(v[e].y), note(v[e].z), note(v[e].w));
            else note(v[e].x), note(v[e].y), note(v[e].z), note(v[e].w);
          }
        }
      }
      for (int i = 4 * n4 + tid; i < n_here; i += kDrawThreads) {
        const uint32_t k = note(x[i]);
        if (STAGED) staged[i] = k;
      }
    } else {
      for (int i0 = 0; i0 < n_here; i0 += 8 * kDrawThreads) {
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = i0 + e * kDrawThreads + tid;
          if (i < n_here) v[e] = __ldg(x + i);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int i = i0 + e * kDrawThreads + tid;
          if (i < n_here) {
            const uint32_t k = note(v[e]);
            if (STAGED) staged[i] = k;
          }
        }
      }
    }
    top_key = __reduce_max_sync(0xffffffffu, top_key);
    low_key = __reduce_min_sync(0xffffffffu, low_key);
  }
  if (lane == 0) {
    sh.keys[warp] = top_key;
    sh.low_keys[warp] = low_key;
  }
  __syncthreads();
  top_key = __reduce_max_sync(0xffffffffu, lane < kDrawWarps ? sh.keys[lane] : 0u);
  low_key = __reduce_min_sync(0xffffffffu, lane < kDrawWarps ? sh.low_keys[lane] : 0xffffffffu);
  if (C > 1) {
    if (tid == 0) {
      sh.own_key[0] = top_key;
      sh.own_key[1] = low_key;
    }
    draw_barrier();
    top_key = __reduce_max_sync(0xffffffffu, lane < C ? remote_u32(draw_remote(&sh.own_key[0], lane)) : 0u);
    low_key = __reduce_min_sync(0xffffffffu, lane < C ? remote_u32(draw_remote(&sh.own_key[1], lane)) : 0xffffffffu);
  }
  low_key += 1u;
  const float top = of_key(top_key), t = p.temperature[draw];
  const int i0 = min(n_here, tid * p.run), i1 = min(n_here, i0 + p.run);
  auto at = [&](int i) -> uint32_t { return STAGED ? staged[i] : order_key(clean(__ldg(x + i))); };
  int turn = 0;
  // N sums over the cluster, the same in every thread
  auto cluster_sums = [&](auto nc, double (&v)[kSums]) {
    constexpr int N = decltype(nc)::value;
#pragma unroll
    for (int s = 0; s < N; ++s) {
      v[s] = warp_sum64(v[s]);
      if (lane == 0) sh.parts[warp][s] = v[s];
    }
    __syncthreads();
    if (tid < N) {
      double sum = 0.0;
#pragma unroll
      for (int w = 0; w < kDrawWarps; ++w) sum += sh.parts[w][tid];
      sh.sums[turn][tid] = sum;
    }
    if (C > 1) draw_barrier(); else __syncthreads();
    if (C > 1) {
      if (warp == 0) {  // lane 8 c + s: sums s of CTAs c and c + 4
        const int s = lane & 7, c = lane >> 3;
        double sum = 0.0;
        if (s < N) {
          if (c < C) sum = remote_f64(draw_remote(&sh.sums[turn][s], c));
          if (c + 4 < C) sum += remote_f64(draw_remote(&sh.sums[turn][s], c + 4));
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (lane < N) sh.result[lane] = sum;
      }
      __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < N; ++s) v[s] = C > 1 ? sh.result[s] : sh.sums[turn][s];
    turn ^= 1;
  };
  int token = 0;
  double whole_row = -1.0;  // the row's mass at temperature 1, where it is known
  if (top_key != 0u) {
    if (!(t > 0.f)) {  // the lowest index of the largest logit
      for (int i = i0; i < i1; ++i)
        if (at(i) == top_key) {
          atomicMin(&sh.first, c0 + i);
          break;
        }
      __syncthreads();
      if (C > 1) {
        draw_barrier();
        int lowest = 0x7fffffff;
        for (int c = 0; c < C; ++c) lowest = min(lowest, (int)remote_u32(draw_remote(&sh.first, c)));
        token = lowest;
      } else {
        token = sh.first;
      }
    } else {
      const double inv_t = 1.0 / (double)t;
      auto mass_of = [&](uint32_t k) -> double { return k == top_key ? 1.0 : exp_down(((double)of_key(k) - (double)top) * inv_t, sh.powers); };
      double whole = -1.0;  // the mass of the whole row at this temperature, where it was summed up
      // The largest key from `lo` on at which the number (by_mass: the mass) of the logits that reach it is `need` (by_mass: `need` of what
      // reaches `lo`) or more; `lo` where not even that has as many.
      auto search = [&](bool by_mass, uint32_t lo, double need) -> uint32_t {
        uint32_t hi = top_key;
        double above = 0.0;    // of the logits above `hi`
        double inside = 1e30;  // logits between
        bool by_key = false;
        for (int pass = 0; (lo < hi && inside > kListed) || pass == 0; ++pass) {
          // Three candidates between: by value, as logits spread like their values do (close below the largest where some lie far away, masked
          // ones say); by key, which ends whatever they are, where the part far away was the one, and every third time.
          uint32_t q1, q2, q3;
          const uint32_t gap = hi - lo;
          const float a = of_key(lo), b = of_key(hi);
          q1 = lo + gap / 4u + (gap < 4u), q2 = lo + gap / 2u + (gap & 1u), q3 = hi - gap / 4u;
          const bool wide = !(b - a <= 64.f * t);
          if (!by_key && pass % 3 != 2 && b < INFINITY) {
            q1 = order_key(clean(wide ? b - 30.f * t : a + 0.25f * (b - a)));
            q2 = order_key(clean(wide ? b - 10.f * t : a + 0.5f * (b - a)));
            q3 = order_key(clean(wide ? b - 4.f * t : a + 0.75f * (b - a)));
          }
          q1 = min(max(q1, lo + 1u), max(hi, lo + 1u));
          q2 = min(max(q2, q1), max(hi, lo + 1u));
          q3 = min(max(q3, q2), max(hi, lo + 1u));
          double v[kSums] = {};
          int n0 = 0, n1 = 0, n2 = 0, n3 = 0;  // logits that reach lo, q1, q2, q3, and no more than hi
          if (by_mass) {
            for (int i = i0; i < i1; ++i) {
              const uint32_t k = at(i);
              if (k < lo || k > hi) continue;
              const double e = mass_of(k);
              ++n0;
              v[0] += e;
              if (k >= q1) { ++n1; v[1] += e; }
              if (k >= q2) { ++n2; v[2] += e; }
              if (k >= q3) { ++n3; v[3] += e; }
            }
          } else {
#pragma unroll 4
            for (int i = i0; i < i1; ++i) {
              const uint32_t k = at(i) <= hi ? at(i) : 0u;
              n0 += k >= lo;
              n1 += k >= q1;
              n2 += k >= q2;
              n3 += k >= q3;
            }
            v[0] = n0; v[1] = n1; v[2] = n2; v[3] = n3;
          }
          v[4] = n0; v[5] = n1; v[6] = n2; v[7] = n3;
          cluster_sums(Sums8(), v);
          if (pass == 0) {
            if (by_mass) {
              if (lo == low_key) whole = v[0];
              need *= v[0];
              if (!(need > 0.0)) return top_key;
            } else if (v[0] < need) {
              return lo;
            }
            if (lo >= hi) return lo;
          }
          by_key = false;
          if (above + v[3] >= need) { lo = q3; inside = v[7]; }
          else if (above + v[2] >= need) { above += v[3]; lo = q2; hi = q3 - 1u; inside = v[6] - v[7]; }
          else if (above + v[1] >= need) { above += v[2]; lo = q1; hi = q2 - 1u; inside = v[5] - v[6]; }
          else { above += v[1]; hi = q1 - 1u; inside = v[4] - v[5]; by_key = wide; }
        }
        if (lo >= hi) return lo;
        // the few between, in the order of their indices, by every CTA
        int mine = 0;
        for (int i = i0; i < i1; ++i) {
          const uint32_t k = at(i);
          mine += k >= lo && k <= hi;
        }
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += other;
        }
        if (lane == 31) sh.keys[warp] = before;
        __syncthreads();
        int base = 0, all = 0;
        for (int w = 0; w < kDrawWarps; ++w) {
          if (w < warp) base += sh.keys[w];
          all += sh.keys[w];
        }
        int to = base + before - mine;
        for (int i = i0; i < i1 && mine > 0; ++i) {
          const uint32_t k = at(i);
          if (k < lo || k > hi) continue;
          sh.listed[to] = k;
          sh.listed_mass[to] = by_mass ? mass_of(k) : 1.0;
          ++to;
        }
        if (tid == 0) sh.own_index[0] = all;
        if (C > 1) draw_barrier(); else __syncthreads();
        // each of them is tried by a thread of rank 0's numbering: what reaches it
        uint32_t best = lo;
        int n_all = 0, from_rank = -1, from = 0;
        for (int c = 0; c < C; ++c) {
          const int n = C > 1 ? (int)remote_u32(draw_remote(&sh.own_index[0], c)) : all;
          if (tid >= n_all && tid < n_all + n) {
            from_rank = c;
            from = tid - n_all;
          }
          n_all += n;
        }
        const uint32_t key = from_rank >= 0 ? (C > 1 ? remote_u32(draw_remote(&sh.listed[from], from_rank)) : sh.listed[from]) : 0u;
        const double weight = from_rank >= 0 ? (C > 1 ? remote_f64(draw_remote(&sh.listed_mass[from], from_rank)) : sh.listed_mass[from]) : 0.0;
        if (C > 1) draw_barrier(); else __syncthreads();  // (everyone has what it needs of the others' lists)
        if (tid < kListed) {
          sh.listed[tid] = key;
          sh.listed_mass[tid] = weight;
        }
        __syncthreads();
        if (from_rank >= 0) {
          double sum = above;
          for (int j = 0; j < n_all; ++j) sum += sh.listed[j] >= key ? sh.listed_mass[j] : 0.0;
          if (sum >= need) best = key;
        }
        best = __reduce_max_sync(0xffffffffu, best);
        __syncthreads();
        if (lane == 0) sh.keys[warp] = best;
        __syncthreads();
        best = __reduce_max_sync(0xffffffffu, lane < kDrawWarps ? sh.keys[lane] : 0u);
        __syncthreads();
        return best;
      };
      uint32_t limit = low_key;  // (key 0 is never drawn)
      const int k = p.top_k[draw];
      if (k > 0 && k < V) limit = search(false, limit, (double)k);
      const float tp = p.top_p[draw];
      if (tp < 1.f) limit = search(true, limit, fmax((double)tp, 0.0));
      const float mp = p.min_p[draw];
      const double least = mp > 0.f ? fmin(log((double)mp), 0.0) : -INFINITY;
      uint32_t quick = limit;  // most of what min-p leaves out is told by its key (which is rounded, so four steps are left for the exact question)
      if (mp > 0.f && top < INFINITY) {
        const uint32_t near = order_key(clean((float)((double)top + least * (double)t)));
        if (near > 4u) quick = max(quick, near - 4u);
      }
      auto kept = [&](uint32_t k) -> double {
        if (k < quick) return 0.0;
        if (k == top_key) return 1.0;
        const double z = ((double)of_key(k) - (double)top) * inv_t;
        return z >= least ? exp_down(z, sh.powers) : 0.0;
      };
      // the thread's run, then the running mass behind every thread's run
      double c = 0.0;
      int newest = -1;
      for (int i = i0; i < i1; ++i) {
        const double e = kept(at(i));
        if (e > 0.0) {
          c += e;
          newest = i;
        }
      }
      double behind = c;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, behind, o);
        if (lane >= o) behind += other;
      }
      __syncthreads();
      if (lane == 31) sh.parts[warp][0] = behind;
      newest = __reduce_max_sync(0xffffffffu, newest);
      if (lane == 0) sh.keys[warp] = (uint32_t)(newest + 1);
      __syncthreads();
      double front = 0.0, all = 0.0;
      for (int w = 0; w < kDrawWarps; ++w) {
        if (w == warp) front = all;
        all += sh.parts[w][0];
      }
      newest = (int)__reduce_max_sync(0xffffffffu, lane < kDrawWarps ? sh.keys[lane] : 0u) - 1;
      if (tid == 0) {
        sh.sums[turn][0] = all;
        sh.own_index[1] = newest < 0 ? -1 : c0 + newest;
      }
      if (C > 1) draw_barrier(); else __syncthreads();
      double total = 0.0, here = 0.0;
      int last = -1;
      for (int r = 0; r < C; ++r) {
        if (r == rank) here = total;
        total += C > 1 ? remote_f64(draw_remote(&sh.sums[turn][0], r)) : all;
        last = max(last, C > 1 ? (int)remote_u32(draw_remote(&sh.own_index[1], r)) : newest);
      }
      turn ^= 1;
      if (quick == low_key && !(mp > 0.f)) whole = total;
      whole = t == 1.f ? whole : -1.0;
      whole_row = whole;
      const double target = (double)p.u[draw] * total;
      const double start = here + front + (behind - c);
      // (the first thread whose run's end passes the target; what rounding leaves between a run's end and the next one's start goes to the next)
      if (c > 0.0 && here + front + behind > target) {
        double run = start;
        for (int i = i0; i < i1; ++i) {
          const double e = kept(at(i));
          run += e;
          if (e > 0.0 && run > target) {
            atomicMin(&sh.found, c0 + i);
            break;
          }
        }
      }
      __syncthreads();
      if (C > 1) {
        draw_barrier();
        int lowest = 0x7fffffff;
        for (int r = 0; r < C; ++r) lowest = min(lowest, (int)remote_u32(draw_remote(&sh.found, r)));
        token = lowest;
      } else {
        token = sh.found;
      }
      if (token == 0x7fffffff) token = last;  // (u of one and more, or none of the runs by rounding: the last kept one)
    }
  }
  if (p.logprobs) {
    // likely logits in 64 bits, the many others (below e^-8 of the largest) in 32: their errors are random and small against the sum
    double v[kSums] = {};
    if (top_key != 0u && whole_row < 0.0) {
      float rest = 0.f;
      for (int i = i0; i < i1; ++i) {
        const uint32_t k = at(i);
        const float xi = of_key(k), d = xi - top;
        if (k == top_key) v[0] += 1.0;
        else if (d > -8.f) v[0] += exp_down((double)xi - (double)top, sh.powers);
        else rest += __expf(d);
      }
      v[0] += (double)rest;
      cluster_sums(Sums1(), v);
    } else {
      v[0] = whole_row;
    }
    if (rank == 0 && tid == 0) {
      const float xt = clean(p.logits[(size_t)row * p.stride + token]);
      p.logprobs[draw] = top_key == 0u ? -INFINITY : (float)((xt == top ? 0.0 : (double)xt - (double)top) - log(v[0]));
    }
  }
  if (rank == 0 && tid == 0) p.out[draw] = token;
  if (C > 1) draw_barrier();  // nobody leaves while its shared memory is read
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
  FTK_REQUIRE(n_draws <= (1 << 24), "sample_draws: %d draws", n_draws);
  DrawParams p{logits, row_stride, n_rows, vocab, rows, temperature, top_k, top_p, min_p, u, out, logprobs, 1, 1};
  // a CTA for every 4,096 logits, eight at most
  while (p.cluster < 8 && vocab > p.cluster * 4096) p.cluster *= 2;
  p.run = ((vocab + p.cluster * kDrawThreads - 1) / (p.cluster * kDrawThreads)) | 1;
  const bool held = p.run <= kMostRun;  // (430,000 logits; longer rows are read again in every pass)
  const size_t smem = held ? (size_t)p.run * kDrawThreads * sizeof(float) : 0;
  auto kern = held ? draw_kernel<true> : draw_kernel<false>;
  FTK_REQUIRE(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) == cudaSuccess, "sample_draws: cannot set up the kernel");
  note_variant(held ? "draws: rows in shared memory" : "draws: rows read again in every pass");
  const dim3 grid((unsigned)(n_draws * p.cluster));
  if (p.cluster > 1) launch_kernel_clusters(kern, p.cluster, grid, dim3(kDrawThreads), smem, (cudaStream_t)stream, p);
  else FTK_LAUNCH(kern, grid, kDrawThreads, smem, stream, p);
  FTK_LAUNCH_CHECK("sample_draws");
  return 0;
}
