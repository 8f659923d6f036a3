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
// A cluster of up to sixteen CTAs takes a draw: a thread has a run of neighbouring logits, kept in shared memory from the one pass over
// memory.  A threshold is searched for by the number of the logits above it, with three candidates a pass, or by their mass, with seven a
// pass in 32 bits and then one pass in 64 that confirms the place; when at most kListed logits are left between, each of them is tried.
// What a CTA has to tell the others it writes into their shared memory in front of the cluster's barrier: reading it there behind
// the barrier would be one trip more a pass.
// What bounds it: for one draw the passes one after the other (a barrier of the cluster each, a microsecond or so with the wait for the
// slowest CTA); for many the instructions of the passes (0.63 of the issue slots taken, the 64-bit pipe 0.1): so logits lie in shared
// memory as numbers, four to a load, and are compared as such; and where top-k (of 128 at most) or top-p leaves no more than kListed of a
// row, every CTA lists those and does the rest in the list (one draw with all filters 33 -> 27 us, 96 of them from 24 rows 128 -> 102).
// Measured, rows of 200,000 normal logits (deviation 3) at T = 0.8, with log-probabilities, one launch between two events on cold caches: one
// draw without filters 22 us, with min-p 18, top-k 50, top-p 0.9 and min-p 27, top-p 0.95 alone 45; 96 draws from 24 rows 86, 55, 102
// and 217 us, from 96 rows 94, 64, 112 and 224.
#include "common.cuh"

namespace ftk {

constexpr int kDrawThreads = 512, kDrawWarps = kDrawThreads / 32;
constexpr int kMostCluster = 16;
constexpr int kListed = 256;      // logits that are tried one by one
constexpr int kMostRun = 108;     // logits of a thread's run that shared memory has room for

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
  int cluster, run;  // CTAs a draw; logits of a thread's run (four times an odd number: eight threads' quarters then lie in different banks)
};

// Logits in an order-preserving integer form: key 0 stands for NaN and -infinity.
__device__ __forceinline__ float clean(float x) { return fmaxf(x, -INFINITY) + 0.f; }  // (of a NaN and a number fmaxf gives the number; -0 is 0)
__device__ __forceinline__ uint32_t order_key(float x) {
  if (x == -INFINITY) return 0u;
  const uint32_t b = __float_as_uint(x);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
  if (k == 0u) return -INFINITY;
  return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// 2^(j / 256)
__device__ const double kPowers[256] = {
    1.00000000000000000e+00, 1.00271127505020252e+00, 1.00542990111280273e+00, 1.00815589811841755e+00, 1.01088928605170048e+00,
    1.01363008495148943e+00, 1.01637831491095310e+00, 1.01913399607773791e+00, 1.02189714865411663e+00, 1.02466779289713572e+00,
    1.02744594911876375e+00, 1.03023163768604098e+00, 1.03302487902122841e+00, 1.03582569360195720e+00, 1.03863410196137873e+00,
    1.04145012468831610e+00, 1.04427378242741375e+00, 1.04710509587928979e+00, 1.04994408580068721e+00, 1.05279077300462642e+00,
    1.05564517836055716e+00, 1.05850732279451276e+00, 1.06137722728926209e+00, 1.06425491288446450e+00, 1.06714040067682370e+00,
    1.07003371182024187e+00, 1.07293486752597556e+00, 1.07584388906279105e+00, 1.07876079775711986e+00, 1.08168561499321525e+00,
    1.08461836221330921e+00, 1.08755906091776966e+00, 1.09050773266525769e+00, 1.09346439907288584e+00, 1.09642908181637688e+00,
    1.09940180263022191e+00, 1.10238258330784089e+00, 1.10537144570174117e+00, 1.10836841172367873e+00, 1.11137350334481755e+00,
    1.11438674259589243e+00, 1.11740815156736928e+00, 1.12043775240960675e+00, 1.12347556733301990e+00, 1.12652161860824185e+00,
    1.12957592856628808e+00, 1.13263851959871920e+00, 1.13570941415780546e+00, 1.13878863475669156e+00, 1.14187620396956158e+00,
    1.14497214443180417e+00, 1.14807647884017894e+00, 1.15118922995298267e+00, 1.15431042059021594e+00, 1.15744007363375112e+00,
    1.16057821202749878e+00, 1.16372485877757748e+00, 1.16688003695248166e+00, 1.17004376968325019e+00, 1.17321608016363732e+00,
    1.17639699165028122e+00, 1.17958652746287584e+00, 1.18278471098434101e+00, 1.18599156566099384e+00, 1.18920711500272103e+00,
    1.19243138258315118e+00, 1.19566439203982733e+00, 1.19890616707438058e+00, 1.20215673145270308e+00, 1.20541610900512386e+00,
    1.20868432362658162e+00, 1.21196139927680124e+00, 1.21524735998046896e+00, 1.21854222982740845e+00, 1.22184603297275762e+00,
    1.22515879363714553e+00, 1.22848053610687002e+00, 1.23181128473407586e+00, 1.23515106393693341e+00, 1.23849989819981654e+00,
    1.24185781207348400e+00, 1.24522483017525798e+00, 1.24860097718920482e+00, 1.25198627786631622e+00, 1.25538075702469110e+00,
    1.25878443954971653e+00, 1.26219735039425074e+00, 1.26561951457880628e+00, 1.26905095719173322e+00, 1.27249170338940276e+00,
    1.27594177839639200e+00, 1.27940120750566932e+00, 1.28287001607877826e+00, 1.28634822954602557e+00, 1.28983587340666572e+00,
    1.29333297322908947e+00, 1.29683955465100964e+00, 1.30035564337965059e+00, 1.30388126519193581e+00, 1.30741644593467732e+00,
    1.31096121152476441e+00, 1.31451558794935464e+00, 1.31807960126606405e+00, 1.32165327760315754e+00, 1.32523664315974132e+00,
    1.32882972420595435e+00, 1.33243254708316150e+00, 1.33604513820414583e+00, 1.33966752405330292e+00, 1.34329973118683532e+00,
    1.34694178623294580e+00, 1.35059371589203447e+00, 1.35425554693689265e+00, 1.35792730621290114e+00, 1.36160902063822475e+00,
    1.36530071720401192e+00, 1.36900242297459052e+00, 1.37271416508766841e+00, 1.37643597075453017e+00, 1.38016786726023799e+00,
    1.38390988196383202e+00, 1.38766204229852907e+00, 1.39142437577192624e+00, 1.39519690996620027e+00, 1.39897967253831124e+00,
    1.40277269122020476e+00, 1.40657599381901544e+00, 1.41038960821727066e+00, 1.41421356237309515e+00, 1.41804788432041518e+00,
    1.42189260216916558e+00, 1.42574774410549421e+00, 1.42961333839197002e+00, 1.43348941336778890e+00, 1.43737599744898237e+00,
    1.44127311912862566e+00, 1.44518080697704665e+00, 1.44909908964203504e+00, 1.45302799584905262e+00, 1.45696755440144377e+00,
    1.46091779418064704e+00, 1.46487874414640573e+00, 1.46885043333698184e+00, 1.47283289086936753e+00, 1.47682614593949935e+00,
    1.48083022782247187e+00, 1.48484516587275239e+00, 1.48887098952439700e+00, 1.49290772829126484e+00, 1.49695541176723546e+00,
    1.50101406962642558e+00, 1.50508373162340647e+00, 1.50916442759342284e+00, 1.51325618745260981e+00, 1.51735904119821474e+00,
    1.52147301890881459e+00, 1.52559815074453842e+00, 1.52973446694728699e+00, 1.53388199784095591e+00, 1.53804077383165683e+00,
    1.54221082540794074e+00, 1.54639218314102145e+00, 1.55058487768499997e+00, 1.55478893977708865e+00, 1.55900440023783693e+00,
    1.56323128997135763e+00, 1.56746963996555300e+00, 1.57171948129234140e+00, 1.57598084510788650e+00, 1.58025376265282458e+00,
    1.58453826525249375e+00, 1.58883438431716395e+00, 1.59314215134226700e+00, 1.59746159790862707e+00, 1.60179275568269341e+00,
    1.60613565641677103e+00, 1.61049033194925428e+00, 1.61485681420486071e+00, 1.61923513519486373e+00, 1.62362532701732887e+00,
    1.62802742185734783e+00, 1.63244145198727497e+00, 1.63686744976696441e+00, 1.64130544764400632e+00, 1.64575547815396495e+00,
    1.65021757392061774e+00, 1.65469176765619430e+00, 1.65917809216161616e+00, 1.66367658032673638e+00, 1.66818726513058246e+00,
    1.67271017964159663e+00, 1.67724535701787847e+00, 1.68179283050742900e+00, 1.68635263344839337e+00, 1.69092479926930528e+00,
    1.69550936148933262e+00, 1.70010635371852348e+00, 1.70471580965805125e+00, 1.70933776310046293e+00, 1.71397224792992597e+00,
    1.71861929812247793e+00, 1.72327894774627399e+00, 1.72795123096183767e+00, 1.73263618202231107e+00, 1.73733383527370622e+00,
    1.74204422515515644e+00, 1.74676738619916905e+00, 1.75150335303187821e+00, 1.75625216037329945e+00, 1.76101384303758390e+00,
    1.76578843593327273e+00, 1.77057597406355471e+00, 1.77537649252652119e+00, 1.78019002651542446e+00, 1.78501661131893496e+00,
    1.78985628232140104e+00, 1.79470907500310717e+00, 1.79957502494053512e+00, 1.80445416780662393e+00, 1.80934653937103196e+00,
    1.81425217550039886e+00, 1.81917111215860849e+00, 1.82410338540705341e+00, 1.82904903140489727e+00, 1.83400808640934243e+00,
    1.83898058677589371e+00, 1.84396656895862598e+00, 1.84896606951045084e+00, 1.85397912508338547e+00, 1.85900577242882048e+00,
    1.86404604839778898e+00, 1.86909998994123860e+00, 1.87416763411029996e+00, 1.87924901805656019e+00, 1.88434417903233453e+00,
    1.88945315439093919e+00, 1.89457598158696561e+00, 1.89971269817655530e+00, 1.90486334181767414e+00, 1.91002795027038985e+00,
    1.91520656139714740e+00, 1.92039921316304740e+00, 1.92560594363612503e+00, 1.93082679098762711e+00, 1.93606179349229435e+00,
    1.94131098952864045e+00, 1.94657441757923322e+00, 1.95185211623097832e+00, 1.95714412417540018e+00, 1.96245048020892732e+00,
    1.96777122323317588e+00, 1.97310639225523432e+00, 1.97845602638795093e+00, 1.98382016485021939e+00, 1.98919884696726634e+00,
    1.99459211217094023e+00,
};
// 2^y for y <= 0: with k = 256 n + j the integer nearest to 256 y and r = y - k / 256 (exact, |r| <= 2^-9), 2^y = 2^n 2^(j / 256) 2^r, where the
// series up to r^3 is within 1.4e-13 (the term behind it, (ln 2 / 512)^4 / 24), and so is every sum of such numbers, some 2^-42.7.  Below
// 2^-1000: zero.  (Nine operations in 64 bits; powers of 1/32 and the series up to r^5, within 2.3e-15, took thirteen.)
__device__ __forceinline__ double exp2_down(double y, const double* powers) {
  double k = fma(y, 256.0, 6755399441055744.0);
  const int n = __double2loint(k);
  k -= 6755399441055744.0;
  const double r = fma(k, -1.0 / 256.0, y);
  double q = fma(r, 5.55041086648215831e-02, 2.40226506959100722e-01);
  q = fma(q, r, 6.93147180559945286e-01);
  const double t = powers[n & 255], v = fma(t, q * r, t);
  return y > -1000.0 ? __hiloint2double(__double2hiint(v) + ((n >> 8) << 20), __double2loint(v)) : 0.0;
}

__device__ __forceinline__ float exp2f_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t draw_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ uint32_t draw_remote(const void* p, int rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(draw_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void put_f64(uint32_t at, double v) { asm volatile("st.shared::cluster.f64 [%0], %1;" ::"r"(at), "d"(v) : "memory"); }
__device__ __forceinline__ void put_u32(uint32_t at, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory"); }
__device__ __forceinline__ void draw_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void draw_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ void draw_barrier() {
  draw_arrive();
  draw_wait();
}
template <typename T>
__device__ __forceinline__ T warp_sum_of(T v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

struct DrawShared {
  double powers[256];
  union {
    double parts[kDrawWarps][8];  // the warps' sums
    uint32_t listed_at[kListed];  // where the listed logits stand in the row
  };
  int counts[kDrawWarps][4];
  double inbox[2][kMostCluster][8];  // what every CTA of the cluster has sent to this one: in turns, so that one barrier a pass is enough
  double listed_mass[kListed];
  uint32_t listed[kListed];
  uint32_t keys[kDrawWarps], low_keys[kDrawWarps];
  double reached;
  int first, crossing;
};

template <int N>
struct SumCount {
  static constexpr int value = N;
};

template <bool STAGED>
__global__ void __launch_bounds__(kDrawThreads, 2) draw_kernel(const __grid_constant__ DrawParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) float staged[];  // the chunk's logits, -infinity behind the row's end
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
  if (C > 1) draw_arrive();  // (waited for in front of the first word to another CTA)
  const int chunk = p.run * kDrawThreads, c0 = min(V, rank * chunk), n_here = min(V - c0, chunk);  // (rank * chunk < 2^31: the host checks)
  const float* x = p.logits + (size_t)row * p.stride + c0;
  if (tid < 256) sh.powers[tid] = kPowers[tid];
  if (tid == 0) {
    sh.first = 0x7fffffff;
    sh.crossing = 0x7fffffff;
  }
  // ---- the chunk comes in; its largest logit
  uint32_t top_key, low_key;  // the largest logit, and the smallest above -infinity
  {
    float most = -INFINITY, least = INFINITY;
    auto note = [&](float v) -> float {
      v = clean(v);
      most = fmaxf(most, v);
      least = fminf(least, v == -INFINITY ? INFINITY : v);
      return v;
    };
    if ((((uintptr_t)x) & 15) == 0) {
      const float4* x4 = reinterpret_cast<const float4*>(x);
      const int n4 = n_here >> 2;
      for (int i0 = 0; i0 < n4; i0 += 7 * kDrawThreads) {
        float4 v[7];
#pragma unroll
        for (int e = 0; e < 7; ++e) {
          const int i = i0 + e * kDrawThreads + tid;
          if (i < n4) v[e] = __ldg(x4 + i);
        }
#pragma unroll
        for (int e = 0; e < 7; ++e) {
          const int i = i0 + e * kDrawThreads + tid;
          if (i < n4) {
            const float4 c = make_float4(note(v[e].x), note(v[e].y), note(v[e].z), note(v[e].w));
            if (STAGED) *reinterpret_cast<float4*>(staged + 4 * i) = c;
          }
        }
      }
      for (int i = 4 * n4 + tid; i < n_here; i += kDrawThreads) {
        const float c = note(x[i]);
        if (STAGED) staged[i] = c;
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
            const float c = note(v[e]);
            if (STAGED) staged[i] = c;
          }
        }
      }
    }
    if (STAGED)
      for (int i = n_here + tid; i < chunk && i < ((n_here + 3) & ~3); i += kDrawThreads) staged[i] = -INFINITY;
    top_key = order_key(most);
    low_key = least == INFINITY && most < INFINITY ? 0xffffffffu : order_key(least) - 1u;
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
  int turn = 0;
  // A word to slot s of every CTA's inbox; from warp 0, by a lane for each of them.
  auto send = [&](int s, double v) {
    if (C == 1) {
      if (lane == 0) sh.inbox[turn][0][s] = v;
    } else if (lane < C) {
      put_f64(draw_remote(&sh.inbox[turn][rank][s], lane), v);
    }
  };
  auto meet = [&]() {
    if (C > 1) draw_barrier(); else __syncthreads();
  };
  if (C > 1) draw_wait();
  if (warp == 0) {
    send(0, top_key);
    send(1, low_key);
  }
  meet();
  top_key = __reduce_max_sync(0xffffffffu, lane < C ? (uint32_t)sh.inbox[turn][lane][0] : 0u);
  low_key = __reduce_min_sync(0xffffffffu, lane < C ? (uint32_t)sh.inbox[turn][lane][1] : 0xffffffffu);
  turn ^= 1;
  low_key += 1u;
  const float t = p.temperature[draw];
  const int i0 = min(n_here, tid * p.run), i1 = min(n_here, i0 + p.run);
  // Where the largest logit is infinite, its like have all of the mass: they count as 0, the others as -infinity.
  const bool endless = top_key == order_key(INFINITY);
  if (endless) {
    if (STAGED) {
      for (int i = i0; i < i1; ++i) staged[i] = staged[i] == INFINITY ? 0.f : -INFINITY;
      __syncthreads();
    }
    top_key = low_key = order_key(0.f);
  }
  const float top = of_key(top_key);
  auto seen = [&](float v) -> float {
    v = clean(v);
    return !endless ? v : v == INFINITY ? 0.f : -INFINITY;
  };
  auto at = [&](int i) -> float { return STAGED ? staged[i] : seen(__ldg(x + i)); };
  // four of the run at a time (-infinity behind its end), so that four exponentials are under way at once
  auto four = [&](int i, float (&v)[4]) {
    if (STAGED) {
      const float4 f = *reinterpret_cast<const float4*>(staged + i);
      v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = i + e < i1 ? at(i + e) : -INFINITY;
    }
  };
  auto most_of = [](const float (&v)[4]) { return fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])); };
  // Sums over the cluster, the same in every thread: NM of masses (a warp's in their own type, the others in 64 bits) and NC of integers
  // (four of them at most, and then four masses).
  auto cluster_sums = [&](auto masses, auto counts, const auto& part, auto& m, int (&n)[4]) {
    constexpr int NM = decltype(masses)::value, NC = decltype(counts)::value;
#pragma unroll
    for (int s = 0; s < NM; ++s) {
      const double v = warp_sum_of(part[s]);
      if (lane == 0) sh.parts[warp][s] = v;
    }
#pragma unroll
    for (int s = 0; s < NC; ++s) {
      const int v = __reduce_add_sync(0xffffffffu, n[s]);
      if (lane == 0) sh.counts[warp][s] = v;
    }
    __syncthreads();
    if (warp == 0) {  // lane 16 h + w: every second sum from h on, of warp w
      const int w = lane & 15, h = lane >> 4;
      double a[(NM + 1) / 2 + 1];
      int c[(NC + 1) / 2 + 1];
#pragma unroll
      for (int e = 0; 2 * e < NM; ++e) a[e] = 2 * e + h < NM ? sh.parts[w][2 * e + h] : 0.0;
#pragma unroll
      for (int e = 0; 2 * e < NC; ++e) c[e] = 2 * e + h < NC ? sh.counts[w][2 * e + h] : 0;
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
#pragma unroll
        for (int e = 0; 2 * e < NM; ++e) a[e] += __shfl_xor_sync(0xffffffffu, a[e], o);
#pragma unroll
        for (int e = 0; 2 * e < NC; ++e) c[e] += __shfl_xor_sync(0xffffffffu, c[e], o);
      }
      // (lane 16 h + w has them for CTA w)
      if (w < C) {
        double* mine = &sh.inbox[turn][rank][h];
        const uint32_t to = C > 1 ? draw_remote(mine, w) : draw_addr(mine);
#pragma unroll
        for (int e = 0; 2 * e < NM; ++e)
          if (2 * e + h < NM) put_f64(to + 16 * e, a[e]);
#pragma unroll
        for (int e = 0; 2 * e < NC; ++e)
          if (2 * e + h < NC) put_f64(to + 32 + 16 * e, c[e]);
      }
    }
    meet();
    // every warp by itself; lane 8 c + s: sums s of CTAs c, c + 4, ...
    const int s = lane & 7, c = lane >> 3;
    double sum = 0.0;
    if (s < NM || (s >= 4 && s < 4 + NC)) {
      double v[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = c + 4 * e < C ? sh.inbox[turn][c + 4 * e][s] : 0.0;
      sum = (v[0] + v[1]) + (v[2] + v[3]);
    }
    sum += __shfl_xor_sync(0xffffffffu, sum, 8);
    sum += __shfl_xor_sync(0xffffffffu, sum, 16);
#pragma unroll
    for (int e = 0; e < NM; ++e) m[e] = __shfl_sync(0xffffffffu, sum, e);
#pragma unroll
    for (int e = 0; e < NC; ++e) n[e] = (int)__shfl_sync(0xffffffffu, sum, 4 + e);
    turn ^= 1;
  };
  // The largest of a number of every thread.
  auto block_max = [&](uint32_t v) -> uint32_t {
    v = __reduce_max_sync(0xffffffffu, v);
    __syncthreads();
    if (lane == 0) sh.keys[warp] = v;
    __syncthreads();
    v = __reduce_max_sync(0xffffffffu, lane < kDrawWarps ? sh.keys[lane] : 0u);
    __syncthreads();
    return v;
  };
  int token = 0;
  double whole_row = -1.0;  // the row's mass at temperature 1, where it is known
  if (top_key != 0u) {
    if (!(t > 0.f)) {  // the lowest index of the largest logit
      for (int i = i0; i < i1; ++i)
        if (at(i) == top) {
          atomicMin(&sh.first, c0 + i);
          break;
        }
      __syncthreads();
      if (warp == 0) send(0, sh.first);
      meet();
      token = (int)__reduce_min_sync(0xffffffffu, lane < C ? (uint32_t)sh.inbox[turn][lane][0] : 0x7fffffffu);
      turn ^= 1;
    } else {
      const double inv_t = 1.0 / (double)t, per_bit = inv_t * 1.4426950408889634074;  // z / ln 2 of a logit's distance
      auto mass_of = [&](float v) -> double { return exp2_down(((double)v - (double)top) * per_bit, sh.powers); };
      int held_by_k = V;  // logits that top-k left
      double over_mine = 0.0;           // of this thread's logits: the mass of those that reach key `over_key`, where that was summed up
      uint32_t over_key = 0xffffffffu;
      double whole = -1.0;  // the mass of the whole row at this temperature, where it was summed up
      // Three candidates between: by value, as logits spread like their values do: close below the largest where some lie far away (masked
      // ones, say: true is returned then), in quarters, or, in a narrow range, around the place that `part` of what it holds lies above; or by
      // key, which ends whatever they are.
      auto candidates = [&](uint32_t lo, uint32_t hi, bool by_key, double part, uint32_t& q1, uint32_t& q2, uint32_t& q3) -> bool {
        const uint32_t gap = hi - lo;
        const float a = of_key(lo), b = of_key(hi);
        q1 = lo + gap / 4u + (gap < 4u), q2 = lo + gap / 2u + (gap & 1u), q3 = hi - gap / 4u;
        const bool wide = !(b - a <= 64.f * t);
        if (!by_key) {
          q1 = order_key(clean(wide ? b - 30.f * t : a + 0.25f * (b - a)));
          q2 = order_key(clean(wide ? b - 10.f * t : a + 0.5f * (b - a)));
          q3 = order_key(clean(wide ? b - 4.f * t : a + 0.75f * (b - a)));
          if (!wide && part >= 0.0 && b - a <= 8.f * t) {
            const float guess = b - (float)part * (b - a), off = 0.06f * (b - a);
            q1 = order_key(clean(guess - off));
            q2 = order_key(clean(guess));
            q3 = order_key(clean(guess + off));
          }
        }
        q1 = min(max(q1, lo + 1u), max(hi, lo + 1u));
        q2 = min(max(q2, q1), max(hi, lo + 1u));
        q3 = min(max(q3, q2), max(hi, lo + 1u));
        return wide;
      };
      // Where few logits are left of the row, every CTA lists them all, and what follows is done in the list.
      int n_list = 0;
      double held_here = 0.0;  // what reaches the logit that this thread has of the list
      // The largest key from `lo` on at which the number (by_mass: the mass) of the logits that reach it is `need` (by_mass: `need` of what
      // reaches `lo`) or more; `lo` where not even that has as many.  (Logits are compared as numbers: what lies above key `hi` reaches the
      // number of key hi + 1.)
      auto search = [&](bool by_mass, uint32_t lo, double need) -> uint32_t {
        uint32_t hi = top_key;
        double above = 0.0;    // of the logits above `hi`
        int inside = held_by_k, mine = 0;  // logits between, and this thread's of them
        bool by_key = false, sure = false, list_all = !by_mass && need <= kListed / 2;
        int from_s = 0, to_s = -1;  // the counts of the last pass whose difference is what each CTA has between
        double part = -1.0;  // of what is between, how much lies above the place that is searched for, about
        if (by_mass) {
          // In 32 bits first, down to where the sums' roundings (2^-16 of them is more than those make) leave it open; then one pass in 64 bits
          // over everything, which finds the mass and confirms the place.
          const uint32_t limit = lo;
          const float limit_x = of_key(limit), per_bit32 = fminf((float)per_bit, 3e38f);
          double reach = 0.0, held = 0.0;  // mass of all, mass between
          bool few = inside <= kListed / 2;
          for (int p32 = 0; p32 < 12 && lo < hi && !few; ++p32) {
            // Seven candidates: in eighths by value or, where a few times T is between, around the place that a mass spread evenly over it
            // would put there; now and then by key, which ends whatever the logits are.
            uint32_t q[8];
            const float a = of_key(lo), b = of_key(hi), width = b - a;
            const bool wide = !(width <= 64.f * t), near = part >= 0.0 && width <= 8.f * t;
            const bool keys = by_key || p32 % 4 == 3;
            const float guess = b - (float)part * width;
            q[0] = lo;
#pragma unroll
            for (int s = 1; s < 8; ++s) {
              const float off[8] = {0.f, -0.25f, -0.08f, -0.02f, 0.f, 0.02f, 0.08f, 0.25f}, down[8] = {0.f, 60.f, 30.f, 20.f, 14.f, 9.f, 5.f, 2.f};
              const float x = wide ? b - down[s] * t : near ? guess + off[s] * width : a + 0.125f * s * width;
              uint32_t k = keys ? lo + (uint32_t)(((unsigned long long)(hi - lo) * s + 7) >> 3) : order_key(clean(x));
              q[s] = max(min(max(k, lo + 1u), hi), q[s - 1]);
            }
            const float lo_x = of_key(lo);
            float qx[8], f[8];
#pragma unroll
            for (int s = 0; s < 8; ++s) {
              qx[s] = s ? of_key(q[s]) : limit_x;
              f[s] = 0.f;
            }
            for (int i = i0; i < i1; i += 4) {
              float v[4];
              four(i, v);
              if (most_of(v) < lo_x) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const float m = exp2f_fast((v[e] - top) * per_bit32);
#pragma unroll
                for (int s = 0; s < 8; ++s)
                  if (v[e] >= qx[s]) f[s] += m;
              }
            }
            double v[8];
            int none[4];
            cluster_sums(SumCount<8>(), SumCount<0>(), f, v, none);
            if (p32 == 0) reach = v[0];
            else v[0] = above + held;
            const double need32 = need * reach, open = reach * (1.0 / 65536.0);
            int sure_s = 0, not_s = 8;  // the last candidate that is reached for sure, the first that is not
            double mass_below = v[0], mass_beyond = above;
#pragma unroll
            for (int s = 1; s < 8; ++s)
              if (v[s] >= need32 + open) { sure_s = s; lo = q[s]; mass_below = v[s]; }
#pragma unroll
            for (int s = 7; s > 0; --s)
              if (v[s] <= need32 - open) { not_s = s; hi = q[s] - 1u; mass_beyond = v[s]; }
            if (sure_s == 0 && not_s == 8) break;
            by_key = sure_s == 0 && wide;
            above = mass_beyond;
            held = mass_below - mass_beyond;
            part = (need32 - above) / fmax(held, 1e-300);
            few = (float)held <= (kListed / 2) * exp2f_fast((of_key(lo) - top) * per_bit32);  // (each has as much as the lowest at least)
          }
          const float lo_x = of_key(lo), over_x = of_key(hi + 1u);
          double v[4] = {0.0, 0.0, 0.0, 0.0};  // what reaches `limit`, `lo`, and what is above `hi`
          int n[4] = {0, 0, 0, 0};
          for (int i = i0; i < i1; i += 4) {
            float x4[4];
            four(i, x4);
            if (most_of(x4) < limit_x) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const double m = mass_of(x4[e]);
              if (x4[e] >= limit_x) v[0] += m;
              if (x4[e] >= lo_x) { v[1] += m; ++n[0]; ++n[1]; }
              if (x4[e] >= over_x) { v[2] += m; --n[0]; }
            }
          }
          mine = n[0];
          const int reaching = n[1];
          over_mine = v[2];
          over_key = hi + 1u;
          cluster_sums(SumCount<3>(), SumCount<2>(), v, v, n);
          if (limit == low_key) whole = v[0];
          need *= v[0];
          if (!(need > 0.0)) return top_key;
          above = v[2];
          inside = n[0];
          sure = v[1] >= need && v[2] < need;
          list_all = sure && n[1] <= kListed;
          if (list_all) {
            above = 0.0;
            inside = n[1];
            mine = reaching;
            from_s = 1;
          }
          if (!sure) {  // (not the place after all: from the start)
            over_key = 0xffffffffu;
            lo = limit;
            hi = top_key;
            above = 0.0;
          }
          by_key = false;
          part = -1.0;
        }
        for (int pass = 0; !sure || (lo < hi && inside > kListed); ++pass) {
          uint32_t k1, k2, k3;
          const bool wide = candidates(lo, hi, by_key || pass % 3 == 2, part, k1, k2, k3);
          const float lo_x = of_key(lo), over_x = of_key(hi + 1u), q1 = of_key(k1), q2 = of_key(k2), q3 = of_key(k3);
          // mass (or number) and number of the logits that reach lo, q1, q2, q3, and (where not all of them will be listed) no more than hi
          double v[4] = {0.0, 0.0, 0.0, 0.0};
          int n[4] = {0, 0, 0, 0}, own_over = 0;
          if (by_mass) {
            for (int i = i0; i < i1; i += 4) {
              float x4[4];
              four(i, x4);
              if (most_of(x4) < lo_x) continue;
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (x4[e] >= lo_x && !(x4[e] >= over_x)) {
                  const double m = mass_of(x4[e]);
                  ++n[0], v[0] += m;
                  if (x4[e] >= q1) { ++n[1]; v[1] += m; }
                  if (x4[e] >= q2) { ++n[2]; v[2] += m; }
                  if (x4[e] >= q3) { ++n[3]; v[3] += m; }
                }
            }
          } else {
            for (int i = i0; i < i1; i += 4) {
              float x4[4];
              four(i, x4);
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                n[0] += x4[e] >= lo_x;
                n[1] += x4[e] >= q1;
                n[2] += x4[e] >= q2;
                n[3] += x4[e] >= q3;
                own_over += !list_all && x4[e] >= over_x;
              }
            }
#pragma unroll
            for (int s = 0; s < 4; ++s) n[s] -= own_over;
          }
          const int own0 = n[0], own1 = n[1], own2 = n[2], own3 = n[3];  // this thread's
          if (by_mass) {
            cluster_sums(SumCount<4>(), SumCount<4>(), v, v, n);
          } else {
            cluster_sums(SumCount<0>(), SumCount<4>(), v, v, n);
            v[0] = n[0]; v[1] = n[1]; v[2] = n[2]; v[3] = n[3];
          }
          if (!sure) {
            if (v[0] < need) return lo;
            if (lo >= hi) return lo;
            sure = true;
          }
          by_key = false;
          double held = v[0] - v[1];
          const int beyond1 = list_all ? 0 : n[1], beyond2 = list_all ? 0 : n[2], beyond3 = list_all ? 0 : n[3];
          if (above + v[3] >= need) { lo = k3; inside = n[3]; mine = own3; held = v[3]; from_s = 3; to_s = -1; }
          else if (above + v[2] >= need) { above += list_all ? 0.0 : v[3]; lo = k2; hi = k3 - 1u; inside = n[2] - beyond3; mine = own2 - (list_all ? 0 : own3); held = v[2] - v[3]; from_s = 2; to_s = list_all ? -1 : 3; }
          else if (above + v[1] >= need) { above += list_all ? 0.0 : v[2]; lo = k1; hi = k2 - 1u; inside = n[1] - beyond2; mine = own1 - (list_all ? 0 : own2); held = v[1] - v[2]; from_s = 1; to_s = list_all ? -1 : 2; }
          else { above += list_all ? 0.0 : v[1]; hi = k1 - 1u; inside = n[0] - beyond1; by_key = wide; mine = own0 - (list_all ? 0 : own1); from_s = 0; to_s = list_all ? -1 : 1; }
          over_key = 0xffffffffu;
          if (by_mass) part = (need - above) / fmax(held, 1e-300);  // (a tail's numbers fall off too fast for that)
        }
        if (lo >= hi && !(list_all && inside <= kListed)) return lo;
        // the few between go to every CTA, in the order of their indices: behind those of the CTAs in front, as the last pass counted them
        int there = 0;
        if (lane < C) {
          const double* counts = sh.inbox[turn ^ 1][lane] + 4;
          there = (int)(counts[from_s] - (to_s >= 0 ? counts[to_s] : 0.0));
        }
        int base = __reduce_add_sync(0xffffffffu, lane < rank ? there : 0);
        int before = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, before, o);
          if (lane >= o) before += other;
        }
        if (lane == 31) sh.keys[warp] = before;
        __syncthreads();
        base += __reduce_add_sync(0xffffffffu, lane < warp ? sh.keys[lane] : 0u);
        int to = base + before - mine;
        const int full = base + before;
        const float lo_x = of_key(lo), over_x = list_all ? NAN : of_key(hi + 1u);  // (nothing reaches NaN)
        for (int i = i0; to < full && i < i1; i += 4) {
          float v[4];
          four(i, v);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (v[e] >= lo_x && !(v[e] >= over_x) && to < kListed) {
              const uint32_t key = order_key(v[e]);
              const double mass = by_mass || list_all ? mass_of(v[e]) : 1.0;
              for (int c = 0; c < C; ++c) {
                put_u32(C > 1 ? draw_remote(&sh.listed[to], c) : draw_addr(&sh.listed[to]), key);
                put_f64(C > 1 ? draw_remote(&sh.listed_mass[to], c) : draw_addr(&sh.listed_mass[to]), mass);
                if (list_all) put_u32(C > 1 ? draw_remote(&sh.listed_at[to], c) : draw_addr(&sh.listed_at[to]), (uint32_t)(c0 + i + e));
              }
              ++to;
            }
        }
        const int n_all = min(inside, kListed);
        if (tid >= n_all && tid < kListed) sh.listed[tid] = 0u;  // (no logit's)
        meet();
        // each of them is tried by a thread: what reaches it
        uint32_t best = lo;
        const uint32_t key = tid < n_all ? sh.listed[tid] : 0u;
        if (tid < n_all) {
          double sum[4] = {above, 0.0, 0.0, 0.0};
          int reach = 0;
          for (int j = 0; j < n_all; j += 4)  // (what is behind the last is key 0)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (sh.listed[j + e] >= key) { sum[e] += sh.listed_mass[j + e]; ++reach; }
          held_here = (sum[0] + sum[1]) + (sum[2] + sum[3]);
          if ((!by_mass && list_all ? (double)reach : held_here) >= need) best = key;
        }
        if (list_all) n_list = n_all;
        best = block_max(best);
        return best;
      };
      uint32_t limit = low_key;  // (key 0 is never drawn)
      const int k = p.top_k[draw];
      if (k > 0 && k < V) {
        limit = search(false, limit, (double)k);
        held_by_k = k;  // (about: ties stay)
      }
      const float tp = p.top_p[draw];
      const bool k_listed = n_list > 0;
      if (tp < 1.f && !k_listed) limit = search(true, limit, fmax((double)tp, 0.0));
      const float mp = p.min_p[draw];
      const double least = mp > 0.f ? fmin(log((double)mp), 0.0) : -INFINITY;
      if (n_list > 0) {
        const uint32_t key = tid < n_list ? sh.listed[tid] : 0u;
        if (tp < 1.f && k_listed) {  // of what top-k left
          if (key == limit) sh.reached = held_here;  // (the same from every thread)
          __syncthreads();
          const double need = fmax((double)tp, 0.0) * sh.reached;
          limit = need > 0.0 ? block_max(key >= limit && held_here >= need ? key : limit) : top_key;
        }
        double m = tid < n_list ? sh.listed_mass[tid] : 0.0;
        if (!(key >= limit && (mp > 0.f ? ((double)of_key(key) - (double)top) * inv_t >= least : true))) m = 0.0;
        double behind = m;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const double other = __shfl_up_sync(0xffffffffu, behind, o);
          if (lane >= o) behind += other;
        }
        __syncthreads();
        if (lane == 31) sh.listed_mass[warp] = behind;
        __syncthreads();
        double front = 0.0, total = 0.0;
#pragma unroll
        for (int w = 0; w < kListed / 32; ++w) {
          if (w == warp) front = total;
          total += sh.listed_mass[w];
        }
        const double target = (double)p.u[draw] * total;
        // the first that passes the target, or (u of one and more, or by rounding) the last that is kept: as 2^31 less its place, or its place
        const bool past = m > 0.0 && front + behind > target;
        const uint32_t pick = block_max(past ? 0x80000000u - (uint32_t)tid : m > 0.0 ? (uint32_t)tid : 0u);
        token = (int)sh.listed_at[pick > kListed ? 0x80000000u - pick : pick];
        whole_row = t == 1.f ? whole : -1.0;
        __syncthreads();  // (the places lie where sums will)
      } else {
      uint32_t quick = limit;  // most of what min-p leaves out is told by its key (which is rounded, so four steps are left for the exact question)
      if (mp > 0.f) {
        const uint32_t near = order_key(clean((float)((double)top + least * (double)t)));
        if (near > 4u) quick = max(quick, near - 4u);
      }
      const float quick_x = of_key(quick);
      auto kept = [&](float v) -> double {
        const double d = (double)v - (double)top, m = exp2_down(d * per_bit, sh.powers);
        return v >= quick_x && d * inv_t >= least ? m : 0.0;
      };
      // the thread's run, then the running mass behind every thread's run
      double c = 0.0;
      int newest = -1;
      if (over_key != 0xffffffffu && !(mp > 0.f)) {  // top-p's search left the mass above its last bracket
        const float over_x = of_key(over_key);
        c = over_mine;
        for (int i = i0; i < i1; i += 4) {
          float v[4];
          four(i, v);
          if (most_of(v) < quick_x) continue;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (v[e] >= quick_x) {
              newest = i + e;
              if (!(v[e] >= over_x)) c += mass_of(v[e]);
            }
        }
      } else {
        for (int i = i0; i < i1; i += 4) {
          float v[4];
          four(i, v);
          if (most_of(v) < quick_x) continue;
          double m[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) m[e] = kept(v[e]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            c += m[e];
            if (m[e] > 0.0) newest = i + e;
          }
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
      if (warp == 0) {
        send(0, all);
        send(1, newest < 0 ? -1.0 : (double)(c0 + newest));
      }
      meet();
      const double theirs = lane < C ? sh.inbox[turn][lane][0] : 0.0;
      const int last = __reduce_max_sync(0xffffffffu, lane < C ? (int)sh.inbox[turn][lane][1] : -1);
      double so_far = theirs;
#pragma unroll
      for (int o = 1; o < kMostCluster; o <<= 1) {
        const double other = __shfl_up_sync(0xffffffffu, so_far, o);
        if (lane >= o) so_far += other;
      }
      const double total = __shfl_sync(0xffffffffu, so_far, C - 1), here = rank ? __shfl_sync(0xffffffffu, so_far, rank - 1) : 0.0;
      turn ^= 1;
      if (quick == low_key && !(mp > 0.f)) whole = total;
      whole = t == 1.f ? whole : -1.0;
      whole_row = whole;
      const double target = (double)p.u[draw] * total;
      // the first thread whose run's end passes the target; its warp takes the run, a lane a logit
      if (c > 0.0 && here + front + behind > target) atomicMin(&sh.crossing, tid);
      __syncthreads();
      const int crossing = sh.crossing;
      int token_here = -1;
      if (crossing >> 5 == warp) {
        double run = __shfl_sync(0xffffffffu, here + front + (behind - c), crossing & 31);
        const int end = min(n_here, (crossing + 1) * p.run);
        for (int j0 = min(n_here, crossing * p.run); j0 < end; j0 += 32) {
          const int i = j0 + lane;
          const double m = i < end ? kept(at(i)) : 0.0;
          double sum = m;
#pragma unroll
          for (int o = 1; o < 32; o <<= 1) {
            const double other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += other;
          }
          const unsigned past = __ballot_sync(0xffffffffu, m > 0.0 && run + sum > target), some = __ballot_sync(0xffffffffu, m > 0.0);
          if (past) {
            token_here = j0 + __ffs((int)past) - 1;
            break;
          }
          if (some) token_here = j0 + 31 - __clz((int)some);  // (its last kept one, should rounding have it)
          run += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (lane == 0 && token_here >= 0) sh.first = c0 + token_here;
      }
      __syncthreads();
      if (warp == 0) send(0, sh.first);
      meet();
      token = (int)__reduce_min_sync(0xffffffffu, lane < C ? (uint32_t)sh.inbox[turn][lane][0] : 0x7fffffffu);
      turn ^= 1;
      if (token == 0x7fffffff) token = last;  // (u of one and more, or none of the runs by rounding: the last kept one)
      }
    }
  }
  if (p.logprobs) {
    // What lies within a factor of 20 of the largest in 64 bits, so that a few large terms leave no error; the others in 32 bits, where an
    // exponential is within 2^-22.5 (and its argument's rounding) and the errors of many are random.
    double v[4] = {whole_row, 0.0, 0.0, 0.0};
    if (top_key != 0u && whole_row < 0.0) {
      float sum[4] = {0.f, 0.f, 0.f, 0.f};
      for (int i = i0; i < i1; i += 4) {
        float v4[4];
        four(i, v4);
        if (most_of(v4) - top > -3.f) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[1] += exp2_down(((double)v4[e] - (double)top) * 1.4426950408889634074, sh.powers);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) sum[e] += __expf(v4[e] - top);
        }
      }
      int n[4];
      v[0] = ((double)(sum[0] + sum[1]) + (double)(sum[2] + sum[3])) + v[1];
      cluster_sums(SumCount<1>(), SumCount<0>(), v, v, n);
    }
    if (rank == 0 && tid == 0) {
      const float xt = seen(p.logits[(size_t)row * p.stride + token]);
      p.logprobs[draw] = top_key == 0u ? -INFINITY : (float)((xt == top ? 0.0 : (double)xt - (double)top) - log(v[0]));
    }
  }
  if (rank == 0 && tid == 0) p.out[draw] = token;
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
  // A CTA for every 4,096 logits, eight at most; sixteen for up to four draws.  Rows of 200,000 (as at the top), eight and sixteen: one draw 29
  // and 22 us, with top-p 57 and 45; four 27 and 20, 55 and 44; eight 27 and 25, with top-p 57 and 55 (57 and 61 where 40 logits stand out of a
  // row), with all filters 33 and 32; sixteen 35 and 37, 80 and 84; 96 from 24 rows 86 and 121.
  while (p.cluster < (n_draws <= 4 ? 16 : 8) && vocab > p.cluster * 4096) p.cluster *= 2;
  p.run = 4 * (((vocab + 4 * p.cluster * kDrawThreads - 1) / (4 * p.cluster * kDrawThreads)) | 1);
  const bool held = p.run <= kMostRun;  // (442,000 logits; longer rows are read again in every pass)
  const size_t smem = held ? (size_t)p.run * kDrawThreads * sizeof(float) : 0;
  auto kern = held ? draw_kernel<true> : draw_kernel<false>;
  static OncePerDevice once[2];
  FTK_REQUIRE(once[held]([&] {
                return set_shared_limit(kern, held ? kMostRun * kDrawThreads * sizeof(float) : 0) &&
                       cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) == cudaSuccess;
              }),
              "sample_draws: cannot set up the kernel");
  note_variant(held ? "draws: rows in shared memory" : "draws: rows read again in every pass");
  const dim3 grid((unsigned)(n_draws * p.cluster));
  if (p.cluster > 1) launch_kernel_clusters(kern, p.cluster, grid, dim3(kDrawThreads), smem, (cudaStream_t)stream, p);
  else FTK_LAUNCH(kern, grid, kDrawThreads, smem, stream, p);
  FTK_LAUNCH_CHECK("sample_draws");
  return 0;
}
