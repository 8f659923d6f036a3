// Shared keys on the 5th-generation tensor cores (tcgen05): up to 256 query rows a piece.  Included by shared_attention.cu.
//
// A piece of work is a range of keys for the query rows of one KV head of up to 2 x (128 / group) members: tiles A and B of 128 rows, which
// read the same keys and values.  No row of a piece may see less than another, so there is no mask but the end of the last key tile.
// Per key tile of 128 and query tile:
//   S = Q K^T     tcgen05.mma from shared memory (queries gathered row by row from the members' places by the softmax warps, keys
//                 straight from the pages by TMA, 16 rows a box; 128-byte swizzle), S in tensor memory;
//   softmax       a thread a row: maximum, exp2, sum in 32 bits; probabilities as bfloat16 over the first half of the scores.  The
//                 running maximum moves only when it grew by more than 8 (a factor of 256: l and o stay far from the ends of 32 bits), so
//                 that the accumulator is rescaled a few times a row;
//   O += P V      P from tensor memory, V from shared memory as it lies in the pages.
// The issuing warp takes the tiles in turn, so the tensor pipe works on one while the other's softmax runs.  A piece with members for
// one query tile only may be *split*: both tiles then hold the same rows, tile A works through the even key tiles and B through the
// odd ones, and each leaves partial results of its own (the chain scores - softmax - product of one tile keeps neither pipe busy).
// One CTA an SM works through
// its share of the list, to and fro (the list is sorted by length); loads, products and softmax run through it on their own.  A
// piece's queries are fetched as soon as the scores of the piece before are done, under its last product.
//
// What bounds it: a pair of query tiles takes 3,950 cycles a key tile, two softmaxes of 1,630 and what they wait for their scores, the
// products 2,112 (66 each, the full rate); a split piece takes 1.4 us a key tile, then behind memory.
//
// Every wait is bounded: a timeout records a code in g_shared_status, lets copies land, frees tensor memory and returns.
#pragma once
#include "tc_common.cuh"

namespace ftk {

__device__ int g_shared_status[4];  // [0] first error code, [1] block; 0 = fine

constexpr int kShRows = 128, kShKeys = 128, kShThreads = 384;   // a warpgroup of 2 loaders + 1 issuer (+ 1 idle), 2 x 4 softmax warps
constexpr int kShHalf = 128 * 64 * 2;                           // bytes of a [128 rows x 64 elements] column of 128-byte rows
constexpr int kShRegsFew = 72, kShRegsMany = 216;               // of 384 x 168: what 128 threads give, 256 take
constexpr int kShKStages(int d) { return d == 128 ? 3 : 5; }    // key and value tiles in flight: what fits beside the queries
constexpr int kShVStages(int d) { return d == 128 ? 2 : 5; }
constexpr int kShSmem(int d) { return (2 + kShKStages(d) + kShVStages(d)) * (d / 64) * kShHalf + 1024; }

// Exponentials: the special-function unit gives 16 an SM and cycle, 2,048 cycles for the 32,768 of a key tile and two query tiles, as much
// as the products take.  Of every eight columns kShPoly pairs go another way: 2^x = 2^n 2^r with n = x rounded to the nearest integer (by adding and
// taking off 1.5 2^23) and 2^r on [-1/2, 1/2] by a polynomial of degree four, the minimax fit of the relative error by Lawson's
// iteration (2.7e-6 evaluated in 32 bits; the probability is rounded to 2^-8 right behind), two numbers an instruction.  None, one and two
// of four pairs: 60.2, 58.3 and 60.1 us for 64 requests over nested spans, 26.9, 26.6 and 27.4 for 200 of heads of 64.
constexpr int kShPoly = 1;
__device__ __forceinline__ uint64_t sh_pair(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void sh_unpair(uint64_t p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p)); }
__device__ __forceinline__ uint64_t sh_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ float sh_max3(float a, float b, float c) {  // (NaN if one of them is)
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// 2^x of two numbers, x at most 100 or so; below -126 as for -126
__device__ __forceinline__ void sh_exp2_poly(uint64_t x, float& e0, float& e1) {
  float x0, x1, t0, t1;
  sh_unpair(x, x0, x1);
  x = sh_pair(fmaxf(x0, -126.f), fmaxf(x1, -126.f));
  const uint64_t magic = sh_pair(12582912.f, 12582912.f), back = sh_pair(-12582912.f, -12582912.f), minus = sh_pair(-1.f, -1.f);
  const uint64_t t = f2_add(x, magic), r = sh_fma2(f2_add(t, back), minus, x);
  uint64_t p = sh_pair(9.570101276e-03f, 9.570101276e-03f);
  p = sh_fma2(p, r, sh_pair(5.591785908e-02f, 5.591785908e-02f));
  p = sh_fma2(p, r, sh_pair(2.402474433e-01f, 2.402474433e-01f));
  p = sh_fma2(p, r, sh_pair(6.931217909e-01f, 6.931217909e-01f));
  p = sh_fma2(p, r, sh_pair(9.999992847e-01f, 9.999992847e-01f));
  sh_unpair(t, t0, t1);
  sh_unpair(p, e0, e1);
  e0 = __int_as_float(__float_as_int(e0) + (__float_as_int(t0) << 23));
  e1 = __int_as_float(__float_as_int(e1) + (__float_as_int(t1) << 23));
}

template <int N>
struct IntC {
  static constexpr int value = N;
};
template <int N> __device__ __forceinline__ void sh_regs_give() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void sh_regs_take() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }

// 32 columns of this thread's row: started; and the wait for every load so far, to which the registers are tied
__device__ __forceinline__ void sh_ld32(uint32_t addr, float* v) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr) : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
template <int N>
__device__ __forceinline__ void sh_ld_wait(float (&v)[N]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+f"(v[i]));
}
__device__ __forceinline__ void sh_st32(uint32_t addr, const float (&v)[32]) {
  const uint32_t* r = reinterpret_cast<const uint32_t*>(v);
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void sh_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
               ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
               : "memory");
}
__device__ __forceinline__ void sh_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 bytes of a row in one store: a whole sector
__device__ __forceinline__ void sh_store8(float* to, const float* v) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               ::"l"(to), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
}

template <int D>
__global__ void __launch_bounds__(kShThreads, 1)
shared_tc_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const __grid_constant__ SharedParams p) {
  constexpr int kHalves = D / 64, kTile = kHalves * kShHalf, kKStages = kShKStages(D), kVStages = kShVStages(D);
  constexpr uint32_t kLoaders = 8 * kHalves, kLoaderMask = (1u << kLoaders) - 1u;  // lanes of a loading warp: one per box
  extern __shared__ unsigned char dyn_smem[];
  __shared__ uint64_t q_full[2], o_free[2], k_full[kKStages], k_empty[kKStages], v_full[kVStages], v_empty[kVStages], s_full[2], p_full[2], pv_done[2];
  __shared__ uint32_t tmem_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int n_work = p.n_items * p.Hkv;
  const int n_rounds = (n_work + (int)gridDim.x - 1) / (int)gridDim.x;
  auto work_of = [&](int i) { return i * (int)gridDim.x + ((i & 1) ? (int)gridDim.x - 1 - (int)blockIdx.x : (int)blockIdx.x); };
  const uint32_t base = (smem_addr(dyn_smem) + 1023u) & ~1023u;
  unsigned char* tiles = dyn_smem + (base - smem_addr(dyn_smem));
  const uint32_t q_s = base, k_s = base + 2 * kTile, v_s = base + (2 + kKStages) * kTile;

  if (threadIdx.x == 0) {
    for (int s = 0; s < kKStages; ++s) {
      mbar_init(&k_full[s], 1); mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < kVStages; ++s) {
      mbar_init(&v_full[s], 1); mbar_init(&v_empty[s], 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&q_full[x], 4); mbar_init(&s_full[x], 1); mbar_init(&p_full[x], 4);
      mbar_init(&pv_done[x], 1); mbar_init(&o_free[x], 4);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) tmem_alloc(&tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp < 4) pdl_wait();  // (the softmax warps have something to do in front of it)
  if (warp == 1) pdl_trigger();  // (behind the wait: the kernel after this one counts on the one before being over)
  const uint32_t tmem = tmem_slot;
  volatile int* abortp = &abort_flag;
  const int G = p.G, tpt = kShRows / G;  // members of one query tile
  auto tiles_of = [](const Piece& it) { return it.ok ? (it.ke - it.kb + kShKeys - 1) / kShKeys : 0; };
  auto piece_of = [&](int w) {
    Piece it = load_piece(p, w / p.Hkv);
    it.ok = it.ok && it.n_mem <= 2 * tpt && it.kb % 16 == 0 &&
            (!it.split || (it.n_mem <= tpt && it.ke - it.kb > kShKeys && 2 * it.n_mem <= p.n_slots - it.slot0));
    return it;
  };
  auto fail = [&](int code) {
    atomicCAS(&g_shared_status[0], 0, code);
    abort_flag = 1;
  };

  if (warp < 4) {
    sh_regs_give<kShRegsFew>();  // (warp 3 only fills the warpgroup)
    if (warp == 0 || warp == 2) {
      // ---------------------------------------------------------- loaders: warp 0 keys, warp 2 values, a lane a box of 16 rows
      if (lane < kLoaders) {
        const int kv = warp == 2, box = lane / kHalves, h = lane % kHalves;
        const CUtensorMap* map = kv ? &map_v : &map_k;
        uint64_t* full = kv ? v_full : k_full;
        uint64_t* empty = kv ? v_empty : k_empty;
        unsigned char* stage0 = tiles + (kv ? 2 + kKStages : 2) * kTile + h * kShHalf + box * 2048;
        const int stages = kv ? kVStages : kKStages;
        bool ok = true;
        int g = 0;  // key tiles of all pieces so far
        for (int i = 0; i < n_rounds && ok; ++i) {
          const int w = work_of(i);
          if (w >= n_work) continue;
          const Piece it = piece_of(w);
          const int kvh = w % p.Hkv, n_tiles = tiles_of(it);
          const int32_t* bt = p.block_table + (size_t)it.bt_row * p.bt_stride;
          // this lane's page of tile j, looked up a tile ahead (a box begins anywhere on a multiple of 16 behind the piece's first key, which
          // is one itself, so it lies in one page)
          auto page_of = [&](int j) {
            const int key = it.kb + j * kShKeys + 16 * box;
            int page = 0;
            if (j < n_tiles && key < it.ke) {
              const int slot = key / p.P;
              page = slot < p.bt_stride ? bt[slot] : 0;
              if (page < 0 || page >= p.num_pages) page = 0;
            }
            return page;
          };
          int page_next = page_of(0);
          for (int j = 0; j < n_tiles && ok; ++j, ++g) {
            const int st = g % stages;
            const int key0 = it.kb + j * kShKeys;
            const int n_box = min(8, (it.ke - key0 + 15) >> 4);  // boxes that hold keys of the piece
            const int page = page_next;
            page_next = page_of(j + 1);
            const int row = (page * p.Hkv + kvh) * p.P + (key0 + 16 * box) % p.P;
            if (!__all_sync(kLoaderMask, mbar_wait(&empty[st], (uint32_t)((g / stages) & 1) ^ 1u, abortp))) {
              if (lane == 0) fail(801 + kv);
              ok = false;
              break;
            }
            if (lane == 0) mbar_expect_tx(&full[st], (uint32_t)n_box * kHalves * 2048);
            __syncwarp(kLoaderMask);
            if (box < n_box) tma_load_2d(stage0 + st * kTile, map, &full[st], h * 64, row);
          }
        }
      }
    } else if (warp == 1) {
      // ---------------------------------------------------------- issuer; the warp zeroes value rows past the piece's end
      // What a piece is comes through a shuffle: the compiler then knows that stages, parities and descriptors are the warp's, and
      // products leave one after the other.  (An issuing warp for each tile lets both tiles' softmax run at the same time and then wait for
      // the tensor pipe together: 2.05 us a key tile and pair against 1.70 where the keys are there.)
      constexpr uint32_t idesc_qk = instr_desc(kShKeys);
      constexpr uint32_t idesc_pv = instr_desc(D) | kMnMajorB;
      const uint64_t q_desc = smem_desc(q_s), k_desc = smem_desc(k_s), v_desc = smem_desc_mn(v_s, kShHalf);  // (addresses add to them, in 16-byte words)
      bool ok = true;
      int g0 = 0;           // key tiles of the pieces before this one
      int gx0 = 0, gx1 = 0;  // key tiles that query tile A, B has worked through, pieces it took part in
      int px0 = 0, px1 = 0;
      for (int i = 0; i < n_rounds && ok; ++i) {
        const int w = work_of(i);
        if (w >= n_work) continue;
        const Piece it = piece_of(w);
        const int n_tiles = __shfl_sync(0xffffffffu, tiles_of(it), 0), n_keys = __shfl_sync(0xffffffffu, it.ke - it.kb, 0);
        const bool split = __shfl_sync(0xffffffffu, (int)it.split, 0) != 0, two = __shfl_sync(0xffffffffu, it.n_mem, 0) > tpt;
        if (n_tiles == 0) continue;
        bool fine = true;  // this lane's waits; the warp votes on them once a key tile
        auto wait = [&](uint64_t* bar, int parity, int code) {
          if (!mbar_wait(bar, (uint32_t)(parity & 1), abortp)) { fail(code); fine = false; }
        };
        auto keys_there = [&](int j) { wait(&k_full[(g0 + j) % kKStages], (g0 + j) / kKStages, 803); };
        // the values of tile j are there; rows behind the piece's end are zeros then, whatever the page or the stage holds in them
        auto values_there = [&](int j) {
          const int vs = (g0 + j) % kVStages, live = n_keys - j * kShKeys;
          wait(&v_full[vs], (g0 + j) / kVStages, 805);
          if (live < kShKeys) {
            for (int z = lane; z < (kShKeys - live) * 8 * kHalves; z += 32) {
              const int r = live + z / (8 * kHalves), h = (z / 8) % kHalves, c = z & 7;
              *reinterpret_cast<uint4*>(tiles + (2 + kKStages + vs) * kTile + h * kShHalf + r * 128 + c * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
            fence_async_smem();
          }
        };
        // S_x = Q_x K(j)^T; `last`: no other query tile needs these keys
        auto scores = [&](auto xc, int j, bool last) {
          constexpr int x = decltype(xc)::value;
          const int ks = (g0 + j) % kKStages;
          __syncwarp();
          tc_fence_after();
          if (elect_one()) if (fine) {
            const uint64_t a = q_desc + x * (kTile >> 4), b = k_desc + ks * (kTile >> 4);
#pragma unroll
            for (int kk = 0; kk < 4 * kHalves; ++kk)  // 16 elements of the head dimension per product
              tc_mma(tmem + (uint32_t)(x * kShKeys), a + (kk >> 2) * (kShHalf >> 4) + 2 * (kk & 3), b + (kk >> 2) * (kShHalf >> 4) + 2 * (kk & 3),
                     idesc_qk, kk != 0);
            tc_commit(&s_full[x]);
            if (last) tc_commit(&k_empty[ks]);
          }
          __syncwarp();
        };
        // O_x += P_x V(j), the jj-th of this query tile in this piece
        auto product = [&](auto xc, int j, int jj, bool last) {
          constexpr int x = decltype(xc)::value;
          const int vs = (g0 + j) % kVStages;
          wait(&p_full[x], (x ? gx1 : gx0) + jj, 805);
          if (jj == 0) wait(&o_free[x], (x ? px1 : px0) + 1, 806);
          __syncwarp();
          tc_fence_after();
          if (elect_one()) if (fine) {
            const uint64_t b = v_desc + vs * (kTile >> 4);
#pragma unroll
            for (int kk = 0; kk < 8; ++kk)  // 16 keys per product
              tc_mma_ts(tmem + (uint32_t)((2 + x) * kShKeys), tmem + (uint32_t)(x * kShKeys + kk * 8), b + kk * (2048 >> 4), idesc_pv, (jj | kk) != 0);
            tc_commit(&pv_done[x]);
            if (last) tc_commit(&v_empty[vs]);
          }
          __syncwarp();
        };
        const IntC<0> A;
        const IntC<1> B;
        keys_there(0);
        wait(&q_full[0], px0, 804);
        scores(A, 0, split || !two);
        if (split) keys_there(1);
        if (split || two) {
          wait(&q_full[1], px1, 804);
          scores(B, split ? 1 : 0, true);
        }
        if (split) {
          for (int j = 0; j < n_tiles && ok; j += 2) {
            values_there(j);
            if (j + 2 < n_tiles) keys_there(j + 2);
            product(A, j, j >> 1, true);
            if (j + 2 < n_tiles) scores(A, j + 2, true);
            if (j + 1 < n_tiles) {
              values_there(j + 1);
              if (j + 3 < n_tiles) keys_there(j + 3);
              product(B, j + 1, j >> 1, true);
              if (j + 3 < n_tiles) scores(B, j + 3, true);
            }
            ok = all_of_warp(fine);
          }
        } else {
          for (int j = 0; j < n_tiles && ok; ++j) {
            const bool more = j + 1 < n_tiles;
            values_there(j);  // (what is waited for under the softmax anyway goes in front of the probabilities)
            if (more) keys_there(j + 1);
            product(A, j, j, !two);
            if (more) scores(A, j + 1, !two);
            if (two) {
              product(B, j, j, true);
              if (more) scores(B, j + 1, true);
            }
            ok = all_of_warp(fine);
          }
        }
        g0 += n_tiles;
        gx0 += split ? (n_tiles + 1) >> 1 : n_tiles;
        ++px0;
        if (split || two) {
          gx1 += split ? n_tiles >> 1 : n_tiles;
          ++px1;
        }
      }
    }
  } else {
    sh_regs_take<kShRegsMany>();
    // ------------------------------------------------------------ softmax and epilogue: warps 4..7 tile A, warps 8..11 tile B, a thread a row
    const int X = warp < 8 ? 0 : 1, quad = warp & 3, r = quad * 32 + lane;
    const float sl2 = p.scale * kLog2e;
    const uint32_t lane_addr = tmem + ((uint32_t)(quad * 32) << 16);
    const uint32_t s_addr = lane_addr + (uint32_t)(X * kShKeys);        // scores, then probabilities over their first half
    const uint32_t o_addr = lane_addr + (uint32_t)((2 + X) * kShKeys);
    // This warp's 32 rows of the queries of the first piece from round `i` on that has some for this tile, on their way to shared memory;
    // returns that round.  (A lane looks its own row's place up, all copies leave together: looked up copy by copy they took 17,000 cycles.)
    auto fetch_queries = [&](int i) {
      for (; i < n_rounds; ++i) {
        const int w = work_of(i);
        if (w >= n_work) continue;
        const Piece it = piece_of(w);
        if (!it.ok || (!it.split && it.n_mem <= X * tpt)) continue;
        const int mem0 = it.split ? 0 : X * tpt, R = min(tpt, it.n_mem - mem0) * G;
        const int tok = r < R ? p.members[it.mem0 + mem0 + r / G] : -1;
        const int row = tok >= 0 && tok < p.n_rows ? tok * p.Hq + w % p.Hkv * G + r % G : -1;  // of the queries' rows; -1: zeros
        constexpr int kPer = 8 * kHalves;  // 16-byte words of a row
        const int c = lane % kPer;
        unsigned char* to = tiles + X * kTile + (c >> 3) * kShHalf;
#pragma unroll 4
        for (int u = 0; u < 32; u += 32 / kPer) {
          const int mine = u + lane / kPer, rr = quad * 32 + mine, from = __shfl_sync(0xffffffffu, row, mine);
          if (rr < R)
            copy16(to + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), (const __nv_bfloat16*)p.q + (size_t)max(from, 0) * D + c * 8, from >= 0);
        }
        copy_commit();
        break;
      }
      return i;
    };
    auto queries_there = [&](int i) {
      if (i >= n_rounds) return;
      copy_wait<0>();
      fence_async_smem();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[X]);
    };
    bool ok = true;
    int gx = 0;  // key tiles this query tile has worked through
    // The first round is dry: a key tile's arithmetic on whatever tensor memory holds, which brings its instructions to the SM (7,000
    // cycles where they come from L2) while the kernel before this one ends and the first keys are on their way.
    bool dry = true;
    for (int i = -1; i < n_rounds && ok;) {
      const int w = dry ? 0 : work_of(i);
      Piece it = {};
      if (!dry) it = piece_of(w);
      const int kvh = w % p.Hkv, mem0 = it.split ? 0 : X * tpt, R = min(tpt, it.n_mem - mem0) * G;
      const int n_tiles = dry ? 1 : it.split ? (tiles_of(it) + 1 - X) >> 1 : tiles_of(it);  // this query tile's
      float m_used = -INFINITY, l = 0.f;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int g = gx + j;
        if (!dry && !__all_sync(0xffffffffu, mbar_wait(&s_full[X], (uint32_t)(g & 1), abortp))) {
          if (lane == 0) fail(807);
          ok = false;
          break;
        }
        tc_fence_after();
        float v[128];
        sh_ld32(s_addr, v);
        sh_ld32(s_addr + 32, v + 32);
        sh_ld32(s_addr + 64, v + 64);
        sh_ld32(s_addr + 96, v + 96);
        sh_ld_wait(v);
        const int live = it.ke - (it.kb + (it.split ? 2 * j + X : j) * kShKeys);
        if (live < kShKeys) {
#pragma unroll
          for (int n = 0; n < 128; ++n)
            if (n >= live) v[n] = -INFINITY;
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int n = 0; n < 128; n += 8)
#pragma unroll
          for (int e = 0; e < 4; ++e) mx4[e] = sh_max3(mx4[e], v[n + 2 * e], v[n + 2 * e + 1]);
        const float mx = sh_max3(sh_max3(mx4[0], mx4[1], mx4[2]), mx4[3], mx4[3]) * sl2;  // (the scale is positive)
        float alpha = 1.f;
        if (mx > m_used + 8.f || (m_used == -INFINITY && mx > -INFINITY)) {
          alpha = m_used == -INFINITY ? 0.f : exp2_fast(m_used - mx);
          m_used = mx;
        }
        l *= alpha;
        if (__any_sync(0xffffffffu, alpha != 1.f) && j > 0) {  // O must hold every product so far before it is scaled
          if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[X], (uint32_t)((g - 1) & 1), abortp))) {
            if (lane == 0) fail(809);
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            float o[32];
            sh_ld32(o_addr + c * 32, o);
            sh_ld_wait(o);
#pragma unroll
            for (int n = 0; n < 32; ++n) o[n] *= alpha;
            sh_st32(o_addr + c * 32, o);
            sh_st_wait();
          }
        }
        const float mb = m_used == -INFINITY ? 0.f : m_used;
        const uint64_t sl22 = sh_pair(sl2, sl2), mb2 = sh_pair(-mb, -mb);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          uint32_t pk[16];
#pragma unroll
          for (int n = 0; n < 32; n += 2) {
            const uint64_t x = sh_fma2(sh_pair(v[c * 32 + n], v[c * 32 + n + 1]), sl22, mb2);
            float e0, e1;
            if ((n >> 1 & 3) >= 4 - kShPoly) {
              sh_exp2_poly(x, e0, e1);
            } else {
              sh_unpair(x, e0, e1);
              e0 = exp2_fast(e0);  // (0 for keys that are not there)
              e1 = exp2_fast(e1);
            }
            sum2[n >> 1 & 1] = f2_add(sum2[n >> 1 & 1], sh_pair(e0, e1));
            pk[n >> 1] = two_bf16(e0, e1);
          }
          sh_st16(s_addr + (uint32_t)(c * 16), pk);
        }
        float sum, sum_odd;
        sh_unpair(f2_add(sum2[0], sum2[1]), sum, sum_odd);
        sum += sum_odd;
        if (!(mx < INFINITY)) sum = NAN;  // a score that is NaN or infinite: so is every output of the row
        l += sum;
        sh_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0 && !dry) mbar_arrive(&p_full[X]);
      }
      if (dry) pdl_wait();
      // the scores of the piece's last tile are done, so its queries have been read: the next piece's take their place
      const int next = ok ? fetch_queries(i + 1) : n_rounds;
      if (dry) {
        queries_there(next);
        dry = false;
        i = next;
        continue;
      }
      if (ok) {
        if (!__all_sync(0xffffffffu, mbar_wait(&pv_done[X], (uint32_t)((gx + n_tiles - 1) & 1), abortp))) {
          if (lane == 0) fail(808);
          ok = false;
        }
        tc_fence_after();
      }
      if (ok) {
        const size_t at = (size_t)(it.slot0 + (it.split ? X * it.n_mem : mem0) + r / G) * p.Hq + kvh * G + r % G;
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          float o[32];
          sh_ld32(o_addr + c * 32, o);
          sh_ld_wait(o);
          if (r < R) {
#pragma unroll
            for (int n = 0; n < 32; n += 8) sh_store8(p.part_o + at * D + c * 32 + n, o + n);
          }
        }
        if (r < R) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(l != l && m_used == -INFINITY ? 0.f : m_used, l);  // (NaN is not a row without keys)
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&o_free[X]);  // the next piece's first product may overwrite the output
      if (ok) queries_there(next);
      gx += n_tiles;
      i = next;
    }
  }
  // ---------------------------------------------------------------- teardown
  if (abort_flag) {
    if (threadIdx.x == 0) g_shared_status[1] = blockIdx.x;
    for (int i = 0; i < 2000; ++i) __nanosleep(100);  // let copies in flight land before the CTA leaves
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

inline bool shared_tc_fits(int head_dim, int page_size, int group) {
  return (head_dim == 64 || head_dim == 128) && page_size >= 16 && page_size % 16 == 0 && group >= 1 && group <= kShRows;
}

template <int D>
static int launch_shared_tc(const SharedParams& p, cudaStream_t s) {
  auto kern = shared_tc_kernel<D>;
  static OncePerDevice once;
  if (!once([&] { return set_shared_limit(kern, kShSmem(D)); })) return 2;
  CUtensorMap mk, mv;
  // a slab [pages, KV heads, P, D] seen as rows of D; a box is 16 rows of one page x 64 elements
  const uint64_t dims[2] = {(uint64_t)D, (uint64_t)p.num_pages * p.Hkv * p.P};
  const uint64_t strides[1] = {(uint64_t)D * 2};
  const uint32_t box[2] = {64, 16};
  if (!make_map(&mk, p.k, 2, dims, strides, box) || !make_map(&mv, p.v, 2, dims, strides, box)) return 4;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms < 1) return 5;
  const long long n_work = (long long)p.n_items * p.Hkv;
  FTK_LAUNCH(kern, (unsigned)(n_work < sms ? n_work : sms), kShThreads, kShSmem(D), s, mk, mv, p);
  return 0;
}

}  // namespace ftk
