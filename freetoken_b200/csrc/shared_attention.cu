// Attention of single tokens over paged keys and values where several requests share keys: the continuations of one prompt, or
// requests under one system prompt.
//
// Per query head, with keys j of the request (all of them lie before its token): o = sum_j p_j v_j / sum_j p_j, p_j = e^(scale q k_j - m).
// A set of keys that several requests share is read once, for all of their rows together; every piece of work leaves (m, l =
// sum p, unnormalised o) per row in 32 bits, and a request's pieces are joined: M = max m_i, o = sum o_i e^(m_i - M) / sum l_i e^(m_i - M).
// Sums, maxima and partial results stay in 32 bits; probabilities are rounded to bfloat16 in front of the product with bfloat16
// values (2^-8 of each at most, independent of one another: as far off as the rounding of the result itself).
//
// Two launches.  The first works through pieces of shared keys (engine/shared_plan.py cuts them): items of 8 int32 = first member,
// members, block-table row, first key, one past the last key, first slot, split, 0; members[] holds query rows; a member's partial results
// lie in slot (first slot + its number in the item).  The second has a cluster of CTAs per (request, KV head): it attends over the
// request's own keys, split over the cluster, and joins them with the request's slots in the order of its list, so results do not
// depend on which block came first.  requests[] = query row, block-table row, first own key, one past the last, first entry in joins[], entries, 0, 0.
//
//   * rows16 kernels: 16 query rows a CTA, bfloat16 on mma.sync (every head size that is a multiple of 16, any page size) or 32 bits
//     on the fma pipe.  The own keys of a request have no more rows than that (one request's heads on a KV head, 16 at a time), and
//     are bound by memory.
//   * shared_tc_kernel (shared_attention_tc.cuh): up to 256 query rows a CTA on tcgen05, for the shared keys of heads of 64 and 128.
//
// Measured, 48 heads on 8 of 128, cold: 8 requests over 2,048 shared keys and up to 300 of their own 15.7 us, 32 over 32,000 and up to 700
// 68 us (179 MB; with every request by itself it would be 4.3 GB); 64 over 4,096 and 16 prompts of 1,200 of four each 58 us.  The shared
// keys take 41 us of the 68 by themselves (3.2 TB/s from memory, the tensor pipe 0.45 busy: the softmax), the own ones 25.  Those are
// bound by a CTA's way from the list to the table, the keys, the other CTAs and the partial results, 6 us whatever it has to do: asking for
// the own keys under the shared ones brought nothing (71 us), neither did giving them to a launch in front (73).
#include <mma.h>

#include "common.cuh"

namespace ftk {

struct SharedParams {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  const int32_t* block_table;
  int bt_stride, bt_rows;
  const int32_t* items;
  int n_items;
  const int32_t* members;
  int n_members;
  const int32_t* requests;
  int n_requests;
  const int32_t* joins;
  int n_joins;
  float* part_o;
  float* part_ml;
  int n_slots;
  int n_rows, Hq, Hkv, G, D, P, num_pages;
  int Gc, chunks;  // query heads of one KV head that a rows16 CTA takes (G, 16 at most), and in how many chunks all are taken
  int page_shift;  // log2 of the page size, -1 where it is no power of two
  int cluster;     // CTAs that share a request's own keys
  int stages;      // places for tiles of 64 keys and values: three, or as many as a CTA's own keys take
  float scale;
  int has_sink;
  float sink;
  const float* sink_heads;
  int early;       // the second launch: the first one went in front of it, its partial results are waited for
};

// A piece's rows: row r is query head head0 + r % heads of query row tok(r / heads).
struct Rows {
  const int32_t* members;  // query rows, or null: tok0 for all
  int tok0, heads, head0, n;
  __device__ __forceinline__ int tok(int r) const { return members ? members[r / heads] : tok0; }
  __device__ __forceinline__ int head(int r) const { return head0 + r % heads; }
};

struct Piece {
  int mem0, n_mem, bt_row, kb, ke, slot0;
  bool split;  // (shared_attention_tc.cuh) the members' slots come twice: of even and of odd key tiles
  bool ok;
};
__device__ __forceinline__ Piece load_piece(const SharedParams& p, int idx) {
  const int32_t* w = p.items + (size_t)idx * 8;
  Piece it{w[0], w[1], w[2], w[3], w[4], w[5], w[6] != 0, false};
  it.ok = it.mem0 >= 0 && it.n_mem > 0 && it.n_mem <= p.n_members - it.mem0 && it.bt_row >= 0 && it.bt_row < p.bt_rows && it.kb >= 0 &&
          it.ke > it.kb && it.slot0 >= 0 && it.n_mem <= p.n_slots - it.slot0;
  return it;
}

// Row of key `pos` of block-table row `bt_row` among a slab's [pages, KV heads, P] rows of D, or -1 where the table names no page of it.
__device__ __forceinline__ int key_row(const SharedParams& p, int bt_row, int kvh, int pos) {
  const int block = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.P;
  if (block >= p.bt_stride) return -1;
  const int page = p.block_table[(size_t)bt_row * p.bt_stride + block];
  if (page < 0 || page >= p.num_pages) return -1;
  return (page * p.Hkv + kvh) * p.P + (pos - block * p.P);
}

__device__ __forceinline__ uint32_t sh_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy16(void* dst, const void* src, bool valid) {  // (zeros where there is nothing to copy)
  const int n = valid ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(sh_addr(dst)), "l"(src), "r"(n));
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;\n" ::); }
template <int N>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;\n" ::"n"(N)); }
__device__ __forceinline__ void matrix4(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(sh_addr(p)));
}
__device__ __forceinline__ void matrix4_trans(uint32_t (&r)[4], const void* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(sh_addr(p)));
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t two_bf16(float lo, float hi) {
  __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float kLog2e = 1.4426950408889634f;

// ================================================================= 16 query rows over keys [kb, ke)
// Both cores leave the rows' maxima m (bfloat16: of scores times log2 e; 32 bits: of scores), sums l and unnormalised outputs o
// [16][D] in shared memory, for all threads to read.
constexpr int kRows = 16, kRowThreads = 128;
struct RowsResult {
  float* m;
  float* l;
  float* o;
};

// ---- bfloat16: the four warps take 16 keys each of a tile of 64, three tiles on their way
constexpr int kTileKeys = 64, kTileStages = 3;
inline size_t rows16_bf16_smem(int d, int stages) {
  const size_t tiles = (size_t)(kRows + 2 * stages * kTileKeys) * (d + 8) * 2, merge = (size_t)(10 * kRows + 4 * kRows * d) * 4 + 16;
  return tiles > merge ? tiles : merge;
}

template <int DMAX, bool EXACT>
__device__ __forceinline__ RowsResult rows16_bf16(const SharedParams& p, const Rows& rw, int bt_row, int kvh, int kb, int ke, unsigned char* smem) {
  const int D = EXACT ? DMAX : p.D, ld = D + 8;  // (16 bytes more: ldmatrix without bank conflicts)
  __nv_bfloat16* sq = reinterpret_cast<__nv_bfloat16*>(smem);
  __nv_bfloat16* sk0 = sq + kRows * ld;
  __nv_bfloat16* sv0 = sk0 + p.stages * kTileKeys * ld;
  __shared__ int key_rows[4][kTileKeys];  // where the keys of tile t lie: key_rows[t & 3]
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pieces = D >> 3;
  const __nv_bfloat16* q = (const __nv_bfloat16*)p.q;
  const __nv_bfloat16* kbase = (const __nv_bfloat16*)p.k;
  const __nv_bfloat16* vbase = (const __nv_bfloat16*)p.v;

  auto look_up = [&](int t) -> int {
    const int pos = kb + t * kTileKeys + (int)threadIdx.x;
    return threadIdx.x < kTileKeys && pos < ke ? key_row(p, bt_row, kvh, pos) : -1;
  };
  auto publish = [&](int t, int row) {
    if (threadIdx.x < kTileKeys) key_rows[t & 3][threadIdx.x] = row;
  };
  auto load = [&](int t) {
    __nv_bfloat16* sk = sk0 + t % kTileStages * kTileKeys * ld;
    __nv_bfloat16* sv = sv0 + t % kTileStages * kTileKeys * ld;
    for (int i = threadIdx.x; i < kTileKeys * pieces; i += kRowThreads) {
      const int j = i / pieces, c = i - j * pieces;
      const int row = key_rows[t & 3][j];
      const bool there = row >= 0;
      const size_t o = (size_t)(there ? row : 0) * D + c * 8;
      copy16(sk + j * ld + c * 8, kbase + o, there);
      copy16(sv + j * ld + c * 8, vbase + o, there);
    }
  };
  int n_tiles = (ke - kb + kTileKeys - 1) / kTileKeys;
  if (p.stages < kTileStages) n_tiles = min(n_tiles, p.stages);  // (fewer places than three are given where they hold every key)
#pragma unroll
  for (int t = 0; t < 3; ++t) publish(t, look_up(t));
  for (int i = threadIdx.x; i < kRows * pieces; i += kRowThreads) {
    const int r = i / pieces, c = i - r * pieces, tok = r < rw.n ? rw.tok(r) : -1;
    const bool there = tok >= 0 && tok < p.n_rows;
    copy16(sq + r * ld + c * 8, q + (there ? ((size_t)tok * p.Hq + rw.head(r)) * D + c * 8 : 0), there);
  }
  __syncthreads();
  if (n_tiles > 0) load(0);
  copy_commit();
  if (n_tiles > 1) load(1);
  copy_commit();

  const int r0 = lane >> 2, r1 = r0 + 8;
  const float sl2 = p.scale * kLog2e;
  float o[DMAX / 8][4];
#pragma unroll
  for (int i = 0; i < DMAX / 8; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
  for (int t = 0; t < n_tiles; ++t) {
    copy_wait<1>();
    __syncthreads();  // tile t has landed for everyone, and everyone is done with tile t - 1
    if (t + 2 < n_tiles) load(t + 2);
    copy_commit();
    const int next = look_up(t + 3);
    if (kb + t * kTileKeys + warp * 16 >= ke) {  // (none of this warp's keys is there)
      publish(t + 3, next);
      continue;
    }
    const __nv_bfloat16* sk = sk0 + (t % kTileStages * kTileKeys + warp * 16) * ld;  // this warp's keys
    const __nv_bfloat16* sv = sv0 + (t % kTileStages * kTileKeys + warp * 16) * ld;
    float s[2][4] = {};
#pragma unroll
    for (int kk = 0; kk < DMAX / 16; ++kk) {
      if (kk * 16 >= D) break;
      uint32_t a[4], b[4];
      matrix4(a, sq + (lane & 15) * ld + kk * 16 + (lane >> 4) * 8);
      matrix4(b, sk + ((lane & 7) + ((lane >> 4) << 3)) * ld + kk * 16 + ((lane >> 3) & 1) * 8);
      mma16816(s[0], a, b[0], b[1]);
      mma16816(s[1], a, b[2], b[3]);
    }
    // keys past the end or without a page are not there for any row
    const int j0 = warp * 16 + (lane & 3) * 2;
    float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const bool there = key_rows[t & 3][j0 + n * 8 + e] >= 0;
        s[n][e] = there ? s[n][e] * sl2 : -INFINITY;
        s[n][2 + e] = there ? s[n][2 + e] * sl2 : -INFINITY;
        mx0 = fmaxf(mx0, s[n][e]);
        mx1 = fmaxf(mx1, s[n][2 + e]);
      }
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1));
    mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1));
    mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
    const float mn0 = fmaxf(m0, mx0), mn1 = fmaxf(m1, mx1);
    const float b0 = mn0 == -INFINITY ? 0.f : mn0, b1 = mn1 == -INFINITY ? 0.f : mn1;
    const float c0 = m0 == -INFINITY ? 0.f : exp2_fast(m0 - b0), c1 = m1 == -INFINITY ? 0.f : exp2_fast(m1 - b1);
    m0 = mn0;
    m1 = mn1;
    float sum0 = 0.f, sum1 = 0.f;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      s[n][0] = exp2_fast(s[n][0] - b0); s[n][1] = exp2_fast(s[n][1] - b0);
      s[n][2] = exp2_fast(s[n][2] - b1); s[n][3] = exp2_fast(s[n][3] - b1);
      sum0 += s[n][0] + s[n][1];
      sum1 += s[n][2] + s[n][3];
    }
    l0 = l0 * c0 + sum0;  // (this thread's quarter of the row's keys)
    l1 = l1 * c1 + sum1;
    uint32_t a[4];
    a[0] = two_bf16(s[0][0], s[0][1]);
    a[1] = two_bf16(s[0][2], s[0][3]);
    a[2] = two_bf16(s[1][0], s[1][1]);
    a[3] = two_bf16(s[1][2], s[1][3]);
    if (__any_sync(0xffffffffu, c0 != 1.f || c1 != 1.f)) {  // (the maximum rarely moves once a few tiles are in)
#pragma unroll
      for (int i = 0; i < DMAX / 8; ++i) {
        o[i][0] *= c0; o[i][1] *= c0;
        o[i][2] *= c1; o[i][3] *= c1;
      }
    }
#pragma unroll
    for (int d2 = 0; d2 < DMAX / 16; ++d2) {
      if (d2 * 16 >= D) break;
      uint32_t b[4];
      matrix4_trans(b, sv + (lane & 15) * ld + d2 * 16 + (lane >> 4) * 8);
      mma16816(o[2 * d2], a, b[0], b[1]);
      mma16816(o[2 * d2 + 1], a, b[2], b[3]);
    }
    publish(t + 3, next);  // read behind the next tile's barrier
  }
  copy_wait<0>();
  l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
  l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
  l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
  __syncthreads();  // the tiles are free: the four warps' results take their place
  float* rm = reinterpret_cast<float*>(smem);  // the result's maxima and sums, then each warp's
  float* rl = rm + kRows;
  float* wm = rl + kRows;
  float* wl = wm + 4 * kRows;
  float* wo = wl + 4 * kRows;
  // (a NaN among scores that are all NaN or not there has no maximum: it must not look like a row without keys)
  if (l0 != l0 && m0 == -INFINITY) m0 = 0.f;
  if (l1 != l1 && m1 == -INFINITY) m1 = 0.f;
  if ((lane & 3) == 0) {
    wm[warp * kRows + r0] = m0; wm[warp * kRows + r1] = m1;
    wl[warp * kRows + r0] = l0; wl[warp * kRows + r1] = l1;
  }
#pragma unroll
  for (int i = 0; i < DMAX / 8; ++i) {
    if (i * 8 >= D) break;
    const int d = i * 8 + (lane & 3) * 2;
    *reinterpret_cast<float2*>(wo + (warp * kRows + r0) * D + d) = make_float2(o[i][0], o[i][1]);
    *reinterpret_cast<float2*>(wo + (warp * kRows + r1) * D + d) = make_float2(o[i][2], o[i][3]);
  }
  __syncthreads();
  const int quads = D >> 2;
  for (int i = threadIdx.x; i < rw.n * quads; i += kRowThreads) {
    const int r = i / quads;
    float mw[4], M = -INFINITY, L = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      mw[w] = wm[w * kRows + r];
      M = fmaxf(M, mw[w]);
    }
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float f = mw[w] == -INFINITY ? 0.f : exp2_fast(mw[w] - M);
      const float4 x = *reinterpret_cast<const float4*>(wo + w * kRows * D + i * 4);
      L += wl[w * kRows + r] * f;
      acc.x += x.x * f; acc.y += x.y * f; acc.z += x.z * f; acc.w += x.w * f;
    }
    *reinterpret_cast<float4*>(wo + i * 4) = acc;
    if (i == r * quads) {
      rm[r] = M;
      rl[r] = L;
    }
  }
  __syncthreads();
  return {rm, rl, wo};
}

// ---- 32 bits: a warp has four rows, a lane a key of a tile of 32 for the scores and every 32nd column for the products
constexpr int kF32Keys = 32;
inline size_t rows16_f32_smem(int d) { return ((size_t)kRows * d + 4 * kF32Keys * (d + 4) + 2 * kRows) * 4; }

template <int DMAX, bool EXACT>
__device__ __forceinline__ RowsResult rows16_f32(const SharedParams& p, const Rows& rw, int bt_row, int kvh, int kb, int ke, unsigned char* smem) {
  constexpr int COLS = DMAX / 32, RW = kRows / 4;
  const int D = EXACT ? DMAX : p.D, ld = D + 4;
  float* rm = reinterpret_cast<float*>(smem);
  float* rl = rm + kRows;
  float* sq = rl + kRows;             // [16][D] queries, in the end the outputs
  float* sk0 = sq + kRows * D;        // two tiles of keys, two of values
  float* sv0 = sk0 + 2 * kF32Keys * ld;
  __shared__ int key_rows[4][kF32Keys];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, pieces = D >> 2;
  const float* q = (const float*)p.q;
  const float* kbase = (const float*)p.k;
  const float* vbase = (const float*)p.v;
  auto look_up = [&](int t) -> int {
    const int pos = kb + t * kF32Keys + (int)threadIdx.x;
    return threadIdx.x < kF32Keys && pos < ke ? key_row(p, bt_row, kvh, pos) : -1;
  };
  auto publish = [&](int t, int row) {
    if (threadIdx.x < kF32Keys) key_rows[t & 3][threadIdx.x] = row;
  };
  auto load = [&](int t) {
    float* sk = sk0 + (t & 1) * kF32Keys * ld;
    float* sv = sv0 + (t & 1) * kF32Keys * ld;
    for (int i = threadIdx.x; i < kF32Keys * pieces; i += kRowThreads) {
      const int j = i / pieces, c = i - j * pieces;
      const int row = key_rows[t & 3][j];
      const bool there = row >= 0;
      const size_t o = (size_t)(there ? row : 0) * D + c * 4;
      copy16(sk + j * ld + c * 4, kbase + o, there);
      copy16(sv + j * ld + c * 4, vbase + o, there);
    }
  };
  const int n_tiles = (ke - kb + kF32Keys - 1) / kF32Keys;
  publish(0, look_up(0));
  publish(1, look_up(1));
  for (int i = threadIdx.x; i < kRows * pieces; i += kRowThreads) {
    const int r = i / pieces, c = i - r * pieces, tok = r < rw.n ? rw.tok(r) : -1;
    const bool there = tok >= 0 && tok < p.n_rows;
    copy16(sq + r * D + c * 4, q + (there ? ((size_t)tok * p.Hq + rw.head(r)) * D + c * 4 : 0), there);
  }
  __syncthreads();
  if (n_tiles > 0) load(0);
  copy_commit();
  float acc[RW][COLS], m[RW], l[RW];
#pragma unroll
  for (int e = 0; e < RW; ++e) {
    m[e] = -INFINITY;
    l[e] = 0.f;
#pragma unroll
    for (int i = 0; i < COLS; ++i) acc[e][i] = 0.f;
  }
  const bool any = warp * RW < rw.n;
  for (int t = 0; t < n_tiles; ++t) {
    const int next = look_up(t + 2);
    if (t + 1 < n_tiles) load(t + 1);
    copy_commit();
    copy_wait<1>();
    __syncthreads();  // tile t has landed for everyone
    const float* sk = sk0 + (t & 1) * kF32Keys * ld;
    const float* sv = sv0 + (t & 1) * kF32Keys * ld;
    if (any) {
      const bool there = key_rows[t & 3][lane] >= 0;
      float dot[RW] = {};
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        const float4 b = *reinterpret_cast<const float4*>(sk + lane * ld + d);
#pragma unroll
        for (int e = 0; e < RW; ++e) {
          const float4 a = *reinterpret_cast<const float4*>(sq + (warp * RW + e) * D + d);
          dot[e] = fmaf(a.x, b.x, dot[e]);
          dot[e] = fmaf(a.y, b.y, dot[e]);
          dot[e] = fmaf(a.z, b.z, dot[e]);
          dot[e] = fmaf(a.w, b.w, dot[e]);
        }
      }
      float pj[RW];
#pragma unroll
      for (int e = 0; e < RW; ++e) {
        const float s = there ? dot[e] * p.scale : -INFINITY;
        const float m_new = fmaxf(m[e], warp_max(s));
        const float base = m_new == -INFINITY ? 0.f : m_new;
        const float corr = m[e] == -INFINITY ? 0.f : expf(m[e] - base);
        pj[e] = there ? expf(s - base) : 0.f;
        l[e] = l[e] * corr + warp_sum(pj[e]);
        m[e] = m_new;
#pragma unroll
        for (int i = 0; i < COLS; ++i) acc[e][i] *= corr;
      }
      const int nk = min(kF32Keys, ke - kb - t * kF32Keys);
#pragma unroll 2
      for (int j = 0; j < nk; ++j) {
        float x[COLS];
#pragma unroll
        for (int i = 0; i < COLS; ++i) x[i] = lane + 32 * i < D ? sv[j * ld + lane + 32 * i] : 0.f;
#pragma unroll
        for (int e = 0; e < RW; ++e) {
          const float pb = __shfl_sync(0xffffffffu, pj[e], j);
#pragma unroll
          for (int i = 0; i < COLS; ++i) acc[e][i] = fmaf(pb, x[i], acc[e][i]);
        }
      }
    }
    publish(t + 2, next);
    __syncthreads();
  }
  copy_wait<0>();
  __syncthreads();
  for (int e = 0; e < RW; ++e) {
    const int r = warp * RW + e;
    float me = 0.f, le = 0.f;
#pragma unroll
    for (int f = 0; f < RW; ++f)
      if (f == e) {
        me = m[f];
        le = l[f];
#pragma unroll
        for (int i = 0; i < COLS; ++i)
          if (lane + 32 * i < D) sq[r * D + lane + 32 * i] = acc[f][i];
      }
    if (lane == 0) {
      rm[r] = le != le && me == -INFINITY ? 0.f : me;  // (NaN is not a row without keys)
      rl[r] = le;
    }
  }
  __syncthreads();
  return {rm, rl, sq};
}

// EXACT: the head size is DMAX itself, so that rows are taken apart by shifts (a CTA with a few keys is bound by its instructions)
template <typename T, int DMAX, bool EXACT>
__device__ __forceinline__ RowsResult rows16(const SharedParams& p, const Rows& rw, int bt_row, int kvh, int kb, int ke, unsigned char* smem) {
  if constexpr (sizeof(T) == 2) return rows16_bf16<DMAX, EXACT>(p, rw, bt_row, kvh, kb, ke, smem);
  else return rows16_f32<DMAX, EXACT>(p, rw, bt_row, kvh, kb, ke, smem);
}
// maxima are of scores times log2 e in bfloat16, of scores in 32 bits
template <typename T>
__device__ __forceinline__ float weight(float m, float M) {
  if (m == -INFINITY) return 0.f;
  return sizeof(T) == 2 ? exp2f(m - M) : expf(m - M);
}

// ================================================================= shared keys, 16 rows a CTA
template <typename T, int DMAX, bool EXACT>
__global__ void __launch_bounds__(kRowThreads) shared_rows_kernel(const __grid_constant__ SharedParams p) {
  pdl_wait();
  pdl_trigger();
  extern __shared__ __align__(16) unsigned char smem[];
  const Piece it = load_piece(p, blockIdx.x);
  const int kvh = blockIdx.y / p.chunks, chunk = blockIdx.y - kvh * p.chunks;
  const int heads = min(p.Gc, p.G - chunk * p.Gc);
  if (!it.ok || it.n_mem * heads > kRows) return;
  const Rows rw{p.members + it.mem0, 0, heads, kvh * p.G + chunk * p.Gc, it.n_mem * heads};
  const RowsResult res = rows16<T, DMAX, EXACT>(p, rw, it.bt_row, kvh, it.kb, it.ke, smem);
  const int D = EXACT ? DMAX : p.D, quads = D >> 2;
  for (int i = threadIdx.x; i < rw.n * quads; i += kRowThreads) {
    const int r = i / quads, d = i % quads * 4;
    const size_t at = (size_t)(it.slot0 + r / heads) * p.Hq + rw.head(r);
    *reinterpret_cast<float4*>(p.part_o + at * D + d) = *reinterpret_cast<const float4*>(res.o + r * D + d);
    if (d == 0) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(res.m[r], res.l[r]);
  }
}

// ================================================================= a request's own keys, joined with the shared ones
__device__ __forceinline__ uint32_t of_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr));
  return v;
}
__device__ __forceinline__ float4 cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T>
__device__ __forceinline__ void store4(T* to, float4 v) {
  if constexpr (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = v;
  else *reinterpret_cast<uint2*>(to) = make_uint2(two_bf16(v.x, v.y), two_bf16(v.z, v.w));
}

constexpr int kJoinRun = 32;  // partial results that are weighed together, one a lane

template <typename T, int DMAX, bool EXACT>
__global__ void __launch_bounds__(kRowThreads, DMAX <= 128 ? 4 : 2) own_keys_kernel(const __grid_constant__ SharedParams p) {
  // With shared pieces in front of it this kernel starts while they run: queries, keys and values were written in front of them,
  // and only their partial results are waited for.
  if (!p.early) pdl_wait();
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ int slots[kJoinRun];
  __shared__ float weights[kJoinRun][kRows], before[kRows], norm[kRows];  // of a run's partial results; of what was summed up in front of it
  const int C = p.cluster, rank = blockIdx.x % C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  int work = blockIdx.x / C;
  const int chunk = work % p.chunks;
  work /= p.chunks;
  const int kvh = work % p.Hkv, req = work / p.Hkv;
  const int32_t* w = p.requests + (size_t)req * 8;
  const int tok = w[0], bt_row = w[1], from = w[2], to = w[3], join0 = w[4];
  const int heads = min(p.Gc, p.G - chunk * p.Gc), head0 = kvh * p.G + chunk * p.Gc;
  const bool ok = tok >= 0 && tok < p.n_rows && bt_row >= 0 && bt_row < p.bt_rows && from >= 0 && join0 >= 0 && w[5] >= 0 && w[5] <= p.n_joins - join0;
  const int n_join = ok ? w[5] : 0;
  // this CTA's share of the keys, in whole tiles
  const int tile = sizeof(T) == 2 ? kTileKeys : kF32Keys;
  const int own = ok ? max(0, to - from) : 0, share = ((own + C - 1) / C + tile - 1) / tile * tile;
  const int kb = from + min(own, rank * share), ke = from + min(own, rank * share + share);
  const Rows rw{nullptr, tok, heads, head0, ok ? heads : 0};
  const RowsResult res = rows16<T, DMAX, EXACT>(p, rw, bt_row, kvh, kb, ke, smem);
  if (C > 1) cluster_barrier();
  const uint32_t my_m = sh_addr(res.m), my_l = sh_addr(res.l), my_o = sh_addr(res.o);  // (at the same place in every CTA)
  if (p.early) pdl_wait();
  pdl_trigger();
  // All partial results of the request: the shared pieces' in their order, then the cluster's.  A run of 32 at a time a warp weighs a row's,
  // a lane each; then every thread sums up four columns of a row (the rows' 32-bit results are spread over the cluster).
  const int D = EXACT ? DMAX : p.D;
  constexpr int kQuads = DMAX * kRows / 4 / kRowThreads;
  const int quads = D >> 2, at0 = rank * kRowThreads + tid, parts = rw.n ? n_join + C : 0;
  float4 acc[kQuads];
#pragma unroll
  for (int u = 0; u < kQuads; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
  float M[kRows / 4], L[kRows / 4];  // of rows warp, warp + 4, ...
#pragma unroll
  for (int e = 0; e < kRows / 4; ++e) {
    M[e] = -INFINITY;
    L[e] = 0.f;
  }
  for (int j0 = 0; j0 < parts; j0 += kJoinRun) {
    const int n = min(kJoinRun, parts - j0), n_slots = max(0, min(n, n_join - j0)), part = j0 + lane;
    int slot = part < n_join ? p.joins[join0 + part] : -1;
    if (slot >= p.n_slots) slot = -1;
    if (warp == 0) slots[lane] = slot;
#pragma unroll
    for (int e = 0; e < kRows / 4; ++e) {
      const int r = warp + 4 * e;
      if (r >= heads) break;
      float2 ml = make_float2(-INFINITY, 0.f);
      if (slot >= 0) ml = __ldcg(reinterpret_cast<const float2*>(p.part_ml + ((size_t)slot * p.Hq + head0 + r) * 2));
      else if (part >= n_join && lane < n)
        ml = C > 1 ? make_float2(cluster_f32(of_rank(my_m + r * 4, part - n_join)), cluster_f32(of_rank(my_l + r * 4, part - n_join))) : make_float2(res.m[r], res.l[r]);
      const float m = fmaxf(M[e], warp_max(ml.x)), f = weight<T>(M[e], m), wgt = weight<T>(ml.x, m);
      L[e] = L[e] * f + warp_sum(ml.y * wgt);  // (a part that holds a NaN has a sum of NaN, whatever it weighs)
      M[e] = m;
      weights[lane][r] = wgt;
      if (lane == 0) {
        before[r] = f;
        if (j0 + kJoinRun >= parts) {  // the last run; a sink is a key without a value, and a row of nothing else gives zeros
          float sum = L[e];
          if (p.has_sink && m != -INFINITY) sum += expf((p.sink_heads ? __ldg(p.sink_heads + head0 + r) : p.sink) - (sizeof(T) == 2 ? m / kLog2e : m));
          norm[r] = sum == 0.f ? 0.f : 1.f / sum;  // (NaN stays)
        }
      }
    }
    __syncthreads();
    // a batch of pieces for all of the thread's columns: every load is on its way before the first use
    constexpr int kBatch = kQuads > 4 ? 2 : kQuads > 2 ? 4 : 8;
    if (j0 > 0) {
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const int i = at0 + u * C * kRowThreads;
        if (i >= rw.n * quads) break;
        const float f = before[i / quads];
        acc[u].x *= f; acc[u].y *= f; acc[u].z *= f; acc[u].w *= f;
      }
    }
    auto add = [&](int u, float f, float4 x) {  // (a part of weight 0 too: 0 x NaN is NaN, as it is within a part)
      acc[u].x = fmaf(x.x, f, acc[u].x); acc[u].y = fmaf(x.y, f, acc[u].y);
      acc[u].z = fmaf(x.z, f, acc[u].z); acc[u].w = fmaf(x.w, f, acc[u].w);
    };
#pragma unroll 1
    for (int j = 0; j < n_slots; j += kBatch) {
      float4 x[kQuads][kBatch];
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const int i = at0 + u * C * kRowThreads;
        if (i >= rw.n * quads) break;
        const float* o = p.part_o + (size_t)(head0 + i / quads) * D + i % quads * 4;
#pragma unroll
        for (int e = 0; e < kBatch; ++e) {
          const int at = slots[(j + e) % kJoinRun];
          x[u][e] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (j + e < n_slots && at >= 0) x[u][e] = __ldcg(reinterpret_cast<const float4*>(o + (size_t)at * p.Hq * D));
        }
      }
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const int i = at0 + u * C * kRowThreads;
        if (i >= rw.n * quads) break;
#pragma unroll
        for (int e = 0; e < kBatch; ++e)
          if (j + e < n_slots) add(u, weights[(j + e) % kJoinRun][i / quads], x[u][e]);
      }
    }
#pragma unroll 1
    for (int j = n_slots; j < n; ++j) {  // the cluster's
#pragma unroll
      for (int u = 0; u < kQuads; ++u) {
        const int i = at0 + u * C * kRowThreads;
        if (i >= rw.n * quads) break;
        add(u, weights[j][i / quads], C > 1 ? cluster_f32x4(of_rank(my_o + i * 16, j0 + j - n_join)) : *reinterpret_cast<const float4*>(res.o + i * 4));
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int u = 0; u < kQuads; ++u) {
    const int i = at0 + u * C * kRowThreads;
    if (i >= rw.n * quads) break;
    const float f = norm[i / quads];
    store4((T*)p.out + ((size_t)tok * p.Hq + head0) * D + i * 4, make_float4(acc[u].x * f, acc[u].y * f, acc[u].z * f, acc[u].w * f));
  }
  if (C > 1) cluster_barrier();  // nobody leaves while its shared memory is read
}

template <typename T>
static size_t rows_smem(int d, int stages) {
  if constexpr (sizeof(T) == 2) return rows16_bf16_smem(d, stages);
  else return rows16_f32_smem(d);
}

template <typename T, int DMAX, bool EXACT>
static int launch_shared_rows(const SharedParams& p, cudaStream_t s) {
  auto kern = shared_rows_kernel<T, DMAX, EXACT>;
  static OncePerDevice once;
  if (!once([&] { return set_shared_limit(kern, rows_smem<T>(DMAX, kTileStages)); })) return 2;
  const size_t smem = rows_smem<T>(p.D, p.stages);
  FTK_LAUNCH(kern, dim3(p.n_items, p.Hkv * p.chunks), kRowThreads, smem, s, p);
  return 0;
}
template <typename T, int DMAX, bool EXACT>
static int launch_own_keys(const SharedParams& p, cudaStream_t s) {
  auto kern = own_keys_kernel<T, DMAX, EXACT>;
  static OncePerDevice once;
  if (!once([&] { return set_shared_limit(kern, rows_smem<T>(DMAX, kTileStages)); })) return 2;
  const size_t smem = rows_smem<T>(p.D, p.stages);
  const dim3 grid((unsigned)(p.n_requests * p.Hkv * p.chunks * p.cluster));
  if (p.cluster > 1) launch_kernel_clusters(kern, p.cluster, grid, dim3(kRowThreads), smem, s, p);
  else FTK_LAUNCH(kern, grid, kRowThreads, smem, s, p);
  return 0;
}

template <typename T>
static int launch_rows(const SharedParams& p, cudaStream_t s) {
  return p.D == 64 ? launch_shared_rows<T, 64, true>(p, s) : p.D == 128 ? launch_shared_rows<T, 128, true>(p, s)
         : p.D < 128 ? launch_shared_rows<T, 128, false>(p, s) : launch_shared_rows<T, 256, false>(p, s);
}
template <typename T>
static int launch_own(const SharedParams& p, cudaStream_t s) {
  return p.D == 64 ? launch_own_keys<T, 64, true>(p, s) : p.D == 128 ? launch_own_keys<T, 128, true>(p, s)
         : p.D < 128 ? launch_own_keys<T, 128, false>(p, s) : launch_own_keys<T, 256, false>(p, s);
}

}  // namespace ftk

#include "shared_attention_tc.cuh"

using namespace ftk;

namespace ftk {
int shared_attention_status(int* out) { return take_status(g_shared_status, out); }  // (merged into ftk_read_status)
int shared_attention_set_status(int code) { return set_status(g_shared_status, code); }
}  // namespace ftk

extern "C" int ftk_shared_attention_tc_fits(int head_dim, int page_size, int group) { return shared_tc_fits(head_dim, page_size, group) ? 1 : 0; }

extern "C" int ftk_shared_attention(const FtkShared* a, void* stream) {
  FTK_REQUIRE(a, "shared_attention: null pointer");
  FTK_REQUIRE(dtype_ok(a->dtype), "shared_attention: bad dtype %d", a->dtype);
  FTK_REQUIRE(a->n_requests >= 0 && a->n_items >= 0 && a->n_members >= 0 && a->n_joins >= 0 && a->n_slots >= 0, "shared_attention: bad counts");
  if (a->n_requests == 0) return 0;
  FTK_REQUIRE(a->q && a->k && a->v && a->out && a->block_table && a->requests, "shared_attention: null pointer");
  FTK_REQUIRE(a->n_items == 0 || (a->items && a->members && a->joins && a->part_o && a->part_ml), "shared_attention: shared pieces need members, joins and scratch");
  FTK_REQUIRE(a->n_kv_heads >= 1 && a->n_q_heads >= 1 && a->n_q_heads % a->n_kv_heads == 0 && a->n_q_heads <= 65535, "shared_attention: %d query heads, %d KV heads",
              a->n_q_heads, a->n_kv_heads);
  FTK_REQUIRE(a->head_dim >= 16 && a->head_dim <= 256 && a->head_dim % 16 == 0, "shared_attention: head_dim=%d must be a multiple of 16 in [16, 256]", a->head_dim);
  FTK_REQUIRE(a->page_size >= 1 && a->num_pages >= 1 && a->bt_stride >= 1 && a->bt_rows >= 1 && a->n_rows >= 1, "shared_attention: bad geometry");
  FTK_REQUIRE((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out | (uintptr_t)a->part_o | (uintptr_t)a->part_ml) & 15) == 0,
              "shared_attention: 16-byte aligned tensors only");
  FTK_REQUIRE(a->cluster == 1 || a->cluster == 2 || a->cluster == 4 || a->cluster == 8, "shared_attention: clusters of 1, 2, 4 or 8 CTAs, got %d", a->cluster);
  SharedParams p = {};
  p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out;
  p.block_table = a->block_table; p.bt_stride = a->bt_stride; p.bt_rows = a->bt_rows;
  p.items = a->items; p.n_items = a->n_items; p.members = a->members; p.n_members = a->n_members;
  p.requests = a->requests; p.n_requests = a->n_requests; p.joins = a->joins; p.n_joins = a->n_joins;
  p.part_o = a->part_o; p.part_ml = a->part_ml; p.n_slots = a->n_slots;
  p.n_rows = a->n_rows; p.Hq = a->n_q_heads; p.Hkv = a->n_kv_heads; p.G = p.Hq / p.Hkv; p.D = a->head_dim; p.P = a->page_size;
  p.num_pages = a->num_pages;
  p.Gc = p.G < kRows ? p.G : kRows;
  p.chunks = (p.G + p.Gc - 1) / p.Gc;
  p.cluster = a->cluster;
  p.scale = a->scale; p.has_sink = a->has_sink; p.sink = a->sink; p.sink_heads = a->sink_heads;
  p.stages = kTileStages;
  p.page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (p.P == 1 << i) p.page_shift = i;
  p.early = a->n_items > 0;
  FTK_REQUIRE((long long)p.Hkv * p.chunks <= 65535 && (long long)p.n_requests * p.Hkv * p.chunks * p.cluster <= 0x7fffffffLL, "shared_attention: %d requests of %d KV heads",
              p.n_requests, p.Hkv);
  FTK_REQUIRE((long long)p.num_pages * p.Hkv * p.P <= 0x7fffffffLL, "shared_attention: a slab of 2^31 rows or more");
  cudaStream_t s = (cudaStream_t)stream;
  const int D = p.D;
  int rc = 0;
  if (p.n_items > 0) {
    const bool tc = a->tile_rows == 2 * kShRows;
    FTK_REQUIRE(tc || a->tile_rows == kRows, "shared_attention: pieces of %d query rows are not taken", a->tile_rows);
    FTK_REQUIRE(!tc || (a->dtype == FTK_BF16 && shared_tc_fits(D, p.P, p.G) && p.scale > 0.f),
                "shared_attention: pieces of 256 rows take bfloat16 heads of 64 or 128, pages of a multiple of 16, at most 128 heads per KV head and a positive scale");
    FTK_REQUIRE(!tc || ((uintptr_t)a->part_o & 31) == 0, "shared_attention: partial results on 32-byte boundaries only");
    note_variant(tc ? "shared attention: tcgen05, 256 rows" : a->dtype == FTK_F32 ? "shared attention: float32, 16 rows" : "shared attention: bfloat16 mma.sync, 16 rows");
    if (tc) rc = D == 64 ? launch_shared_tc<64>(p, s) : launch_shared_tc<128>(p, s);
    else rc = a->dtype == FTK_F32 ? launch_rows<float>(p, s) : launch_rows<__nv_bfloat16>(p, s);
    FTK_REQUIRE(rc == 0, "shared_attention: cannot set up the kernel for shared keys (%d)", rc);
    FTK_LAUNCH_CHECK("shared_attention");
  }
  if (a->own_tiles < kTileStages) p.stages = a->own_tiles > 1 ? a->own_tiles : 1;
  note_variant(a->dtype == FTK_F32 ? "shared attention: float32, own keys" : "shared attention: bfloat16 mma.sync, own keys");
  rc = a->dtype == FTK_F32 ? launch_own<float>(p, s) : launch_own<__nv_bfloat16>(p, s);
  FTK_REQUIRE(rc == 0, "shared_attention: cannot set up the kernel for own keys (%d)", rc);
  FTK_LAUNCH_CHECK("shared_attention (own keys)");
  return 0;
}
