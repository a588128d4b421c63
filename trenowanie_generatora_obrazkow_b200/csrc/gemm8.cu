// Products of 8-bit block operands (blocks8.h) on the tensor cores of sm_100a:
//
//   C[m, n] (+)= sum_k A[m, k] B[n, k] 2^(ea[m, k / 128] + eb[n, k / 128])  (+ bias[n])        C bf16, fp16 or fp32
//
// Both operands are K-major, so one kernel serves the forward (x, W), the input's gradient (dy, W^T) and the weight's
// gradient (dy^T, x^T): packing writes the transposed forms in the pass that reads the tensor.
//
// The scales are powers of two, so the tensor core applies them itself (kind::mxf8f6f4 with block scales: one byte for
// each row and 32 of k, here the same byte for the four steps of a block): no accumulator passes through registers before
// the whole sum is there. A scale atom (128 rows x 4 blocks, 512 bytes) goes from shared to tensor memory with one copy
// every fourth block.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "block_ops.h"
#include "blocks8.cuh"
#include "blocks8.h"
#include "common.cuh"
#include "vec.cuh"

namespace tgo {

int num_sms();  // gemm.cu

namespace {

constexpr int BM = 128, BK = 128;

// Two CTAs of a cluster share a tile of 256 x BN (PAIR, cta_group::2): each loads 128 rows of A and half of B's, so a block
// of k moves 32 KB (BN 256) or 28 KB (BN 192) into an SM in the 512 or 384 cycles that its products take. An SM takes in some
// 64 bytes a cycle while all do: one CTA with 128 x 256 (48 KB) ran at 2.4 PFLOP/s where the pairs reach 2.9 to 3.1.
// S: void, or the 16-bit type of a SwiGLU epilogue's [a | b], whose results leave in 8 bits alone (see there)
template <int BN, bool PAIR, typename S>
struct Cfg {
  static constexpr bool SWIGLU = !std::is_void<S>::value;
  static constexpr int EPI_WARPS = SWIGLU ? 16 : 4, THREADS = 64 + 32 * EPI_WARPS;
  static constexpr int A_BYTES = BM * BK, B_ROWS = PAIR ? BN / 2 : BN, B_BYTES = B_ROWS * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = STAGE_BYTES == 32768 ? 6 : 7;
  static constexpr int B_ATOMS = (BN + 127) / 128;         // a tile of 192 begins at the start or the middle of an atom
  static constexpr int SF_BYTES = (1 + B_ATOMS) * ATOM;    // of a stage: A's atom, B's atoms
  static constexpr int C_STAGE = SWIGLU ? 1024 : 4096;    // epilogue staging of one warp
  static constexpr int MAXIMA = SWIGLU ? (4 * 3 + 4 + 1) * BM * 4 : 0;
  static constexpr int SMEM = 1024 + STAGES * STAGE_BYTES + ((STAGES * SF_BYTES + 1023) & ~1023) + EPI_WARPS * C_STAGE + MAXIMA;
  // Tensor memory (512 columns): two accumulators and the scale factors. Two of 256 columns leave no room, so they share
  // 16 columns, which the epilogue reads first: the next sum waits for that, some 2600 cycles a tile.
  static constexpr int ACC1 = BN == 256 ? 240 : BN;
  static constexpr int SFA = 496, SFB = 500;
};

// e4m3 A and B, fp32 D, scales of type e8m0; sf: byte of the scale words that this step uses
__device__ __forceinline__ constexpr uint32_t idesc_mx(int M, int N, uint32_t sf) {
  return (sf << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | (sf << 29);
}
template <bool PAIR>
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
#define UMMA_MX(CTAS)                                                                                                     \
  asm volatile(                                                                                                           \
      "{\n\t.reg .pred p;\n\t"                                                                                           \
      "setp.ne.b32 p, %6, 0;\n\t"                                                                                         \
      "tcgen05.mma.cta_group::" CTAS ".kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d), \
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                                    \
      : "memory")
  if constexpr (PAIR) UMMA_MX("2");
  else UMMA_MX("1");
#undef UMMA_MX
}
// one atom, 32 rows of 16 bytes: four columns, the same in every quarter of the lanes
template <bool PAIR>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {  // a pair: in both CTAs, each from its own
  if constexpr (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// arrives once on the barrier (a pair: on both CTAs') when what this thread has issued is done
template <bool PAIR>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (PAIR) umma_commit_pair_mc(bar, 0x3);
  else umma_commit(bar);
}
// shared-memory descriptor without swizzle: groups of 8 rows of 16 bytes, 128 bytes apart
__device__ __forceinline__ uint64_t sdesc_plain(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <int OUT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (OUT == ELEM_BF16) return pack_bf16x2(a, b);
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// 32 values of a row to the staging tile, in the swizzled order of C's map (16-bit: rows of 64 bytes; fp32: of 128)
template <int OUT>
__device__ __forceinline__ void stage_row(uint8_t* buf, int lane, const float (&v)[32]) {
  if constexpr (OUT == ELEM_F32) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      *reinterpret_cast<float4*>(buf + lane * 128 + ((j ^ (lane & 7)) << 4)) =
          make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<uint4*>(buf + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)) =
          make_uint4(pack2<OUT>(v[8 * j], v[8 * j + 1]), pack2<OUT>(v[8 * j + 2], v[8 * j + 3]),
                     pack2<OUT>(v[8 * j + 4], v[8 * j + 5]), pack2<OUT>(v[8 * j + 6], v[8 * j + 7]));
  }
}
// a lane's column of a staged 32 x 32 tile to C; eight rows at a time, so that the reads do not wait for the stores
template <typename T>
__device__ __forceinline__ void store_rows(const Gemm8Problem& q, long long at, const float* s, int rows, bool add, int lane) {
  T* c = reinterpret_cast<T*>(q.C) + at;
#pragma unroll
  for (int j = 0; j < 32; j += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = s[(j + k) * 32 + (lane ^ (j + k))];
    if constexpr (sizeof(T) == 4) {
      if (add) {
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (j + k < rows) v[k] += c[(j + k) * q.ldc];
      }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (j + k < rows) c[(j + k) * q.ldc] = from_f<T>(v[k]);
  }
}

struct Gemm8Swiglu {
  CUtensorMap g8t_map;
  Side ck, g8, g8t;
};

struct NoSwiglu {};
template <typename S>
using SwigluOf = std::conditional_t<std::is_void<S>::value, NoSwiglu, Gemm8Swiglu>;

// The tiles of a unit (a CTA, a pair), one after another. The tiles of the first product (the longer ones) are dealt out in
// turn; where that leaves `late` units with one more than the others, these others take `spare` rounds of the second product's
// tiles before all take part: two products end together that apart would each leave units idle in their last wave.
struct Schedule {
  int unit, units, mine, late, spare;
  __device__ Schedule(const Gemm8Params& p, int unit_, int units_)
      : unit(unit_), units(units_), late(p.late), spare(p.spare) {
    mine = p.q[0].tiles > unit ? (p.q[0].tiles - unit + units - 1) / units : 0;
  }
  __device__ __forceinline__ bool at(const Gemm8Params& p, int step, int& product, int& tile) const {
    product = 0;
    tile = step * units + unit;
    if (step < mine) return true;
    if (p.n < 2) return false;
    const int t = step - mine, early = units - late;
    product = 1;
    if (unit >= late && t < spare) tile = t * early + unit - late;
    else tile = spare * early + (unit >= late ? t - spare : t) * units + unit;
    return tile < p.q[1].tiles;
  }
};

// ------------------------------------------------------------------------------------------------- SwiGLU epilogue
// One CTA's half of a tile of 256 rows x (128 columns a | the same 128 columns b): a and b, rounded to S, stay in registers, g
// = silu(a) b in fp32; they leave as 8-bit blocks alone: the checkpoint of a and b, g along its rows, g along its columns. A
// tile is a block of both axes, so no other CTA is asked for a maximum. Sixteen warps: quarter (32 rows, a thread each) x
// strip (32 columns), what two blocks' values and a third in fp32 leave room for in registers. The strips of a row meet in
// shared memory, as do the quarters of a column, whose maximum over a warp's rows is one integer reduction. Codes of rows
// leave from the registers, 32 bytes a store; those of columns through 1 KB of staging a warp, by TMA. (Through staging and
// TMA all of them cost one of the loads' six stages: 713 us instead of 673; 680 with sigmoids in two factors.) At 32768 x 2048
// -> 2 x 5504 a tile takes 13.7 k cycles, the tensor core is busy for 55 to 60 % of them: 3.1 k go by until the shared columns
// are read, 1.3 k in waits for loads, the rest is put down to the epilogue's traffic in shared memory beside the operands' (11.8
// k without checkpoint and g's columns).
// Product and activation apart took 555 + 331 us, and a and b crossed memory twice (1.4 GB).
struct SwigluShared {
  float rows[4][3][BM];  // [strip][a, b, g][row]
  float cols[4][BM];     // [quarter][column]: of g
  float inv[BM];         // 2^-e of g's columns
};
__device__ __forceinline__ bool all_of_512(bool ok) {  // barrier of the epilogue's warps, with their verdict
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.and.pred q, 1, 512, p;\n\tselp.u32 %0, 1, 0, q;\n}"
               : "=r"(r) : "r"((uint32_t)ok) : "memory");
  return r != 0;
}
template <typename S>
struct PairOf;
template <>
struct PairOf<__nv_bfloat16> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) { return pack_bf16x2(a, b); }
  static __device__ __forceinline__ float2 get(uint32_t u) {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
};
template <>
struct PairOf<__half> {
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  static __device__ __forceinline__ float2 get(uint32_t u) { return __half22float2(*reinterpret_cast<const __half2*>(&u)); }
};
__device__ __forceinline__ void store32(uint8_t* p, const uint32_t (&w)[8]) {  // 32-byte aligned
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}
__device__ __forceinline__ float finite_or_nan(float v) { return fabsf(v) == INFINITY ? NAN : v; }
// 16 pairs of a row: the largest finite magnitude; infinities become NaN
template <typename S>
__device__ __forceinline__ float finite_top16(uint32_t (&u)[16]) {
  auto top = [&] {
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 v = PairOf<S>::get(u[j]);
      m = max3(m, fabsf(v.x), fabsf(v.y));
    }
    return m;
  };
  float m = top();
  if (m == INFINITY) {
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float2 v = PairOf<S>::get(u[j]);
      u[j] = PairOf<S>::pack(finite_or_nan(v.x), finite_or_nan(v.y));
    }
    m = top();
  }
  return m;
}

template <int BN, bool PAIR, typename S>
__global__ void __launch_bounds__((Cfg<BN, PAIR, S>::THREADS), 1)
    gemm8_kernel(const __grid_constant__ Gemm8Maps maps, const __grid_constant__ Gemm8Params p,
                 const __grid_constant__ SwigluOf<S> sw) {
  using F = Cfg<BN, PAIR, S>;
  constexpr bool SWIGLU = F::SWIGLU;
  constexpr int STAGES = F::STAGES, TM = PAIR ? 2 * BM : BM, EPI_WARPS = (PAIR ? 2 : 1) * F::EPI_WARPS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const smem_sf = smem + STAGES * F::STAGE_BYTES;
  uint8_t* const smem_c = smem + STAGES * F::STAGE_BYTES + ((STAGES * F::SF_BYTES + 1023) & ~1023);
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tfull_bar[2], tempty_bar[2], done_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;

  const int warp = warp_id(), lane = lane_id();
  const int rank = PAIR ? (int)cluster_ctarank() : 0;
  const bool leader = rank == 0;  // issues the pair's products; its barriers count both CTAs' loads and epilogues
  const Schedule sched(p, PAIR ? blockIdx.x >> 1 : blockIdx.x, PAIR ? gridDim.x >> 1 : gridDim.x);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], EPI_WARPS);
    }
    mbar_init(&done_bar, 1);
    abort_sh = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane < p.n) {
    prefetch_tmap(&maps.a[lane]);
    prefetch_tmap(&maps.b[lane]);
    if constexpr (PAIR) prefetch_tmap(&maps.sa[lane]), prefetch_tmap(&maps.sb[lane]);
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      tmem_alloc_pair(&tmem_base_sh, 512);
      tmem_relinquish_pair();
    } else {
      tmem_alloc(&tmem_base_sh, 512);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  if constexpr (PAIR) cluster_sync();  // the peer's barriers are there before anything arrives on them
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;
  // The two warps that feed the tensor core run as whole warps and elect a lane where an instruction wants one thread: the
  // operands then stay in uniform registers. With one lane in the loop each product cost its thread some 70 cycles of moving
  // operands, and the thread, not the tensor core, was the bound (690 cycles for a block of 4 x 128).
  if (warp == 0) {
    // ---------------- loads ----------------
    int stage = 0, filled = 0;
    uint32_t phase = 0;
    bool free = true, ok = true;  // free: the stage is known to be free
    int which, tile;
    for (int step = 0; ok && sched.at(p, step, which, tile); ++step) {
      const Gemm8Problem& q = p.q[which];
      const CUtensorMap *tmA = &maps.a[which], *tmB = &maps.b[which], *tmSA = &maps.sa[which], *tmSB = &maps.sb[which];
      const int num_n = (q.N + BN - 1) / BN;  // SwiGLU: N is a multiple of 256
      const int kq = (q.kb + 3) / 4;      // scale atoms of a row tile
      const int nbt = (q.N + 127) / 128;  // row tiles of B's scales
      const int mt = tile / num_n, nt = tile % num_n;
      // SwiGLU: one CTA brings the rows of a, the other those of b
      const int m0 = mt * TM + rank * BM, n0 = SWIGLU ? nt * 128 + rank * (q.N / 2) : nt * BN + rank * F::B_ROWS;
      for (int kb = 0; kb < q.kb; ++kb) {
        if (!free) {
          ok = __all_sync(0xffffffffu, mbar_wait_poll(&empty_bar[stage], phase ^ 1, p.err, ERR_MBAR_TIMEOUT_PRODUCER) &&
                                           !abort_sh);
          if (!ok) break;
        }
        const int next = stage + 1 == STAGES ? 0 : stage + 1;
        const uint32_t next_phase = next == 0 ? phase ^ 1 : phase;
        free = __all_sync(0xffffffffu, mbar_test_wait(&empty_bar[next], next_phase ^ 1));
        if (elect_one()) {
          uint8_t* sa = smem + stage * F::STAGE_BYTES;
          uint8_t* sf = smem_sf + stage * F::SF_BYTES;
          const bool scales = (kb & 3) == 0;
          if constexpr (PAIR) {
            if (leader) mbar_expect_tx(&full_bar[stage], 2 * (F::STAGE_BYTES + (scales ? F::SF_BYTES : 0)));
            const uint32_t bar = mapa_shared(smem_u32(&full_bar[stage]), 0);
            tma_load_3d_pair(sa, tmA, bar, kb * BK, m0, 0);
            tma_load_3d_pair(sa + F::A_BYTES, tmB, bar, kb * BK, n0, 0);
            if (scales) {
              tma_load_3d_pair(sf, tmSA, bar, 0, kb >> 2, mt * 2 + rank);
              if constexpr (SWIGLU) {
                tma_load_3d_pair(sf + ATOM, tmSB, bar, 0, kb >> 2, nt);
                tma_load_3d_pair(sf + 2 * ATOM, tmSB, bar, 0, kb >> 2, q.N / 256 + nt);
              } else {
                tma_load_3d_pair(sf + ATOM, tmSB, bar, 0, kb >> 2, nt * BN / 128);
              }
            }
          } else {
            const int nb = min(F::B_ATOMS, nbt - nt * (BN / 128));
            mbar_expect_tx(&full_bar[stage], F::STAGE_BYTES + (scales ? (1 + nb) * ATOM : 0));
            tma_load_3d(sa, tmA, &full_bar[stage], kb * BK, m0, 0);
            tma_load_3d(sa + F::A_BYTES, tmB, &full_bar[stage], kb * BK, n0, 0);
            if (scales) {
              bulk_load(sf, q.sfa + ((long long)mt * kq + (kb >> 2)) * ATOM, ATOM, &full_bar[stage]);
              for (int i = 0; i < nb; ++i)
                bulk_load(sf + (1 + i) * ATOM, q.sfb + ((long long)(nt * (BN / 128) + i) * kq + (kb >> 2)) * ATOM, ATOM,
                          &full_bar[stage]);
            }
          }
        }
        __syncwarp();
        filled = min(filled + 1, STAGES);
        stage = next;
        phase = next_phase;
      }
    }
    if (!ok) abort_sh = 1;
    // the last loads have landed before the block (the pair) ends, also after a wait that ran out
    for (int i = 0; i < filled && leader; ++i) {
      stage = stage == 0 ? STAGES - 1 : stage - 1;
      if (stage == STAGES - 1) phase ^= 1;
      if (!__all_sync(0xffffffffu, mbar_wait(&full_bar[stage], phase, p.err, ERR_MBAR_TIMEOUT_PRODUCER))) break;
    }
  } else if (warp == 1) {
    if (leader) {
      // ---------------- products ----------------
      const uint64_t a0 = sdesc_sw128(smem_u32(smem), 16, 1024), b0 = sdesc_sw128(smem_u32(smem) + F::A_BYTES, 16, 1024);
      const uint64_t s0 = sdesc_plain(smem_u32(smem_sf));
      const uint32_t sfa = tmem_base + F::SFA, sfb = tmem_base + F::SFB;
      // a look at the next block's barrier comes before this block's products
      int stage = 0, unit = 0;
      uint32_t phase = 0;
      bool ok = true, ready = false;
      int which, tile;
      for (int step = 0; ok && sched.at(p, step, which, tile); ++step) {
        const int kbs = p.q[which].kb, chunk_kb = p.q[which].chunk_kb;
        const uint32_t sfb_n = sfb + (BN % 128 != 0 && (tile % ((p.q[which].N + BN - 1) / BN) & 1) ? 2 : 0);  // 64 columns in
        for (int c = 0; c * chunk_kb < kbs && ok; ++c, ++unit) {
          // accumulators that share columns: the unit before has given up its shared ones; else: the one before that
          // has been read
          constexpr int back = BN == 256 ? 1 : 2;
          if (unit >= back) {
            const int u = unit - back;
            ok = __all_sync(0xffffffffu, mbar_wait_poll(&tempty_bar[u & 1], (u >> 1) & 1, p.err, ERR_MBAR_TIMEOUT_MMA) &&
                                             !abort_sh);
            if (!ok) break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + ((unit & 1) ? F::ACC1 : 0);
          const int k0 = c * chunk_kb, k1 = min(kbs, k0 + chunk_kb);
          for (int kb = k0; kb < k1; ++kb) {
            if (!ready) {
              ok = __all_sync(0xffffffffu, mbar_wait_poll(&full_bar[stage], phase, p.err, ERR_MBAR_TIMEOUT_MMA) && !abort_sh);
              if (!ok) break;
            }
            const int next = stage + 1 == STAGES ? 0 : stage + 1;
            const uint32_t next_phase = next == 0 ? phase ^ 1 : phase;
            ready = __all_sync(0xffffffffu, mbar_test_wait(&full_bar[next], next_phase));
            tc_fence_after();
            if (elect_one()) {
              if ((kb & 3) == 0) {
                const uint64_t s = sdesc_add(s0, stage * F::SF_BYTES);
#pragma unroll
                for (int i = 0; i <= F::B_ATOMS; ++i)
                  copy_scales<PAIR>(i == 0 ? sfa : sfb + (i - 1) * 4, sdesc_add(s, i * ATOM));
              }
              const uint64_t a = sdesc_add(a0, stage * F::STAGE_BYTES), b = sdesc_add(b0, stage * F::STAGE_BYTES);
              const uint32_t id = idesc_mx(TM, BN, kb & 3);
#pragma unroll
              for (int k = 0; k < 4; ++k)
                umma_mx<PAIR>(d, a + 2 * k, b + 2 * k, id, sfa, sfb_n, (kb != k0 || k != 0) ? 1u : 0u);
              commit<PAIR>(&empty_bar[stage]);
              if (kb == k1 - 1) commit<PAIR>(&tfull_bar[unit & 1]);
            }
            __syncwarp();
            stage = next;
            phase = next_phase;
          }
        }
      }
      if (!ok) {  // what was issued is over before tensor memory is given back
        abort_sh = 1;
        if (elect_one()) {
          commit<PAIR>(&done_bar);
          mbar_wait(&done_bar, 0, p.err, ERR_MBAR_TIMEOUT_MMA);
        }
        __syncwarp();
      }
    }
  } else if constexpr (SWIGLU) {
    // ---------------- SwiGLU epilogue ----------------
    const int quarter = warp & 3, strip = (warp - 2) >> 2, r = quarter * 32 + lane;
    uint8_t* const buf = smem_c + (warp - 2) * F::C_STAGE;  // 32 columns of 32 bytes
    SwigluShared& sh = *reinterpret_cast<SwigluShared*>(smem_c + F::EPI_WARPS * F::C_STAGE);
    const Gemm8Problem& q = p.q[0];
    const int nhb = q.N / 256, nmb = (q.M + 127) / 128;
    int unit = 0, which, tile;
    for (int step = 0; sched.at(p, step, which, tile); ++step, ++unit) {
      const int hb = tile % nhb, mb = (tile / nhb) * 2 + rank;
      int got = 0;
      if (lane == 0) got = mbar_wait_poll(&tfull_bar[unit & 1], (unit >> 1) & 1, p.err, ERR_MBAR_TIMEOUT_EPILOGUE) ? 1 : 0;
      const bool ok = __shfl_sync(0xffffffffu, got, 0) != 0;
      tc_fence_after();
      const uint32_t t = tmem_base + ((unit & 1) ? F::ACC1 : 0) + ((uint32_t)(quarter * 32) << 16) + 32 * strip;
      uint32_t pa[16], pb[16];
      // the accumulators' shared columns first: the last 16 of the even one's b, the first 16 of the odd one's a
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint32_t ra[16], rb[16];
        tmem_ld_32x32b_x16(t + 16 * c, ra);
        tmem_ld_32x32b_x16(t + 128 + 16 * (c ^ 1), rb);
        tmem_ld_wait();
        if (c == 0) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty_bar[unit & 1]), 0));
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          pa[8 * c + j] = PairOf<S>::pack(__uint_as_float(ra[2 * j]), __uint_as_float(ra[2 * j + 1]));
          pb[8 * (c ^ 1) + j] = PairOf<S>::pack(__uint_as_float(rb[2 * j]), __uint_as_float(rb[2 * j + 1]));
        }
      }
      if (sw.ck.codes != nullptr) {
        sh.rows[strip][0][r] = finite_top16<S>(pa);
        sh.rows[strip][1][r] = finite_top16<S>(pb);
      }
      if (!all_of_512(ok)) {  // every warp's wait ends by itself, so all are here
        abort_sh = 1;
        break;
      }
      // strip k writes the scales of a, b, g and of g's columns
      auto row_scale = [&](int k, const Side& o, int b, int blocks) {
        const int byte = scale_byte(fmaxf(fmaxf(sh.rows[0][k][r], sh.rows[1][k][r]), fmaxf(sh.rows[2][k][r], sh.rows[3][k][r])));
        if (strip == k && mb < nmb) {
          uint8_t* s = o.scales + scale_at(mb * BM + r, b, o.quads);
          s[0] = (uint8_t)byte;
          if (b == blocks - 1)
            for (int i = 1; i < 4 - (b & 3); ++i) s[i] = 0;
        }
        return scale_inv(byte);
      };
      const int m0 = mb * BM + quarter * 32, h0 = hb * 128 + 32 * strip;
      const bool row_there = mb * BM + r < q.M;
      // a row's 32 codes of this strip: one sector, straight from the registers
      auto put = [&](const Side& o, int col, const uint32_t(&w)[8]) {
        if (row_there) store32(o.codes + (long long)(mb * BM + r) * o.width + col, w);
      };
      auto put_pairs = [&](int col, const uint32_t(&u)[16], float inv) {
        const float2 s = make_float2(inv, inv);
        uint32_t w[8];
#pragma unroll
        for (int n = 0; n < 8; ++n) w[n] = codes4(mul2(PairOf<S>::get(u[2 * n]), s), mul2(PairOf<S>::get(u[2 * n + 1]), s));
        put(sw.ck, col, w);
      };
      if (sw.ck.codes != nullptr) {
        const float inv_a = row_scale(0, sw.ck, hb, 2 * nhb), inv_b = row_scale(1, sw.ck, nhb + hb, 2 * nhb);
        put_pairs(h0, pa, inv_a);
        put_pairs(q.N / 2 + h0, pb, inv_b);
      }
      float g[32];
      float mg = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float2 v = swiglu<false>(PairOf<S>::get(pa[j]), PairOf<S>::get(pb[j]));
        g[2 * j] = v.x;
        g[2 * j + 1] = v.y;
        mg = max3(mg, fabsf(v.x), fabsf(v.y));
      }
      if (mg == INFINITY) {
        mg = 0.f;
#pragma unroll
        for (int j = 0; j < 32; ++j) mg = fmaxf(mg, fabsf(g[j] = finite_or_nan(g[j])));
      }
      sh.rows[strip][2][r] = mg;
      if (sw.g8t.codes != nullptr) {
        uint32_t mine = 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(fmaxf(fabsf(g[j]), 0.f)));  // passes over NaN
          if (lane == j) mine = top;
        }
        sh.cols[quarter][32 * strip + lane] = __uint_as_float(mine);
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");  // g's maxima are there, those of a and b read
      const float inv_g = row_scale(2, sw.g8, hb, nhb);
      if (sw.g8t.codes != nullptr && strip == 3) {
        const int byte = scale_byte(fmaxf(fmaxf(sh.cols[0][r], sh.cols[1][r]), fmaxf(sh.cols[2][r], sh.cols[3][r])));
        sh.inv[r] = scale_inv(byte);
        if (mb < nmb) {
          uint8_t* s = sw.g8t.scales + scale_at(hb * 128 + r, mb, sw.g8t.quads);
          s[0] = (uint8_t)byte;
          if (mb == nmb - 1)
            for (int i = 1; i < 4 - (mb & 3); ++i) s[i] = 0;
        }
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");  // the scales of g's columns are there
      if (sw.g8t.codes != nullptr && m0 < nmb * BM) {
        if (lane == 0) bulk_wait_group_read<0>();
        __syncwarp();
        uint8_t* to = buf + lane;
#pragma unroll
        for (int j = 0; j < 32; j += 2) {
          const float2 k = *reinterpret_cast<const float2*>(&sh.inv[32 * strip + j]);
          const uint32_t w = codes2(g[j] * k.x, g[j + 1] * k.y);
          to[j * 32] = (uint8_t)w;
          to[(j + 1) * 32] = (uint8_t)(w >> 8);
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_3d(&sw.g8t_map, buf, m0, h0, 0);
          bulk_commit_group();
        }
      }
      uint32_t w[8];
      const float2 s = make_float2(inv_g, inv_g);
#pragma unroll
      for (int n = 0; n < 8; ++n)
        w[n] = codes4(mul2(make_float2(g[4 * n], g[4 * n + 1]), s), mul2(make_float2(g[4 * n + 2], g[4 * n + 3]), s));
      put(sw.g8, h0, w);
    }
    if (lane == 0) bulk_wait_group_all();
  } else {
    // ---------------- epilogue: a warp owns 32 rows of the tile ----------------
    const int quarter = warp & 3;
    uint8_t* const cbuf = smem_c + quarter * F::C_STAGE;
    int turn = 0, unit = 0, which, tile;
    bool ok = true, any_tma = false;
    for (int step = 0; ok && sched.at(p, step, which, tile); ++step) {
      const Gemm8Problem& q = p.q[which];
      const CUtensorMap* tmC = &maps.c[which];
      const int num_n = (q.N + BN - 1) / BN;
      const int m0 = (tile / num_n) * TM + rank * BM + quarter * 32, n0 = (tile % num_n) * BN;
      const bool f32 = q.elem == ELEM_F32;
      for (int c = 0; c * q.chunk_kb < q.kb; ++c, ++unit) {
        int got = 0;
        if (lane == 0) got = mbar_wait_poll(&tfull_bar[unit & 1], (unit >> 1) & 1, p.err, ERR_MBAR_TIMEOUT_EPILOGUE) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        if (!ok) {
          abort_sh = 1;
          break;
        }
        tc_fence_after();
        const bool add = f32 && (c > 0 || q.add);
        if (lane == 0) {
          // chunks of one sum join in order: what the lane has sent has been written; else: the staging tile is free, whatever
          // the last product's type was
          if (c > 0 && q.c_tma) bulk_wait_group_all();
          else if (any_tma) bulk_wait_group_read<0>();
        }
        const uint32_t t = tmem_base + ((unit & 1) ? F::ACC1 : 0) + ((uint32_t)(quarter * 32) << 16);
#pragma unroll 1
        for (int i = 0; i < BN / 32; ++i) {
          // the columns that the accumulators share come first: the last of the even one, the first of the odd one
          const int col = 32 * (BN == 256 && !(unit & 1) ? BN / 32 - 1 - i : i);
          uint32_t r[32];
          tmem_ld_32x32b_x32(t + col, r);
          tmem_ld_wait();
          if (i == (BN == 256 ? 0 : BN / 32 - 1)) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) mbar_arrive_cluster(mapa_shared(smem_u32(&tempty_bar[unit & 1]), 0));
              else mbar_arrive(&tempty_bar[unit & 1]);
            }
          }
          if (m0 >= q.M || n0 + col >= q.N) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (q.bias != nullptr && c == 0) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += n0 + col + j < q.N ? __ldg(q.bias + n0 + col + j) : 0.f;
          }
          if (q.c_tma) {
            any_tma = true;
            uint8_t* buf = cbuf;
            if (f32) {
              if (lane == 0) bulk_wait_group_read<0>();
              __syncwarp();
              stage_row<ELEM_F32>(buf, lane, v);
            } else {  // two tiles in turn
              buf += (turn++ & 1) * (F::C_STAGE / 2);
              if (lane == 0) bulk_wait_group_read<1>();
              __syncwarp();
              if (q.elem == ELEM_BF16) stage_row<ELEM_BF16>(buf, lane, v);
              else stage_row<ELEM_F16>(buf, lane, v);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (add) tma_reduce_add_3d(tmC, buf, n0 + col, m0, 0);
              else tma_store_3d(tmC, buf, n0 + col, m0, 0);
              bulk_commit_group();
            }
          } else {  // rows that a tensor map cannot address: through the staging tile, a row of 32 values at a time
            float* s = reinterpret_cast<float*>(cbuf);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) s[lane * 32 + (j ^ lane)] = v[j];
            __syncwarp();
            if (n0 + col + lane < q.N) {
              const int rows = min(32, q.M - m0);
              const long long at = (long long)m0 * q.ldc + n0 + col + lane;
              if (f32) store_rows<float>(q, at, s, rows, add, lane);
              else if (q.elem == ELEM_BF16) store_rows<__nv_bfloat16>(q, at, s, rows, add, lane);
              else store_rows<__half>(q, at, s, rows, add, lane);
            }
          }
        }
      }
    }
    if (any_tma && lane == 0) bulk_wait_group_all();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync();  // neither CTA leaves while the pair still has products or arrivals in flight
  if (warp == 1) {
    tc_fence_after();
    if constexpr (PAIR) tmem_dealloc_pair(tmem_base, 512);
    else tmem_dealloc(tmem_base, 512);
  }
}

template <int BN, bool PAIR, typename S = void>
cudaError_t launch(const Gemm8Maps& t, Gemm8Params& p, const SwigluOf<S>& sw, Gemm8Tile tile, cudaStream_t s) {
  using F = Cfg<BN, PAIR, S>;
  auto kern = gemm8_kernel<BN, PAIR, S>;
  static_assert(F::SMEM + 256 <= 232448, "dynamic + static shared memory");
  static std::atomic<uint64_t> set{0};  // bit d: done on device d
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev > 63 || !((set.load(std::memory_order_relaxed) >> dev) & 1)) {
    e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F::SMEM);
    if (e != cudaSuccess) return e;
    if (dev <= 63) set.fetch_or(1ull << dev);
  }
  constexpr int TM = PAIR ? 2 * BM : BM;
  long long all = 0;
  for (int i = 0; i < p.n; ++i) {
    const long long tiles = (long long)((p.q[i].M + TM - 1) / TM) * ((p.q[i].N + BN - 1) / BN);
    if (tiles >= (1ll << 29)) return cudaErrorInvalidValue;
    p.q[i].tiles = (int)tiles;
    all += tiles;
  }
  const int units = (int)std::min<long long>(all, PAIR ? num_sms() / 2 : num_sms());
  p.late = p.spare = 0;
  if (p.n == 2 && p.q[0].tiles % units != 0) {
    p.late = p.q[0].tiles % units;
    const long long a = gemm8_tile_cycles(p.q[0], tile, true), b = gemm8_tile_cycles(p.q[1], tile, true);
    p.spare = (int)std::min<long long>((a + b / 2) / b, 1 << 20);
  }
  cudaLaunchConfig_t c{};
  c.gridDim = dim3(PAIR ? 2 * units : units);
  c.blockDim = dim3(F::THREADS);
  c.dynamicSmemBytes = F::SMEM;
  c.stream = s;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = 2;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  c.attrs = &cluster;
  c.numAttrs = PAIR ? 1 : 0;
  e = cudaLaunchKernelEx(&c, kern, t, p, sw);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace

// A block of 128 costs 480 (128 x 128, bound by its loads; 380 where they do not fill the GPU), 430 (256 x 192, loads) or 512
// (256 x 256, the products), a sum's beginning and end 300, 800 or 2600 (its accumulators share columns).
long long gemm8_tile_cycles(const Gemm8Problem& q, Gemm8Tile tile, bool fills) {
  const long long sums = (q.kb + q.chunk_kb - 1) / q.chunk_kb;
  if (tile == TILE_128x128) return (long long)q.kb * (fills ? 480 : 380) + sums * 300;
  return tile == TILE_PAIR_192 ? (long long)q.kb * 430 + sums * 800 : (long long)q.kb * 512 + sums * 2600;
}

static bool valid(const Gemm8Params& p) {
  if (p.n < 1 || p.n > 2) return false;
  for (int i = 0; i < p.n; ++i) {
    const Gemm8Problem& q = p.q[i];
    if (q.M <= 0 || q.N <= 0 || q.kb <= 0 || q.chunk_kb <= 0 || q.chunk_kb % 4 != 0) return false;
    if (q.elem != ELEM_F32 && (q.add || q.chunk_kb < q.kb)) return false;
    if (q.elem < ELEM_BF16 || q.elem > ELEM_F32 || (q.add && q.bias != nullptr)) return false;
  }
  return true;
}
cudaError_t gemm8_launch(const Gemm8Maps& t, Gemm8Params p, Gemm8Tile tile, cudaStream_t s) {
  if (!valid(p)) return cudaErrorInvalidValue;
  const NoSwiglu none{};
  switch (tile) {
    case TILE_PAIR_256: return launch<256, true>(t, p, none, tile, s);
    case TILE_PAIR_192: return launch<192, true>(t, p, none, tile, s);
    case TILE_128x128: return launch<128, false>(t, p, none, tile, s);
  }
  return cudaErrorInvalidValue;
}

cudaError_t gemm8_swiglu_launch(const Gemm8Maps& t, Gemm8Params p, Gemm8SwigluOut o, cudaStream_t s) {
  if (!valid(p) || p.n != 1 || p.q[0].N % 256 != 0 || p.q[0].bias != nullptr || o.g8 == nullptr ||
      (o.g8t != nullptr && o.g8t_map == nullptr)) return cudaErrorInvalidValue;
  const int H = p.q[0].N / 2, M = p.q[0].M;
  Gemm8Swiglu sw{};
  sw.ck = side(o.ck, o.ck_scales, M, 2 * H);
  sw.g8 = side(o.g8, o.g8_scales, M, H);
  sw.g8t = side(o.g8t, o.g8t_scales, H, M);
  if (o.g8t != nullptr) sw.g8t_map = *o.g8t_map;
  if (p.q[0].elem == ELEM_BF16) return launch<256, true, __nv_bfloat16>(t, p, sw, TILE_PAIR_256, s);
  if (p.q[0].elem == ELEM_F16) return launch<256, true, __half>(t, p, sw, TILE_PAIR_256, s);
  return cudaErrorInvalidValue;
}

}  // namespace tgo
