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

#include "blocks8.h"
#include "common.cuh"

namespace tgo {

int num_sms();  // gemm.cu

namespace {

constexpr int BM = 128, BK = 128, THREADS = 192;
constexpr int ATOM = 512;

template <int BN>
struct Cfg {
  static constexpr int A_BYTES = BM * BK, B_BYTES = BN * BK;
  static constexpr int STAGE_BYTES = A_BYTES + B_BYTES;
  static constexpr int STAGES = BN == 256 ? 4 : 6;
  static constexpr int SF_BYTES = (1 + BN / 128) * ATOM;  // of a stage: A's atom, B's atoms
  static constexpr int C_STAGE = 4096;                    // epilogue staging of one warp
  static constexpr int SMEM = 1024 + STAGES * (STAGE_BYTES + SF_BYTES) + 4 * C_STAGE;
  // Tensor memory (512 columns): two accumulators and the scale factors. Two of 256 columns leave no room, so they share
  // 16 columns, which the epilogue reads first.
  static constexpr int ACC1 = BN == 256 ? 240 : BN;
  static constexpr int SFA = 496, SFB = 500;
};

// e4m3 A and B, fp32 D, scales of type e8m0; sf: byte of the scale words that this step uses
__device__ __forceinline__ constexpr uint32_t idesc_mx(int M, int N, uint32_t sf) {
  return (sf << 4) | ((uint32_t)(N >> 3) << 17) | (1u << 23) | ((uint32_t)(M >> 7) << 27) | (sf << 29);
}
__device__ __forceinline__ void umma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
      : "memory");
}
// one atom, 32 rows of 16 bytes: four columns, the same in every quarter of the lanes
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// shared-memory descriptor without swizzle: groups of 8 rows of 16 bytes, 128 bytes apart
__device__ __forceinline__ uint64_t sdesc_plain(uint32_t saddr) {
  return (uint64_t)((saddr & 0x3FFFFu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}

template <int OUT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (OUT == OUT_BF16) return pack_bf16x2(a, b);
  __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<uint32_t*>(&h);
}

// 32 values of a row to the staging tile, in the swizzled order of C's map (16-bit: rows of 64 bytes; fp32: of 128)
template <int OUT>
__device__ __forceinline__ void stage_row(uint8_t* buf, int lane, const float (&v)[32]) {
  if constexpr (OUT == OUT_F32) {
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
template <int OUT>
__device__ __forceinline__ void store_one(void* C, long long at, float v, bool add) {
  if constexpr (OUT == OUT_F32) {
    float* c = reinterpret_cast<float*>(C) + at;
    *c = add ? *c + v : v;
  } else if constexpr (OUT == OUT_BF16) {
    reinterpret_cast<__nv_bfloat16*>(C)[at] = __float2bfloat16_rn(v);
  } else {
    reinterpret_cast<__half*>(C)[at] = __float2half_rn(v);
  }
}

template <int BN, int OUT>
__global__ void __launch_bounds__(THREADS, 1)
    gemm8_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                 const __grid_constant__ CUtensorMap tmC, const Gemm8Params p) {
  using F = Cfg<BN>;
  constexpr int STAGES = F::STAGES;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* const smem_sf = smem + STAGES * F::STAGE_BYTES;
  uint8_t* const smem_c = smem_sf + STAGES * F::SF_BYTES;
  __shared__ __align__(8) uint64_t full_bar[STAGES], empty_bar[STAGES], tfull_bar[2], tempty_bar[2], done_bar;
  __shared__ uint32_t tmem_base_sh;
  __shared__ volatile int abort_sh;

  const int warp = warp_id(), lane = lane_id();
  const int num_m = (p.M + BM - 1) / BM, num_n = (p.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int chunks = (p.kb + p.chunk_kb - 1) / p.chunk_kb;
  const int kq = (p.kb + 3) / 4;       // scale atoms of a row tile
  const int nbt = (p.N + 127) / 128;   // row tiles of B's scales

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 4);
    }
    mbar_init(&done_bar, 1);
    abort_sh = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
  }
  if (warp == 1) {
    tmem_alloc(&tmem_base_sh, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_sh;

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- loads ----------------
      int stage = 0, filled = 0;
      uint32_t phase = 0;
      for (int tile = blockIdx.x; tile < num_tiles && !abort_sh; tile += gridDim.x) {
        const int mt = tile / num_n, nt = tile % num_n;
        for (int kb = 0; kb < p.kb; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1, p.err, ERR_MBAR_TIMEOUT_PRODUCER)) {
            abort_sh = 1;
            break;
          }
          uint8_t* sa = smem + stage * F::STAGE_BYTES;
          uint8_t* sf = smem_sf + stage * F::SF_BYTES;
          const bool scales = (kb & 3) == 0;
          const int nb = min(BN / 128, nbt - nt * (BN / 128));
          mbar_expect_tx(&full_bar[stage], F::STAGE_BYTES + (scales ? (1 + nb) * ATOM : 0));
          tma_load_3d(sa, &tmA, &full_bar[stage], kb * BK, mt * BM, 0);
          tma_load_3d(sa + F::A_BYTES, &tmB, &full_bar[stage], kb * BK, nt * BN, 0);
          if (scales) {
            bulk_load(sf, p.sfa + ((long long)mt * kq + (kb >> 2)) * ATOM, ATOM, &full_bar[stage]);
            for (int i = 0; i < nb; ++i)
              bulk_load(sf + (1 + i) * ATOM, p.sfb + ((long long)(nt * (BN / 128) + i) * kq + (kb >> 2)) * ATOM, ATOM,
                        &full_bar[stage]);
          }
          filled = min(filled + 1, STAGES);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      // the last loads have landed before the block ends, also after a wait that ran out
      for (int i = 0; i < filled; ++i) {
        stage = stage == 0 ? STAGES - 1 : stage - 1;
        if (stage == STAGES - 1) phase ^= 1;
        if (!mbar_wait(&full_bar[stage], phase, p.err, ERR_MBAR_TIMEOUT_PRODUCER)) break;
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      // ---------------- products ----------------
      const uint64_t a0 = sdesc_sw128(smem_u32(smem), 16, 1024), b0 = sdesc_sw128(smem_u32(smem) + F::A_BYTES, 16, 1024);
      const uint64_t s0 = sdesc_plain(smem_u32(smem_sf));
      const uint32_t sfa = tmem_base + F::SFA, sfb = tmem_base + F::SFB;
      int stage = 0, unit = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
        for (int c = 0; c < chunks && ok; ++c, ++unit) {
          // accumulators that share columns: the unit before has given up its shared ones; else: the one before that
          // has been read
          constexpr int back = BN == 256 ? 1 : 2;
          if (unit >= back) {
            const int u = unit - back;
            ok = !abort_sh && mbar_wait(&tempty_bar[u & 1], (u >> 1) & 1, p.err, ERR_MBAR_TIMEOUT_MMA);
            if (!ok) break;
          }
          tc_fence_after();
          const uint32_t d = tmem_base + ((unit & 1) ? F::ACC1 : 0);
          const int k0 = c * p.chunk_kb, k1 = min(p.kb, k0 + p.chunk_kb);
          for (int kb = k0; kb < k1; ++kb) {
            ok = !abort_sh && mbar_wait(&full_bar[stage], phase, p.err, ERR_MBAR_TIMEOUT_MMA);
            if (!ok) break;
            tc_fence_after();
            if ((kb & 3) == 0) {
              const uint64_t s = sdesc_add(s0, stage * F::SF_BYTES);
#pragma unroll
              for (int i = 0; i <= BN / 128; ++i) copy_scales(i == 0 ? sfa : sfb + (i - 1) * 4, sdesc_add(s, i * ATOM));
            }
            const uint64_t a = sdesc_add(a0, stage * F::STAGE_BYTES), b = sdesc_add(b0, stage * F::STAGE_BYTES);
            const uint32_t id = idesc_mx(BM, BN, kb & 3);
#pragma unroll
            for (int k = 0; k < 4; ++k) umma_mx(d, a + 2 * k, b + 2 * k, id, sfa, sfb, (kb != k0 || k != 0) ? 1u : 0u);
            umma_commit(&empty_bar[stage]);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1;
            }
          }
          if (ok) umma_commit(&tfull_bar[unit & 1]);
        }
      }
      if (!ok) {  // what was issued is over before tensor memory is given back
        abort_sh = 1;
        umma_commit(&done_bar);
        mbar_wait(&done_bar, 0, p.err, ERR_MBAR_TIMEOUT_MMA);
      }
    }
  } else {
    // ---------------- epilogue: warp q owns rows 32 q .. 32 q + 31 of the tile ----------------
    const int q = warp & 3;
    uint8_t* const cbuf = smem_c + q * F::C_STAGE;
    constexpr int BUFS = OUT == OUT_F32 ? 1 : 2;
    int turn = 0, unit = 0;
    bool ok = true;
    for (int tile = blockIdx.x; tile < num_tiles && ok; tile += gridDim.x) {
      const int m0 = (tile / num_n) * BM + q * 32, n0 = (tile % num_n) * BN;
      for (int c = 0; c < chunks; ++c, ++unit) {
        int got = 0;
        if (lane == 0) got = mbar_wait(&tfull_bar[unit & 1], (unit >> 1) & 1, p.err, ERR_MBAR_TIMEOUT_EPILOGUE) ? 1 : 0;
        ok = __shfl_sync(0xffffffffu, got, 0) != 0;
        if (!ok) {
          abort_sh = 1;
          break;
        }
        tc_fence_after();
        const bool add = OUT == OUT_F32 && (c > 0 || p.add);
        // chunks of one sum join in order: what the lane has sent has been written
        if (c > 0 && p.c_tma && lane == 0) bulk_wait_group_all();
        const uint32_t t = tmem_base + ((unit & 1) ? F::ACC1 : 0) + ((uint32_t)(q * 32) << 16);
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
            if (lane == 0) mbar_arrive(&tempty_bar[unit & 1]);
          }
          if (m0 >= p.M || n0 + col >= p.N) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          if (p.bias != nullptr && c == 0) {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] += n0 + col + j < p.N ? __ldg(p.bias + n0 + col + j) : 0.f;
          }
          if (p.c_tma) {
            uint8_t* buf = cbuf + (turn % BUFS) * (F::C_STAGE / BUFS);
            ++turn;
            if (lane == 0) bulk_wait_group_read<BUFS - 1>();
            __syncwarp();
            stage_row<OUT>(buf, lane, v);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              if (add) tma_reduce_add_3d(&tmC, buf, n0 + col, m0, 0);
              else tma_store_3d(&tmC, buf, n0 + col, m0, 0);
              bulk_commit_group();
            }
          } else {  // rows that a tensor map cannot address: through the staging tile, a row of 32 values at a time
            float* s = reinterpret_cast<float*>(cbuf);
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 32; ++j) s[lane * 32 + (j ^ lane)] = v[j];
            __syncwarp();
            if (n0 + col + lane < p.N) {
              const int rows = min(32, p.M - m0);
#pragma unroll 4
              for (int j = 0; j < rows; ++j)
                store_one<OUT>(p.C, (long long)(m0 + j) * p.ldc + n0 + col + lane, s[j * 32 + (lane ^ j)], add);
            }
          }
        }
      }
    }
    if (p.c_tma && lane == 0) bulk_wait_group_all();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int BN, int OUT>
cudaError_t launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Gemm8Params& p,
                   cudaStream_t s) {
  auto kern = gemm8_kernel<BN, OUT>;
  static_assert(Cfg<BN>::SMEM + 1024 <= 232448, "dynamic + static shared memory");
  const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<BN>::SMEM);
  if (e != cudaSuccess) return e;
  const long long tiles = (long long)((p.M + BM - 1) / BM) * ((p.N + BN - 1) / BN);
  if (tiles >= (1ll << 31)) return cudaErrorInvalidValue;
  kern<<<(int)std::min<long long>(tiles, num_sms()), THREADS, Cfg<BN>::SMEM, s>>>(ta, tb, tc, p);
  return cudaGetLastError();
}

}  // namespace

cudaError_t gemm8_launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Gemm8Params& p, int bn,
                         int out, cudaStream_t s) {
  if (p.M <= 0 || p.N <= 0 || p.kb <= 0 || p.chunk_kb <= 0 || p.chunk_kb % 4 != 0) return cudaErrorInvalidValue;
  if (out != OUT_F32 && (p.add || p.chunk_kb < p.kb)) return cudaErrorInvalidValue;
  if (p.add && p.bias != nullptr) return cudaErrorInvalidValue;
  if (bn == 256) {
    if (out == OUT_BF16) return launch<256, OUT_BF16>(ta, tb, tc, p, s);
    if (out == OUT_F16) return launch<256, OUT_F16>(ta, tb, tc, p, s);
    return launch<256, OUT_F32>(ta, tb, tc, p, s);
  }
  if (bn != 128) return cudaErrorInvalidValue;
  if (out == OUT_BF16) return launch<128, OUT_BF16>(ta, tb, tc, p, s);
  if (out == OUT_F16) return launch<128, OUT_F16>(ta, tb, tc, p, s);
  return launch<128, OUT_F32>(ta, tb, tc, p, s);
}

}  // namespace tgo
