// Launch interfaces of the 8-bit block operators: packing into e4m3 with a power-of-two scale for each block of 128,
// products of such operands, SwiGLU with its input kept in 8 bits. Plain CUDA types only; the torch-facing checks are in
// blocks8_ops.cpp.
//
// The 8-bit form of X [R, K] (blocks along K): codes [R, Kp] e4m3, Kp = K rounded up to 128, zeros past K, and one byte
// e + 127 per block (its scale is 2^e) in atoms of 512 bytes [ceil(R / 128)][ceil(Kp / 512)][32][4][4]: row 128 i + 32 c + r,
// block 4 j + b stands at [i][j][r][c][b]. This is the order in which the tensor core takes scale factors (32 lanes of
// four columns of four bytes), so an atom goes to tensor memory with one copy. Bytes of rows past R and blocks past Kp
// are 0.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace tgo {

struct Pack8Params {
  const void* x;        // [M, K] of the element type, rows ld elements apart
  long long ld;
  int M, K, elem;       // elem: ElemType
  uint8_t* codes;       // [M, Kp] blocks along K, or null
  uint8_t* scales;
  uint8_t* codes_t;     // [K, Mp] blocks along M (of x^T), or null
  uint8_t* scales_t;
  float* sums;          // [ceil(M / 128)][K] sums over the rows of each tile, or null (with codes_t)
};
cudaError_t pack8_launch(const Pack8Params& p, cudaStream_t s);
// up to three tensors in one launch, each with codes and no sums
struct Pack8Jobs {
  Pack8Params job[3];
  int n;
};
cudaError_t pack8_jobs_launch(const Pack8Jobs& p, cudaStream_t s);
// out[k] (+)= sum of tiles' rows of sums [T][K], in order
cudaError_t colsum_launch(const float* sums, int T, int K, float* out, bool add, cudaStream_t s);
// codes [R, Kp] -> out [R, K] rows ldo apart
cudaError_t unpack8_launch(const uint8_t* codes, const uint8_t* scales, int R, int K, void* out, long long ldo, int elem,
                           cudaStream_t s);

struct Gemm8Problem {
  int M, N, kb;             // kb: blocks of 128 along the contraction
  const uint8_t* sfa;       // scale bytes of A and B
  const uint8_t* sfb;
  void* C;                  // [M, N], rows ldc elements apart
  long long ldc;
  const float* bias;        // [N] or null
  int elem;                 // of C
  int add;                  // C += (fp32 C only)
  int chunk_kb;             // contraction blocks per accumulator (a multiple of 4); further ones join in fp32 in order
  int c_tma;                // C goes through its tensor map
  int tiles;                // set by the launcher
};
enum Gemm8Tile : int { TILE_128x128 = 0, TILE_PAIR_192 = 1, TILE_PAIR_256 = 2 };  // pairs of CTAs: 256 x 192, 256 x 256
// One or two independent products in a launch. a, b: uint8 maps {Kp, rows, 1} with boxes {128, 128, 1} (b of TILE_PAIR_192:
// {128, 96, 1}), 128-byte swizzle; c: {N, M, 1}, box {32, 32, 1}; sa, sb (pairs alone): the scale atoms as 32-bit words
// {128, ceil(kb / 4), row tiles}, boxes {128, 1, 1} and {128, 1, 2}
struct Gemm8Maps {
  CUtensorMap a[2], b[2], c[2], sa[2], sb[2];
};
struct Gemm8Params {
  Gemm8Problem q[2];
  int n;
  int late;                 // set by the launcher, as `spare`: see gemm8.cu
  int spare;
  int* err;
};
// cycles of one output tile (its products, and its sums' beginnings and ends)
long long gemm8_tile_cycles(const Gemm8Problem& q, Gemm8Tile tile, bool fills);
cudaError_t gemm8_launch(const Gemm8Maps& t, Gemm8Params p, Gemm8Tile tile, cudaStream_t s);

// The first product of a SwiGLU MLP, [a | b] = A B^T (B [2 H, K], H a multiple of 128, 16-bit q.elem), and its activation: what
// the backward and the second product read, in 8 bits. Maps: as TILE_PAIR_256, sb's box {128, 1, 1}; g8t as bytes {Mp, H, 1}, box
// {32, 32, 1}, no swizzle.
struct Gemm8SwigluOut {
  uint8_t *ck, *ck_scales;    // [M, 2 H], or null
  uint8_t *g8, *g8_scales;    // [M, H]
  uint8_t *g8t, *g8t_scales;  // [H, Mp], or null
  const CUtensorMap* g8t_map;
};
cudaError_t gemm8_swiglu_launch(const Gemm8Maps& t, Gemm8Params p, Gemm8SwigluOut o, cudaStream_t s);

// y [M, N] = Q(x) W^T + bias for few rows, x packed on the way (one launch). Sixteen rows, W cold, against packing and product
// apart: 2048 -> 6144 9.6 us (3.1 + 11.2), 5504 -> 2048 11.0 (3.0 + 18.7), 1280 -> 3456 6.4 (2.8 + 8.9), 640 -> 1920 4.3 (3.0 + 7.1),
// 5504 -> 11008 32.9 (3.1 + 25.7).
constexpr int kFewRows = 16;
struct FewRowsParams {
  const void* x;            // [M, K], rows ldx apart
  long long ldx;
  const uint8_t* codes;     // W [N, Kp]
  const uint8_t* scales;
  const float* bias;        // [N] or null
  void* y;                  // [M, N] contiguous, in x's type
  int M, N, K;
};
cudaError_t few_rows_launch(const FewRowsParams& p, int elem, cudaStream_t s);

// SwiGLU over ab [M, 2 H] (rows ld apart). With g8: H a multiple of 128, of 16-bit types neither ck nor g8t (those are
// gemm8_swiglu_launch's), and map: ab {2 H, M, 1} in its type, box {128, 128, 1}
struct Swiglu8Params {
  const void* ab;
  long long ld;
  int M, H;
  void* g;                  // [M, H] in ab's type, or null
  uint8_t* ck;              // ab in 8 bits, [M, 2 Hp]: a's and b's blocks each from their own first column, or null
  uint8_t* ck_scales;       // of [M, 2 Hp]
  uint8_t* g8;              // g in 8 bits [M, Hp], or null
  uint8_t* g8_scales;
  uint8_t* g8t;             // [H, Mp] blocks along M, or null
  uint8_t* g8t_scales;
  const CUtensorMap* map;
  int* err;
};
cudaError_t swiglu8_fwd_launch(const Swiglu8Params& p, int elem, cudaStream_t s);
struct Swiglu8BwdParams {
  const void* dg;           // [M, H], rows ld apart
  long long ld;
  const uint8_t* ck;        // as the forward wrote it
  const uint8_t* ck_scales;
  int M, H;
  void* dab;                // [M, 2 H] in dg's type, or null
  uint8_t* d8;              // dab in 8 bits [M, 2 H] (H a multiple of 128), or null
  uint8_t* d8_scales;
  uint8_t* d8t;             // [2 H, Mp]
  uint8_t* d8t_scales;
  const CUtensorMap* map;     // with d8: dg {H, M, 1} in its type and ck {2 H, M, 1} as bytes, boxes {128, 128, 1}
  const CUtensorMap* ck_map;
  int* err;
};
cudaError_t swiglu8_bwd_launch(const Swiglu8BwdParams& p, int elem, cudaStream_t s);

}  // namespace tgo
