// Newton-Schulz products on the tensor cores: what muon.cu needs of newton_schulz.cu.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "hybridagent_b200.h"

namespace ha {

// Fixed-point scales of the 16-bit planes (powers of two, so they cost no rounding): an element of
// X is at most its largest singular value and starts near 1 / sqrt(rows * cols); fp16 holds
// normal numbers from 2^-14 up to 65504.
constexpr float kScaleX = 4096.0f;   // X planes hold 2^12 x
constexpr float kScaleG = 1024.0f;   // Gram and polynomial planes hold 2^10 times theirs
constexpr float kScaleLo = 2048.0f;  // the low plane holds 2^11 (2^12 x - high plane)

// A batch of `n` matrices of one shape in workspace.  Rows are padded to 8 elements.
struct NsBatch {
  int64_t n, rows, cols;
  int64_t ld_x, ld_g, m;         // padded row lengths; m = min(rows, cols)
  int64_t plane_x, plane_g;      // elements of one matrix
  __half *hi[2], *lo;            // X before and after a step; low plane
  __half* square[3];             // m x m: Gram matrices and factors
  float4* diagonal[3];           // what rounding took from their diagonals, m_pad elements for each matrix
  int64_t m_pad;
  uint32_t* counter;             // one for each matrix, zero before the run
  uint32_t* error;               // set to 1 if a wait ran out
  bool bf16;                     // the result is wanted as bf16 (a run of this shape alone) ...
  uint16_t* dst;                 // ... in packed matrices with 16-byte aligned rows, if set
  int out;                       // after a run: the high plane that holds the result, or -1 if dst does
  bool rounded;                  // after a run: the result is bf16 (not 2^12 times it in fp16)
};
constexpr int kNsShapes = 6;     // of one run

// The largest |a t + b t^3 + c t^5| and |a + b t^2 + c t^4| of a step for 0 <= t <= s: how far it can
// carry singular values up to s, and what it multiplies X by.
double ns_growth(const float* coef, double s);
double ns_factor(const float* coef, double s);
constexpr double kMaxGrowth = 4.0, kMaxFactor = 60.0;  // what the planes hold, with room for rounding

// Bytes that one matrix takes (a multiple of 256).
int64_t ns_bytes_per_matrix(int64_t rows, int64_t cols);
// Lays the planes of b->n matrices out from `base` on.
void ns_carve(NsBatch* b, void* base);

// Map of X-shaped planes, read or written in box_cols x box_rows pieces (128-byte swizzled rows).
int ns_map(CUtensorMap* map, const __half* plane, const NsBatch& b, int box_cols, int box_rows);

// Matrices whose shorter side is at most 128, if the steps' factors fit (newton_schulz_narrow.cu).
bool narrow_fits(int64_t rows, int64_t cols, const float* coef, int steps);
int narrow_run(NsBatch* shape, const float* coef, int steps, int sms, cudaStream_t st);

// Stages that a shape takes at most; a run's shapes take kNsStages together.
int ns_stages(int steps);
constexpr int kNsStages = 128;

// Runs `steps` Newton-Schulz steps on hi[0] (+ lo) of up to kNsShapes shapes, whose counters lie one after
// another in their order.
int ns_run(NsBatch* shapes, int n, const float* coef, int steps, cudaStream_t st);

}  // namespace ha
