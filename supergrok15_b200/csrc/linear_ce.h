// Cross-entropy of a linear head without keeping the logits: arguments of the kernels (linear_ce.cu: CUDA cores and the row pass,
// linear_ce_sm100.cu: tensor cores).
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sg {

// One piece of the rows.  u is the only thing of the size [rows, vocabulary], and a piece is cut so that it stays below a fixed size.
struct LceArgs {
    const void *x, *w;                  // [rows, D] and [V, D]; the last index is contiguous
    int64_t ldx, ldw;
    const int64_t* target;              // [rows]; a target that is ignore_index or outside [0, V) is not counted
    int64_t ignore_index;
    int rows, V, D;
    void* u;                            // [rows, ldu], the type of x; null: no gradient is wanted
    int64_t ldu;                        // V rounded up to whole 16 bytes
    float *tile_max, *tile_sum;         // [tiles][rows]: maximum m of the row's logits in a tile of columns; sum of exp(z - m) without the target's column
    float* z_target;                    // [rows]: the target's logit
    float* loss;                        // [rows]
};

// dx = f d w (+ f dx_prev), dw = f d^T x (+ f dw_prev) for the d that lce_rows left in u; f = gout[0] * inv_count[0] / (the factor that u
// carries), or 1 without gout.  A null dx or dw is not wanted.
struct LceGrads {
    void *dx, *dw;                      // [rows, D], [V, D], dense
    const float* dw_prev;               // fp32 [V, D] of earlier pieces (may be dw itself), or null
    bool f32_out;                       // dx and dw are fp32, else the type of x
    const float *gout, *inv_count;
};

// u holds d times this: fp16 has no exponent to spare for probabilities (2^-17 for a flat row of 128,000 columns), bf16 and fp32 have
template <typename T> struct LceUnit { static constexpr float value = 1.f; };
template <> struct LceUnit<__half> { static constexpr float value = 32768.f; };

// columns per statistics tile of the kernels that will run
int lce_tile_columns(int dtype, const LceArgs& a);
// floats that lce_grads needs besides (partial sums of dx)
int64_t lce_scratch(int dtype, const LceArgs& a, bool dx, bool dw);

// Return 0 or the number of the step that failed.
int lce_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st);
int lce_rows(int dtype, const LceArgs& a, cudaStream_t st);
int lce_grads(int dtype, const LceArgs& a, const LceGrads& g, float* scratch, int* err, cudaStream_t st);
// out = in * gout * inv_count / (the factor of u), rounded to dtype
int lce_finish(int dtype, const float* in, void* out, int64_t n, const float* gout, const float* inv_count, cudaStream_t st);
// The tensor-core kernels; `err` (a device word) becomes non-zero when a wait inside a kernel ran out.
constexpr int LCE_SM100_COLUMNS = 128;
bool lce_sm100_takes(int dtype, const LceArgs& a);
int64_t lce_sm100_scratch(int rows, int V, int D, bool with_dw);
int lce_sm100_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st);
int lce_sm100_grads(int dtype, const LceArgs& a, const LceGrads& g, float* scratch, int* err, cudaStream_t st);
// out[0] = mean of the counted rows' losses, out[1] = 1 / max(count, 1)
void ce_mean(const float* loss, const int64_t* target, int64_t rows, int V, int64_t ignore_index, float* out, cudaStream_t st);

}  // namespace sg
