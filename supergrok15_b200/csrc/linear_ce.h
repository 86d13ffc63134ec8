// Cross-entropy of a linear head without keeping the logits: arguments of the kernels (linear_ce.cu: CUDA cores and the row pass,
// linear_ce_sm100.cu: tensor cores).
#pragma once
#include <cstdint>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

namespace sg {

// One piece of the counted rows.  Rows whose target is ignore_index or lies outside [0, V) are left out before anything is computed
// (lce_gather), so how many rows there are is known on the device only: the arrays are sized for all of them, and every kernel reads the count.
// u is the only thing of the size [rows, vocabulary], and a piece is cut so that it stays below a fixed size.
struct LceArgs {
    const void *x, *w;                  // [rows, D], the counted rows of this piece one after the other, and [V, D]; the last index is contiguous
    int64_t ldx, ldw;                   // rows of x start on 128 bytes on the tensor cores (lce_pitch), so that a box of 64 columns is whole lines
    const int64_t* target;              // [rows], in [0, V)
    const int* count;                   // counted rows of all pieces; this one holds [first, first + rows) of them
    int first, rows, V, D;
    void* u;                            // [rows, ldu], the type of x; null: no gradient is wanted
    int64_t ldu;                        // lce_pitch of V
    float2* stats;                      // [rows][tiles]: reference r of the row's logits in a tile of columns (in powers of two), sum of 2^(z log2 e - r)
                                        // without the target's column
    float* row_scale;                   // [rows], bf16 on the tensor cores: what a row of u still has to be multiplied by; else null
    float* z_target;                    // [rows]: the target's logit
    float* loss;                        // [rows]
    // the last piece's row pass adds up: loss_all [all counted rows] -> out_loss = mean, inv_count = 1 / max(count, 1); done: a zero
    const float* loss_all;
    float *out_loss, *inv_count;
    unsigned* done;
};
#ifdef __CUDACC__
__device__ __forceinline__ int lce_active(const LceArgs& a) {
    const int n = __ldcg(a.count) - a.first;
    return n < 0 ? 0 : (n < a.rows ? n : a.rows);
}
#endif

// dx_part[s] = (part s of) f d w in fp32, [parts][row_pitch][D], dw = f d^T x (+ f dw_prev) for the d that lce_rows left in u;
// f = gout[0] * inv_count[0] / (the factor that u carries), or 1 without gout.  A null dx_part or dw is not wanted.
struct LceGrads {
    float* dx_part;
    int parts;                          // lce_dx_parts
    int64_t row_pitch;
    void* dw;                           // [V, D], dense
    const float* dw_prev;               // fp32 [V, D] of earlier pieces (may be dw itself), or null
    bool f32_dw;                        // dw is fp32, else the type of x
    const float *gout, *inv_count;
};

// Whether lce_rows leaves u as it is and scales the rows of x instead (see linear_ce.cu): the references of nearly all tiles are equal
bool lce_scales_rows(int dtype, const LceArgs& a);

// elements from row to row of what the operator lays out itself
inline int64_t lce_pitch(int64_t n, int64_t elem) { const int64_t per = (elem == 2 ? 128 : 16) / elem; return (n + per - 1) / per * per; }

// u holds d times this: fp16 has no exponent to spare for probabilities (2^-17 for a flat row of 128,000 columns), bf16 and fp32 have
template <typename T> struct LceUnit { static constexpr float value = 1.f; };
template <> struct LceUnit<__half> { static constexpr float value = 32768.f; };

constexpr int LCE_COLUMNS = 128;        // columns per statistics tile
// parts that dx is summed in, and rows from one part to the next
int lce_dx_parts(int dtype, const LceArgs& a, bool with_dw, int64_t* row_pitch);

// Return 0 or the number of the step that failed.
// The counted rows in order: place[row] = where it went or -1, xc and tc = their rows of x (pitch ldx) and targets, count[0] = how many, done[0] = 0.
// xc has lce_pitch(D) elements per row; its rows from the count to the next multiple of 64 are zero.  blocks: scratch of lce_gather_blocks(rows) ints.
int lce_gather_blocks(int rows);
int lce_gather(int dtype, const void* x, int64_t ldx, const int64_t* target, int64_t ignore_index, int rows, int V, int D, int* place, void* xc, int64_t* tc,
               int* count, unsigned* done, int* blocks, cudaStream_t st);
int lce_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st);
int lce_rows(int dtype, const LceArgs& a, bool last, cudaStream_t st);
int lce_grads(int dtype, const LceArgs& a, const LceGrads& g, int* err, cudaStream_t st);
// out[i] = the sum of the parts in order, `pitch` floats from one to the next
int lce_add_parts(const float* part, int parts, int64_t pitch, int64_t n, float* out, cudaStream_t st);
// dx[row] of all rows: zero where place is -1; early[place] * gout * inv_count / (the factor of u) where place < first; else the sum of the
// parts of row place - first (scaled already).  D columns, dtype.
int lce_scatter(int dtype, const int* place, int rows, int D, int first, const float* early, const float* part, int parts, int64_t row_pitch, const float* gout,
                const float* inv_count, void* dx, cudaStream_t st);

// The tensor-core kernels; `err` (a device word) becomes non-zero when a wait inside a kernel ran out.
bool lce_sm100_takes(int dtype, const LceArgs& a);
int lce_sm100_dx_parts(int rows, int V, int D, bool with_dw, int64_t* row_pitch);
int lce_sm100_logits(int dtype, const LceArgs& a, int* err, cudaStream_t st);
int lce_sm100_grads(int dtype, const LceArgs& a, const LceGrads& g, int* err, cudaStream_t st);

}  // namespace sg
