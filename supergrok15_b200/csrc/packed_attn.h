// Arguments of the packed-attention kernels (packed_attn.cu: CUDA cores, packed_attn_sm100.cu: tensor cores).
#pragma once
#include "packed_seq.cuh"

namespace sg {

struct PackedAttn {
    const void *q, *k, *v;              // [total, heads, hd], [total, heads / group, hd]; the last index is contiguous
    int64_t q_ld, k_ld, v_ld;           // elements between rows
    int64_t q_hs, k_hs, v_hs;           // elements between heads
    void* out;                          // [total, heads, hd], dense
    void* out_lo;                       // 16-bit training: what the rounding took from `out`, in the same type and layout; else null
    float* lse;                         // [heads, total], null without a backward pass
    const void* dout;                   // backward: dense like out
    float* delta;                       // scratch [heads, total]
    void *dq, *dk, *dv;                 // dense
    float* kv_parts;                    // scratch of 2 * packed_attn_sm100_split(p) * total * key heads * hd floats, where that is above 1
    float* units;                       // scratch of packed_attn_sm100_units(dtype, p) floats, where that is above 0
    PackedSeqs seqs;
    int heads, group, hd, causal;
    float scale;
};

// Return 0 or the number of the step that failed.
int packed_attn_fwd(int dtype, const PackedAttn& p, cudaStream_t st);
int packed_attn_bwd(int dtype, const PackedAttn& p, cudaStream_t st);
// what the tensor-core kernels' loads ask of a 16-bit [rows, heads, hd] view: a 16-byte aligned base, pitches of whole 16 bytes below 2^39
inline bool packed_tma_view(const void* base, int64_t ld, int64_t hs, int64_t rows, int64_t heads) {
    const auto pitch = [](int64_t n, int64_t count) { return count <= 1 || (n > 0 && n % 8 == 0 && n < (int64_t)1 << 38); };
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && pitch(ld, rows) && pitch(hs, heads);
}
// The tensor-core kernels; `err` (a device word) becomes non-zero when a wait inside a kernel ran out.
bool packed_attn_sm100_takes(int dtype, const PackedAttn& p);
int packed_attn_sm100_split(const PackedAttn& p);
int64_t packed_attn_sm100_units(int dtype, const PackedAttn& p);
int packed_attn_sm100_fwd(int dtype, const PackedAttn& p, int* err, cudaStream_t st);
int packed_attn_sm100_bwd(int dtype, const PackedAttn& p, int* err, cudaStream_t st);

}  // namespace sg
