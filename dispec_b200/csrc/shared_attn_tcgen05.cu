// Attention of sequences with a shared beginning on the tensor cores (the formula: shared_attn.cu; how the work is cut and what a
// row sees: shared_schedule.cuh).  Compiled once per head size (-DDSP_HEAD_DIM=32, 64 or 128; of 32, without the
// kernel for many rows).
#include "shared_attn_few.cuh"
#if DSP_HEAD_DIM >= 64
#include "shared_attn_many.cuh"
#endif

// The arguments come checked from dsp_shared_attention (shared_attn.cu), which also launches the merge.
extern "C" int DSP_CAT(dsp_shared_attention_few_d, DSP_HEAD_DIM)(const DspSharedAttention* a, cudaStream_t stream) {
  return launch_shared_few(*a, stream);
}
#if DSP_HEAD_DIM >= 64
extern "C" int DSP_CAT(dsp_shared_attention_many_d, DSP_HEAD_DIM)(const DspSharedAttention* a, cudaStream_t stream) {
  return launch_shared_many(*a, stream);
}
#endif
