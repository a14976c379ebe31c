// Attention of drafted trees on the tensor cores (the formula: tree_attn.cu; the kernel: rows_attn_tcgen05.cuh; how the work is
// cut and what a node sees: tree_schedule.cuh).  Compiled once per head size (-DDSP_HEAD_DIM=64 or 128).
#include "tree_schedule.cuh"
#include "rows_attn_tcgen05.cuh"

// The arguments come checked from dsp_tree_attention (tree_attn.cu), which also launches the merge.
extern "C" int DSP_CAT(dsp_tree_attention_tcgen05_d, DSP_HEAD_DIM)(const DspTreeAttention* a, cudaStream_t stream) {
  return launch_rows_attn_tcgen05<TreeWork>(*a, stream);
}
