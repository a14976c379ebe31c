/* What C code is told of a tensor (written by describe.cpp). */
#ifndef DSP_TENSOR_DESC_H
#define DSP_TENSOR_DESC_H
enum { DSP_T_F32 = 0, DSP_T_BF16 = 1, DSP_T_I32 = 2, DSP_T_I64 = 3, DSP_T_OTHER = -1 };
#define DSP_T_DIMS 5
typedef struct {
  void* data;
  int dtype, device; /* device -1: not on a CUDA device */
  int dims;          /* -1: None; sizes and strides of the first DSP_T_DIMS */
  int contiguous;
  long size[DSP_T_DIMS], stride[DSP_T_DIMS];
} DspTensor;
#endif
