// The 4-bit matrix product kernels and their launcher (one translation unit of their own).
#define RQ_Q4_INSTANTIATE
#include "q4_mm.cuh"
