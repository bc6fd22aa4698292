// The kernels of include/gqa_batch.h for bf16: a translation unit of its own, so that the two types compile side by side.
#include "gqa_batch_kernel.hpp"

template hipError_t mla::gqa::batch_launch<false>(const mla::gqa::BatchP & p, const mla::gqa::BatchPlan & pl, int dk, hipStream_t st);
