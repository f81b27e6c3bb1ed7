/* The C ABI without a GPU: allocations come from the heap, and the operators
 * do nothing but count that they were reached. */
#include <stddef.h>
#include <stdlib.h>

int operators_reached;

int vc_cuda_alloc(size_t bytes, void** pointer) { return (*pointer = malloc(bytes)) ? 0 : 4; }
int vc_cuda_free(void* pointer) { free(pointer); return 0; }
const char* vc_cuda_last_error(void) { return "not there"; }
int vc_cuda_available(void) { return 1; }

#define OPERATOR(name) int name(void) { ++operators_reached; return 0; }
OPERATOR(vc_cuda_rms_norm)
OPERATOR(vc_cuda_rms_norm_backward)
OPERATOR(vc_cuda_rms_norm_q8)
OPERATOR(vc_cuda_quantize_q8)
OPERATOR(vc_cuda_matmul_q8)
OPERATOR(vc_cuda_sample)

#define ABSENT(name) int name(void) { return 5; }
ABSENT(vc_cuda_device_name)
ABSENT(vc_cuda_upload)
ABSENT(vc_cuda_download)
ABSENT(vc_cuda_binary)
ABSENT(vc_cuda_unary)
ABSENT(vc_cuda_matmul)
ABSENT(vc_cuda_transpose_last2)
ABSENT(vc_cuda_reduce_all)
ABSENT(vc_cuda_reduce_axis)
ABSENT(vc_cuda_scatter_axis)
ABSENT(vc_cuda_axpy)
ABSENT(vc_cuda_synchronize)
ABSENT(vc_cuda_broadcast_to)
ABSENT(vc_cuda_reduce_axis_backward)
ABSENT(vc_cuda_sum_to_shape)
ABSENT(vc_cuda_binary_backward)
ABSENT(vc_cuda_unary_backward)
ABSENT(vc_cuda_softmax)
ABSENT(vc_cuda_log_softmax)
ABSENT(vc_cuda_softmax_backward)
ABSENT(vc_cuda_log_softmax_backward)
ABSENT(vc_cuda_cross_entropy)
ABSENT(vc_cuda_cross_entropy_backward)
