/* gfx950 code object of the text operators: every kernel that the runtime
 * looks up in it by name (h3_gpu_text.inc). */
#include "kernels/common.h"
#include "kernels/rotary.h"
#include "kernels/paged_attention.h"
#include "kernels/linear_int4.h"
