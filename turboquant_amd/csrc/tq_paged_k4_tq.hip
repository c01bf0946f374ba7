// tq_paged_k4_tq.hip -- the fused decode kernels for 4-bit TQ (PQ records with the QJL correction)
// records in pages, with the inline split-K merge.
#include "tq_decode_kernel.h"

namespace tqa {
template void launch_stream_bm<4, kModeTq, true, PageArgs>(AttnArgs &, int, int, dim3, hipStream_t, PageArgs *);
}  // namespace tqa
