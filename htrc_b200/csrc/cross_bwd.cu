// placeholder
#include "cross.cuh"
extern "C" int htrc_cross_workspace_size(const HtrcCrossArgs*, size_t*) { return HTRC_ERR_UNSUPPORTED; }
extern "C" int htrc_cross_backward(const HtrcCrossArgs*, htrc_stream_t) { return HTRC_ERR_UNSUPPORTED; }
