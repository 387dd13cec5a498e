// A context's status word, for tests that put a code there.
#include "common.cuh"

extern "C" void* t_status(void* ctx) { return static_cast<loom_b200_ctx*>(ctx)->status_dev; }
