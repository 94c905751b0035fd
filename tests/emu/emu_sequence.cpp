// TEST INFRASTRUCTURE: the sequence operators (causal_conv.hip, selective_scan.hip, layer_norm.hip, dropout.hip) compiled for the HOST
// against tests/emu/shim (see emu_conv_s16.cpp).
#include <hip/hip_runtime.h>

#include <cstdarg>

namespace pbsed {
alignas(16) thread_local float smem[40 * 1024];
}
#include "causal_conv.hip"
#include "dropout.hip"
#include "layer_norm.hip"
#include "selective_scan.hip"

namespace pbsed {
static char g_err[512];
void set_error(const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_err, sizeof(g_err), fmt, ap);
    va_end(ap);
}
int check_launch(const char*) { return 0; }
int device_cus() { return 8; }
}  // namespace pbsed
extern "C" const char* emu_last_error() { return pbsed::g_err; }
