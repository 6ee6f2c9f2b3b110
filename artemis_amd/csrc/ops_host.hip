// ops_host.hip -- error text and identification of libartemis_ops.so.
#include <stdarg.h>
#include <stdio.h>

#include "ops_common.hpp"

namespace aops {

static thread_local char g_last_error[512] = "";

int fail(int code, const char *fmt, ...)
{
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
    va_end(ap);
    return code;
}

int check_launch(const char *what)
{
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail((int)e, "%s: %s", what, hipGetErrorString(e));
    return 0;
}

}  // namespace aops

extern "C" {

const char *artemis_ops_version(void)
{
    return "artemis_ops abi 1 gfx950 hip (layer norm, window attention, adamw 32 and 8 bit)";
}

const char *artemis_ops_last_error(void) { return aops::g_last_error; }

}  // extern "C"
