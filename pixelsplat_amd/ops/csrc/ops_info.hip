// Which sources libpixelsplat_ops.so was built from.
#include "pixelsplat_ops.h"

#ifndef PS_BUILD_HASHES
#define PS_BUILD_HASHES ""
#endif

extern "C" const char* ps_ops_build_info(void) { return "pixelsplat_ops gfx950 | " PS_BUILD_HASHES; }
