// The hash of the sources the library was built from, in a source of its own: the others then need not be compiled
// again when only the hash changes.
#include "fbev.h"

#ifndef FBEV_SOURCE_HASH
#define FBEV_SOURCE_HASH "unknown"
#endif
extern "C" const char* fbev_source_hash(void) { return FBEV_SOURCE_HASH; }
