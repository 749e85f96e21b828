// The device-side status word of the library (0 = fine).  A kernel that gives up on a bounded wait records why here
// instead of spinning, one that meets borders of sequences which it cannot follow says so; the host reads and clears it through
// cs2d_device_status().
#pragma once

#include <cstddef>
#include <cstdio>

namespace cs2d {

enum { ERR_BULK_COPY_TIMEOUT = 1, ERR_STAGE_TIMEOUT = 2, ERR_WORKER_TIMEOUT = 4, ERR_SEQ_OFFSETS = 8 };

// What the word says.
inline void status_text(char *text, size_t size, int status) {
    const int waits = status & (ERR_BULK_COPY_TIMEOUT | ERR_STAGE_TIMEOUT | ERR_WORKER_TIMEOUT);
    const char *offsets = (status & ERR_SEQ_OFFSETS) ? "sequence offsets that do not ascend or leave the tensor" : "";
    if (waits || !offsets[0])
        snprintf(text, size, "a kernel gave up on a bounded wait (status %d:%s%s%s%s%s); its outputs are invalid", status,
                 (status & ERR_BULK_COPY_TIMEOUT) ? " bulk copy" : "", (status & ERR_STAGE_TIMEOUT) ? " staging warps" : "",
                 (status & ERR_WORKER_TIMEOUT) ? " row workers" : "", offsets[0] ? " and " : "", offsets);
    else
        snprintf(text, size, "a kernel met %s (status %d:); its outputs are invalid", offsets, status);
}

}  // namespace cs2d
