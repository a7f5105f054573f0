// What kernels record for al_device_errors, and what that makes of it (host
// code only, without HIP, so that it is tested without a GPU).
#pragma once

#include <string>

#include "../../include/arclight_fattn.h"

// The device's words: of each kind a flag, then what the first of them was.
enum DeviceErrorWord {
    kErrSetRows = 0,                            // [1]: the row index
    kErrMerge = 2,
    kErrPaged = 4,                              // [5]: a PagedError, [6]: its value
    kErrLora = 8,                               // [9]: the adapter
    kErrWords = 12
};

enum PagedError { kPagedBadPage = 1, kPagedBadLength = 2, kPagedBadCount = 3, kPagedBadSeq = 4, kPagedBadPos = 5 };

inline std::string paged_error_text(const int what, const int value) {
    const std::string v = std::to_string(value);
    switch (what) {
        case kPagedBadPage:   return "sequence " + v + " has a page outside the pool";
        case kPagedBadLength: return "a length of " + v + " cells is not within the table";
        case kPagedBadCount:  return "a sequence with " + v + " new tokens";
        case kPagedBadSeq:    return "a token of sequence " + v + ", which the table does not have";
        default:              return "a token at position " + v + ", which is not within the table";
    }
}

// The status for the recorded words, and in `text` every kind of error among
// them, as all are cleared together. A merge that gave up is the library's own
// failure and keeps its status beside errors of the paged cache or the
// adapters, which are the caller's.
inline int device_error_status(const int (&w)[kErrWords], std::string & text) {
    text.clear();
    auto add = [&](const std::string & s) { text += (text.empty() ? "" : "; ") + s; };
    if (w[kErrSetRows]) add("set_rows: row index " + std::to_string(w[kErrSetRows + 1]) + " out of range (ops.cpp:171)");
    if (w[kErrMerge]) add("fattn: a merging workgroup gave up waiting for the other splits' records");
    if (w[kErrPaged]) add("paged cache: " + paged_error_text(w[kErrPaged + 1], w[kErrPaged + 2]));
    if (w[kErrLora]) add("lora: a row of adapter " + std::to_string(w[kErrLora + 1]) + ", which is not there or whose rank does not fit");
    if (text.empty()) return AL_OK;
    return w[kErrMerge] && !w[kErrSetRows] ? AL_ERR_HIP : AL_ERR_INVALID;
}
