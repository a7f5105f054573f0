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
    kErrDraft = 12,                             // [13]: a DraftError, [14]: its value
    kErrWords = 16
};

enum PagedError {
    kPagedBadPage = 1, kPagedBadLength = 2, kPagedBadCount = 3, kPagedBadSeq = 4, kPagedBadPos = 5, kPagedBadCell = 6, kPagedBadPath = 7,
    kPagedBadKept = 8, kPagedBadCopy = 9, kPagedBadCells = 10
};
enum DraftError { kDraftBadParent = 1, kDraftBadCount = 2, kDraftBadToken = 3, kDraftBadRow = 4 };

inline std::string paged_error_text(const int what, const int value) {
    const std::string v = std::to_string(value);
    switch (what) {
        case kPagedBadPage:   return "sequence " + v + " has a page outside the pool";
        case kPagedBadLength: return "a length of " + v + " cells is not within the table";
        case kPagedBadCount:  return "a sequence with " + v + " new tokens";
        case kPagedBadSeq:    return "a token of sequence " + v + ", which the table does not have";
        case kPagedBadCell:   return "a token of cell " + v + ", which is not within the table";
        case kPagedBadPath:   return "new token " + v + " is not one that can be kept in its place of the path";
        case kPagedBadKept:   return "a path of " + v + " tokens, more or fewer than there can be";
        case kPagedBadCopy:   return "page " + v + " of a copy is not in the pool";
        case kPagedBadCells:  return "a copy of " + v + " cells of a page";
        default:              return "a token at position " + v + ", which is not within the table";
    }
}

inline std::string draft_error_text(const int what, const int value) {
    const std::string v = std::to_string(value);
    switch (what) {
        case kDraftBadParent: return "a node whose parent is " + v + ", which does not come before it";
        case kDraftBadCount:  return "a tree of " + v + " nodes, more or fewer than there can be";
        case kDraftBadToken:  return "a node of token " + v + ", which the vocabulary does not have";
        default:              return "sequence " + v + " has no probabilities to draw from";
    }
}

// The status for the recorded words, and in `text` every kind of error among
// them, as all are cleared together. A merge that gave up is the library's own
// failure and keeps its status beside errors of the paged cache, the adapters
// or drafts, which are the caller's.
inline int device_error_status(const int (&w)[kErrWords], std::string & text) {
    text.clear();
    auto add = [&](const std::string & s) { text += (text.empty() ? "" : "; ") + s; };
    if (w[kErrSetRows]) add("set_rows: row index " + std::to_string(w[kErrSetRows + 1]) + " out of range (ops.cpp:171)");
    if (w[kErrMerge]) add("fattn: a merging workgroup gave up waiting for the other splits' records");
    if (w[kErrPaged]) add("paged cache: " + paged_error_text(w[kErrPaged + 1], w[kErrPaged + 2]));
    if (w[kErrLora]) add("lora: a row of adapter " + std::to_string(w[kErrLora + 1]) + ", which is not there or whose rank does not fit");
    if (w[kErrDraft]) add("draft: " + draft_error_text(w[kErrDraft + 1], w[kErrDraft + 2]));
    if (text.empty()) return AL_OK;
    return w[kErrMerge] && !w[kErrSetRows] ? AL_ERR_HIP : AL_ERR_INVALID;
}
