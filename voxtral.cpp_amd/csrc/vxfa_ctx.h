// vxfa_ctx.h — a context's workspace and switches, shared by the entry points'
// translation units (vxfa_api.cpp, vxfa_paged.cpp).
#pragma once

#include <stddef.h>
#include <stdlib.h>

// Device workspace of a context, allocated once by vxfa_ctx_create (no call
// allocates, frees or synchronises): the split-KV partial records and f16
// staging for F32 K/V of prefill calls.
constexpr size_t kRecordBytes = (size_t)8 << 20;        // decode records: e.g. 256 (batch, kv head) pairs x 8 splits, or 8 x 64
constexpr size_t kStageBytes = (size_t)32 << 20;        // F32 K and V of 8192 rows x 1024 as f16
constexpr size_t kWorkspaceBytes = kRecordBytes + kStageBytes;

// Launch-shape overrides for tuning sweeps (VXFA_DECODE_SPLIT,
// VXFA_PREFILL_WAVES; 0 = heuristic) and route switches for tests and
// measurements, read from the environment when a context is created.
struct Tuning {
    int split_override = 0;
    int waves_override = 0;
    // VXFA_PREFILL_PP=0 routes hd 64 prefill to the general kernel
    bool pp_enabled = true;
    // VXFA_PREFILL_PAIR=0 routes short masked hd 128 prefill to the general kernel
    bool pair_enabled = true;
    // VXFA_PAIR_INTERVALS=0: with F32 K/V and a mask tensor the short masked
    // prefill classifies its blocks from the mask itself rather than from the
    // intervals a pre-pass finds in the staging launch
    bool pair_intervals = true;
    // VXFA_DECODE_ROWS: batched decode with a mask tensor of one head plane
    // finds its rows' live ranges by a pre-pass always (1) or never (0)
    int decode_rows = -1;
    // VXFA_PREFILL_GROUP: hd 128 prefill on the grouped kernel wherever it can (1)
    // or never (0)
    int group = -1;
    // VXFA_ROPE_Q=0: no scratch for rotated queries, as for a call whose rows do
    // not fit it
    bool rope_q = true;
    // VXFA_PAGED_PIECES: pieces of the longest walk of a paged chunk call (0: the
    // plan's choice)
    int paged_pieces = 0;
    void read_env() {
        if (const char* e = getenv("VXFA_DECODE_SPLIT")) split_override = atoi(e);
        if (const char* e = getenv("VXFA_PREFILL_WAVES")) waves_override = atoi(e);
        if (const char* e = getenv("VXFA_PREFILL_PP")) pp_enabled = atoi(e) != 0;
        if (const char* e = getenv("VXFA_PREFILL_PAIR")) pair_enabled = atoi(e) != 0;
        if (const char* e = getenv("VXFA_PAIR_INTERVALS")) pair_intervals = atoi(e) != 0;
        if (const char* e = getenv("VXFA_ROPE_Q")) rope_q = atoi(e) != 0;
        if (const char* e = getenv("VXFA_PREFILL_GROUP")) group = atoi(e) != 0;
        if (const char* e = getenv("VXFA_PAGED_PIECES")) paged_pieces = atoi(e);
        if (const char* e = getenv("VXFA_DECODE_ROWS")) decode_rows = atoi(e) != 0;
    }
};

// Where one call may put its device scratch (split-KV partial records of a
// decode call, f16 staging of F32 K/V of a prefill call) and its error
// message: a context's workspace, or the library's static scratch array.
struct Workspace {
    int device;
    char* base;           // one area, 256-byte aligned: a decode call's split-KV
    size_t bytes;         // records, or a prefill call's staged K/V, mask row
                          // intervals and piece records, in that order
    char* pieces;         // prefill piece records, where they have an area of their own (of
                          // kWorkspaceBytes) rather than what is left at base
    size_t rec_bytes;     // of it, most that decode records take
    size_t stage_bytes;   // of it, most that staged F32 K/V take
    char* err;            // message of the last failure
    size_t err_len;
    Tuning tune;
};

struct vxfa_ctx {
    int device = 0;
    char* ws = nullptr;           // kWorkspaceBytes of device memory
    char last_error[256] = {0};
    Tuning tune;                  // read once when the context is created
    Workspace view() {
        return Workspace{device, ws, kWorkspaceBytes, nullptr, kRecordBytes, kStageBytes, last_error,
                         sizeof(last_error), tune};
    }
};
