// Host-side validation and layout for the objectives (losses over rows of logits).
// Pure C++ (no HIP headers), as mamw_plan.h.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "muonadamw_amd.h"

namespace mamw {

// Rows of one count where sequences do not matter: every row's workgroup adds up all counts, which is a load a lane up to
// 65536 rows.
constexpr int kCountRows = 1024;
// Counts of sequences, at most: a load a lane.  With a count a sequence the loss took 72 us instead of 50 over 2048
// sequences of 8 rows of 4000 bf16.
constexpr int kCountGroups = 64;
// Workgroups of the kernel that adds up the rows' parts of a result, at most.
constexpr int kResultBlocks = 64;
// Rows of teacher's entries that one workgroup prepares.
constexpr int kTeacherRows = 16;
// Bits of the table of a teacher's indices in rows that are not held whole (128 KiB of LDS at most).
constexpr int64_t kMaxTailVocab = int64_t(1) << 20;

// A workspace: how many rows count, of each kCountRows (or how many sequences have such rows, of each group of them); the
// length of each row's sequence (policy, by sequence) or its teacher's entries; the rows' parts of the result.
struct ObjectiveWorkspace {
    int64_t items;      // counts
    size_t ticket_at;   // bytes from the start; kResultBlocks parts of 16 bytes behind 256
    size_t lengths_at;
    size_t partials_at;
    size_t bytes;
};
ObjectiveWorkspace objective_workspace(int64_t items, int64_t lengths, int64_t partials);

// MAMW_OK or the first error; *ws is set where it is MAMW_OK.  `grad` may be NULL.
int check_rows(const mamw_rows* x, const void* grad);
int check_per_row(const mamw_per_row& a, bool needed, int32_t type, int32_t other_type = -1);
int check_policy(const mamw_rows* x, const mamw_policy* p, const void* grad, ObjectiveWorkspace* ws);
int check_preference(const mamw_rows* x, const mamw_preference* p, ObjectiveWorkspace* ws);
int check_distill(const mamw_rows* x, const mamw_distill* p, const void* grad, ObjectiveWorkspace* ws);
int check_workspace(const ObjectiveWorkspace& ws, const void* workspace, size_t bytes);
int check_temperature(float t);

}  // namespace mamw
