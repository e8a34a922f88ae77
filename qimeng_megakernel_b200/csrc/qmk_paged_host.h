// Host-side interface between the C ABI of the decode step (qmk_api.cu) and the paged-cache entry points (qmk_paged.cu).
#pragma once
#include "../../include/qmk_b200.h"

// What qmk_prefix_attention checks before it launches anything.
int qmk_prefix_attention_check(const qmk_prefix_attention_args* a, int device);

// qmk_prefix_attention as part of a step: failures on the device go to a status record (null: to nowhere; the rows are NaN).
struct qmk_attention_watch {
  unsigned* status;          // device address of the record
  int phase;                 // number of the phase, for the record
  long long wait_cycles;     // budget of a wait in SM clocks
  int wait_first;            // failure test: waits for an arrival that nothing makes
};
int qmk_prefix_attention_launch(const qmk_prefix_attention_args* a, const qmk_attention_watch* w, int device, void* cuda_stream);
