// Arguments of the kernels between a round's logits and its tokens (token_counts.cu, sample_rows.cu), shared with the bindings that fill them.
#pragma once
#include <stdint.h>

namespace spark {

// This file as a number (given by the build): the bindings launch only kernels that were compiled from the same one.
#ifndef SPARK_SAMPLING_LAYOUT
#define SPARK_SAMPLING_LAYOUT 0u
#endif

constexpr int SAMPLE_MAX_V = 768 * 1024;           // columns of a row: 98 KB of the largest of every 32 logits, if one CTA has it (asserted in sample_rows.cu)
constexpr int SAMPLE_MAX_LIST = 1024;              // drafted tokens, biases of a row
constexpr int SAMPLE_MAX_TOP = 256;                // most probable tokens of a row

enum LogitType : int { LT_F32 = 0, LT_BF16 = 1, LT_F16 = 2 };

struct CountTokens {
  int* counts;                                     // [n_slots, V], rows ld_counts apart: 2 * times generated + (1 if in the prompt)
  const int *tokens, *n, *slots;                   // [S, P], rows ld_tokens apart; [S]; [S] (null: the requests' numbers)
  int* status;
  long long ld_counts, ld_tokens;
  int S, P, V, n_slots, prompt, reset;
};

struct Adjustments {                               // of rows; null pointers: none of the kind
  const int *counts, *slots;                       // a row's row of `counts` (null: its number; negative: it has no penalties)
  const int* drafted;                              // [R, n_drafted] tokens that count as generated on top, negative: none
  const float *repetition, *presence, *frequency;  // [R]
  const int* bias_ids;                             // [R, n_bias], negative: none
  const float* bias;
  const uint32_t* allowed;                         // [R, words] bits
  long long ld_counts;
  int n_slots, n_drafted, n_bias, words;
};

struct AdjustRows {
  const void* x;                                   // [R, V] of ids offset .. offset + V
  float* out;
  long long ldx, ldo;
  int* status;
  int R, V, type, offset, sms;
  Adjustments a;
};

struct SampleRows {
  const void* x;                                   // [R, V]
  long long ldx;
  const float* temps;                              // [R] each
  const long long *seeds, *positions;
  const int* top_k;                                // null: off
  const float *top_p, *min_p;
  int *out, *status;
  int R, V, type, sms;
};

struct LogprobRows {
  const void* x;
  long long ldx;
  const int* tokens;                               // [R]
  float* logprob;                                  // [R]
  int* rank;                                       // [R]
  int* ids;                                        // [R, top]
  float* logprobs;                                 // [R, top]
  int* status;
  int R, V, type, sms, top;
};

}  // namespace spark
