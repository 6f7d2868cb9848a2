// Verification of drafted tokens: parameters shared by the launcher and the kernels (gfa_verify.hip).
#pragma once
#include <stdint.h>

namespace gfa {

// Vocabulary entries that a wave takes at once, eight a lane; a segment is a multiple of them.
constexpr int kVerifyStep = 512;

struct VerifyParams {
  const void *target, *draft;  // (T, V), rows apart by ts, ds elements; draft NULL: tokens proposed for certain
  int64_t ts, ds;
  const int64_t* tokens;  // (T)
  const float *accept, *sample;
  const int *lens, *cu;  // cu NULL: `each` tokens a request
  int T, V, R, each;
  int segment, segments;  // entries of a wave, waves of a request
  double* sums;           // (R, segments, 2): residual weights and target's probabilities
  int* taken;             // (R): drafted tokens accepted
  int64_t* follows;       // (T)
  int *accepted, *lens_out;
};

}  // namespace gfa
