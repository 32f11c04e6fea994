// Launchers of topbeam.hip that the generation driver uses.
#pragma once
#include "common.h"

// scores: 0 for beam 0, -inf for the others; nobody is finished
void pcm_launch_beam_start(double *scores, uint8_t *finished, int beams,
                           int batch, hipStream_t st);
// sequences of the final beams from the (token, parent) records of G steps,
// both [G][beams][batch]
void pcm_launch_beam_trace(const int64_t *tokens, const int32_t *parents,
                           const double *scores, int beams, int batch, int G,
                           int64_t *best_out, int64_t *beams_out,
                           double *scores_out, hipStream_t st);
