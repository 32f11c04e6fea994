// Launchers of topbeam.hip that the generation driver uses.
#pragma once
#include "common.h"

// scores: 0 for beam 0, -inf for the others; nobody is finished.  end_in (nullable):
// the end token on the device; *end_at becomes it, or -1 (no token) if it is
// negative or, reported in *status, not below vocab
void pcm_launch_beam_start(double *scores, uint8_t *finished, int beams,
                           int batch, const int64_t *end_in, int vocab,
                           int32_t *end_at, int32_t *status, hipStream_t st);
// pcm_beam_select with the end token at end_at on the device (-1: no token; nobody
// may be finished then), or null: end_token
int pcm_launch_beam_select(const void *logits, int32_t dtype, int64_t ld,
                           const double *scores, const uint8_t *finished,
                           int32_t beams, int32_t batch, int32_t vocab,
                           int32_t width, double temperature, int32_t end_token,
                           const int32_t *end_at, int64_t *tokens,
                           int32_t *parents, double *scores_out,
                           uint8_t *finished_out, void *workspace,
                           size_t workspace_bytes, hipStream_t st);
// sequences of the final beams from the (token, parent) records of G steps,
// both [G][beams][batch]
void pcm_launch_beam_trace(const int64_t *tokens, const int32_t *parents,
                           const double *scores, int beams, int batch, int G,
                           int64_t *best_out, int64_t *beams_out,
                           double *scores_out, hipStream_t st);
