// Beam selection (beam.hip): what its launch takes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mlq {

constexpr int kBeamMostBeams = 64;  // of a group
constexpr int kBeamMostKeep = 64;
constexpr int kBeamMostVocab = 1 << 30;
constexpr int kBeamPart = 8192;     // logits of a part of a row
constexpr int kBeamSmallPart = 2048;

// Logits of a part: small ones where the large ones are few.  Large and small: 1 beam over 32000 tokens 13.5 and 11.5 us,
// 4 (16 large parts) 13.9 and 11.4, 16 (64) 14.4 and 16.0, 8 over 128011 (128) 14.5 and 17.5.
inline int beam_part(long long rows, int vocab) {
    return rows * ((vocab + kBeamPart - 1) / kBeamPart) < 32 ? kBeamSmallPart : kBeamPart;
}
// Parts of as many rows at the most.
inline size_t beam_parts(long long rows, int vocab) {
    const size_t large = static_cast<size_t>(rows) * ((vocab + kBeamPart - 1) / kBeamPart);
    // (fewer rows or tokens may be cut finer: below 32 large parts, four of each)
    return large > 128 ? large : 128;
}

// A part of a row: its largest logit and the sum of exp(logit - largest).
struct BeamPart {
    double sum;
    float largest;  // NaN: a logit is NaN or +Inf
    int pad;
};

struct BeamCall {
    const float* logits;  // [groups][beams][vocab]
    const float* scores;  // [groups][beams]
    const int* ended;     // [groups][beams], or null
    int end_token, groups, beams, vocab, keep;
    int *parents, *tokens;  // [groups][keep]
    float* out_scores;      // [groups][keep]
    // Workspace: of every part its BeamPart and the keys of its best `keep` logits, [groups][keep][parts of the group].
    BeamPart* parts;
    unsigned long long* best;
};
hipError_t launch_beam_select(const BeamCall& c, hipStream_t s);

}  // namespace mlq
