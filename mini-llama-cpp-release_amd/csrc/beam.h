// Beam selection (beam.hip): what its launch takes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstddef>
#include <cstdint>

namespace mlq {

constexpr int kBeamMostBeams = 64;  // of a group
constexpr int kBeamMostKeep = 64;
constexpr int kBeamPart = 8192;     // logits of a part of a row
constexpr int kBeamSmallPart = 2048;

// Logits of a part: small ones where the rows are too few for a workgroup a CU.
inline int beam_part(long long rows, int vocab) {
    return rows * ((vocab + kBeamPart - 1) / kBeamPart) < 256 ? kBeamSmallPart : kBeamPart;
}
// Parts of as many rows at the most.
inline size_t beam_parts(long long rows, int vocab) {
    const size_t large = static_cast<size_t>(rows) * ((vocab + kBeamPart - 1) / kBeamPart);
    // (fewer rows or tokens may be cut finer: below 256 large parts, four of each)
    return large > 1024 ? large : 1024;
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
