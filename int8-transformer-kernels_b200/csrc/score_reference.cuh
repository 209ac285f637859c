// The value that a softmax row's scores are taken against, in fp32, for scores of any finite size.
//
// A probability is 2^(y * q - reference) for a score y * q in log2 units.  fp32 steps reach 1/2 at 2^23 and 32 at 2^28, so
// from there on a reference that is one fp32 number lies a step's fraction away from the score it was made from: above it
// the largest probability is lost, below it the products leave the range of fp16, and moving the reference by a
// difference smaller than half a step does not move it at all.  Below kFarScore that offset is at most 1/4, the same
// for the whole row, and cancels.  From kFarScore on the reference is kept as the rounded product and the product's
// remainder, which a fused multiply-add gives exactly; the largest score then comes out where it belongs.
//
// Plain C++ on the host as well: tests run this arithmetic on the CPU.
#pragma once

#include <cmath>

#ifdef __CUDACC__
#define I8TK_HD __host__ __device__ __forceinline__
#else
#define I8TK_HD inline
#endif

namespace i8tk {

constexpr float kFarScore = 4194304.0f;          // 2^22
constexpr float kMostScore = 8.507059173e37f;    // 2^126

// The exponent of a probability is  fma(y, q, nm)  for a near reference, to which `lift` (what the row's probabilities are
// raised by, log2 units) has been added, and  fma(y, q, nm) + rest + lift  for a far one.
struct ScoreReference {
    float nm;
    float rest;
    bool far;

    I8TK_HD float base(float lift) const { return far ? lift : 0.f; }
    I8TK_HD float exponent(float y, float q, float lift) const { return fmaf(y, q, nm) + rest + base(lift); }
    // From here on the score y * q has the exponent `lift`.  Returns what the exponents of the other scores change by.
    // A score beyond kMostScore makes the row NaN.
    I8TK_HD float move_to(float y, float q, float lift) {
        const ScoreReference old = *this;
        const float score = y * q;
        if (!(fabsf(score) <= kMostScore)) {
            nm = NAN;
            rest = 0.f;
            far = false;
            return nm;
        }
        far = fabsf(score) >= kFarScore;
        nm = far ? -score : lift - score;
        rest = far ? -fmaf(y, q, -score) : 0.f;
        return (nm - old.nm) + (rest - old.rest) + (base(lift) - old.base(lift));
    }
};

// The same for scores that are rounded to fp32 before they meet the reference: what to add to them so that the score mx
// comes out at `at`; at 0 where the sum would be rounded by much.
I8TK_HD float negative_reference(float mx, float at) { return fabsf(mx) < kFarScore ? at - mx : -mx; }

}  // namespace i8tk
