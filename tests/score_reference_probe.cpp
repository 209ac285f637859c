// C entries over csrc/score_reference.cuh, built for the host by tests/test_score_reference.py.
#include "../int8-transformer-kernels_b200/csrc/score_reference.cuh"

using i8tk::ScoreReference;

// state: {nm, rest, far}
static ScoreReference load(const float* state) {
    ScoreReference r;
    r.nm = state[0], r.rest = state[1], r.far = state[2] != 0.f;
    return r;
}
extern "C" float probe_exponent(const float* state, float y, float q, float lift) { return load(state).exponent(y, q, lift); }
extern "C" float probe_move(float* state, float y, float q, float lift) {
    ScoreReference r = load(state);
    const float change = r.move_to(y, q, lift);
    state[0] = r.nm, state[1] = r.rest, state[2] = r.far ? 1.f : 0.f;
    return change;
}
extern "C" float probe_negative_reference(float mx, float at) { return i8tk::negative_reference(mx, at); }
