// What the two forms of the decayed attention's chain share: its streams, its arguments and its plan.
#pragma once

#include "ews_token.cuh"

namespace ews {
namespace decay {

using namespace token;

// One stream (batch, steps, heads, width): element strides, and the query heads that share one of its heads.
template <typename T>
struct Stream {
    const T* p;
    long sb, st, sh;
    int group, width, vec;
};

template <typename T>
struct Chain {
    Stream<T> x, y, z;
    T* out;          // (batch, steps, heads, dz), or
    float* out32;    // the same in float32 (shared heads: summed afterwards)
    const float* rate;
    const int* lengths;
    const float* init;  // state the chain starts from (may be null); element (i, j) of a head at i * init_r + j * init_c
    float* fin;         // state it ends with (may be null)
    long init_r, init_c, fin_r, fin_c;
    float oscale, init_scale, fin_scale;
    float* seg;      // (batch * heads, segments, dx, dz): the segments' own states, then their starting states
    int batch, steps, heads, rev;
    int segs, span, slices;  // segments of `span` tokens
    int down;                // the chain takes the segments from the last to the first
    int* status;
};

// The tensor-core form (bfloat16, 16-byte-aligned streams): ews_decay_tc.cu. Segments are counted from the axis's
// start whichever way the chain runs.
int tc_segments(int batch, int steps, int heads, bool state, int* span);
bool tc_fits(const Chain<bf16>& a);
int tc_chain(const Chain<bf16>& a, bool state_only, bool exact, cudaStream_t s);

// The same for float32 in three bfloat16 planes (x and y up to F32_WIDE wide; any alignment, any length, none included):
// ews_decay_f32.cu.
constexpr int F32_WIDE = 64;
bool f32_fits(const Chain<float>& a);
int f32_chain(const Chain<float>& a, bool state_only, cudaStream_t s);

}  // namespace decay
}  // namespace ews
