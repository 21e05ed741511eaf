// Gate activations of the gated Dense layer (zn_gate of the C ABI): the four
// epilogue activations as the GEMMs apply them, SiLU and the tanh form of
// GELU.  One definition, so every kernel that applies a gate rounds alike.
#ifndef ZN_GATE_H
#define ZN_GATE_H

#include <hip/hip_runtime.h>

constexpr float kGeluA = 0.79788456080286535588f;  // sqrt(2 / pi)
constexpr float kGeluB = 0.044715f;

__device__ __forceinline__ float zn_gate(float g, int act) {
    switch (act) {
    case 1: return g > 0.0f ? g : 0.0f;
    case 2: return 1.0f / (1.0f + expf(-g));
    case 3: return tanhf(g);
    case 4: return g / (1.0f + expf(-g));
    case 5: return 0.5f * g * (1.0f + tanhf(kGeluA * (g + kGeluB * g * g * g)));
    default: return g;
    }
}

// s = sigmoid(g) and c = 1 - s, each to its own relative precision.
__device__ __forceinline__ void zn_sigmoid_pair(float g, float &s, float &c) {
    const float e = expf(-__builtin_fabsf(g)), r = 1.0f / (1.0f + e);
    s = g >= 0.0f ? r : e * r;
    c = g >= 0.0f ? e * r : r;
}

// y = act(g) and its derivative d.
__device__ __forceinline__ void zn_gate_slope(float g, int act, float &y, float &d) {
    switch (act) {
    case 1:
        y = g > 0.0f ? g : 0.0f;
        d = g > 0.0f ? 1.0f : 0.0f;
        return;
    case 2: {
        float c;
        zn_sigmoid_pair(g, y, c);
        d = y * c;
        return;
    }
    case 3:
        y = tanhf(g);
        d = 1.0f - y * y;
        return;
    case 4: {
        float s, c;
        zn_sigmoid_pair(g, s, c);
        y = g * s;
        d = s * (1.0f + g * c);
        return;
    }
    case 5: {
        const float t = tanhf(kGeluA * (g + kGeluB * g * g * g));
        y = 0.5f * g * (1.0f + t);
        d = 0.5f * (1.0f + t);
        // past 10 the tanh is 1 to the last bit and the next term 0; its g * g may overflow
        if (__builtin_fabsf(g) < 10.0f) d += 0.5f * g * (1.0f - t * t) * (kGeluA * (1.0f + 3.0f * kGeluB * g * g));
        return;
    }
    default:
        y = g;
        d = 1.0f;
    }
}

#endif
