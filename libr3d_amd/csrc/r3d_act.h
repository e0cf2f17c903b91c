/* r3d_act.h -- activations in f32, by the names that the rows know them by. */
#ifndef R3D_ACT_H
#define R3D_ACT_H

#include <string.h>

namespace r3d {

enum { ACT_NONE = 0, ACT_RELU, ACT_SILU, ACT_SIGMOID, ACT_GELU, ACT_GELU_TANH, ACT_COUNT };

/* The activation that a name stands for; -1 for another name. */
inline int act_by_name(const char* s) {
    static const char* const kNames[ACT_COUNT] = {"none", "relu", "silu", "sigmoid", "gelu", "gelu_tanh"};
    for (int i = 0; i < ACT_COUNT; ++i)
        if (!strcmp(s, kNames[i])) return i;
    return -1;
}

}  // namespace r3d

#endif /* R3D_ACT_H */
