/* r3d_operands.h -- what the plans of the second table's rows ask of an operand's shape and strides. */
#ifndef R3D_OPERANDS_H
#define R3D_OPERANDS_H

#include <stdint.h>
#include "rad_abi.h"
#include "rad_plugin.h"

namespace r3d {

static const int64_t kDimMax = 0x7FFFFFFLL;

inline bool pitch_ok(int64_t p) { return p >= 0 && p <= (int64_t(1) << 40); }

/* One f32 a row: rank 1 [rows], or rank 2 [rows, 1]; the stride may be 0 (one scale for all). */
inline int scale_column(const RadTensor* t, int64_t rows, int64_t* stride) {
    if (t->dtype != RAD_F32) return RAD_E_UNSUPPORTED;
    if ((t->rank != 1 && t->rank != 2) || (t->rank == 2 && t->shape[1] != 1)) return RAD_E_SHAPE;
    if (t->shape[0] < rows) return RAD_E_SHAPE;
    *stride = t->stride[0];
    return pitch_ok(*stride) ? RAD_OK : RAD_E_STRIDE;
}

/* The pitch of a [rows, cols] operand whose rows lie anywhere: rank 2 with its own row stride,
 * or higher ranks whose outer axes are dense; rank 1 is one row. */
inline int rows_of(const RadTensor* t, int64_t rows, int64_t cols, int64_t* pitch) {
    const long long n = rad_tensor_numel(t);
    if (n < 0 || rows > INT64_MAX / cols || n < rows * cols) return RAD_E_SHAPE;
    if (t->rank == 1) {
        if (rows != 1 || n != cols) return RAD_E_SHAPE;
        if (t->stride[0] != 1) return RAD_E_STRIDE;
        *pitch = cols;
        return RAD_OK;
    }
    if (t->rank < 2 || t->shape[t->rank - 1] != cols) return RAD_E_SHAPE;
    if (t->stride[t->rank - 1] != 1) return RAD_E_STRIDE;
    for (int i = 0; i + 2 < (int)t->rank; ++i) {
        int64_t span = 0;
        if (__builtin_mul_overflow(t->shape[i + 1], t->stride[i + 1], &span) || t->stride[i] != span)
            return RAD_E_STRIDE;
    }
    *pitch = t->stride[t->rank - 2];
    return pitch_ok(*pitch) ? RAD_OK : RAD_E_STRIDE;
}

/* Bytes of an element of the types that these rows move; 0 for another. */
inline int elt_bytes(uint32_t dtype) {
    switch (dtype) {
        case RAD_F32: case RAD_I32: return 4;
        case RAD_BF16: return 2;
        case RAD_I8: case RAD_U8: case RAD_F8E4M3: case RAD_E8M0: return 1;
        default: return 0;
    }
}

/* Whether an element lies off its own size. */
inline bool misaligned(const RadTensor* t) {
    const int b = t ? elt_bytes(t->dtype) : 0;
    return b > 1 && ((uintptr_t)t->data & (uintptr_t)(b - 1));
}

/* Rows as they lie in memory, pitch in elements. */
struct Span {
    const void* data;
    int64_t rows, cols, pitch;
    int size;                /* bytes an element */
};

/* Whether two operands' rows have an element's memory in common.  Column ranges of rows that lie a common
 * pitch apart are told from each other; of other pairs it is enough that what they span overlaps. */
inline bool spans_meet(const Span& u, const Span& v) {
    const uintptr_t a = (uintptr_t)u.data, b = (uintptr_t)v.data;
    const uintptr_t ae = a + (uintptr_t)(((u.rows - 1) * u.pitch + u.cols) * u.size);
    const uintptr_t be = b + (uintptr_t)(((v.rows - 1) * v.pitch + v.cols) * v.size);
    if (ae <= b || be <= a) return false;
    const uintptr_t p = (uintptr_t)u.pitch * (uintptr_t)u.size;
    if (u.rows == 1 || v.rows == 1 || !p || p != (uintptr_t)v.pitch * (uintptr_t)v.size) return true;
    const uintptr_t d = b >= a ? (b - a) % p : (p - (a - b) % p) % p;   /* where in u's row v's begins */
    return d < (uintptr_t)u.cols * (uintptr_t)u.size || d + (uintptr_t)v.cols * (uintptr_t)v.size > p;
}

/* Whether an output's memory overlaps an input's other than by being the same elements at the same places,
 * which is no harm where a lane reads its elements before it writes them. */
inline bool spans_clash(const Span& out, const Span& in) {
    const bool same = out.data == in.data && out.size == in.size && out.cols == in.cols &&
                      (out.pitch == in.pitch || (out.rows == 1 && in.rows == 1));
    return !same && spans_meet(out, in);
}

}  // namespace r3d

#endif /* R3D_OPERANDS_H */
