// Checks of the matrices that the token-layer entries take.
#include "device_matrix.cuh"

namespace bou {

int validate_matrix(const BulletOuB200Matrix* m, unsigned types, const char* name) {
    if (m == nullptr) return fail_messagef("%s must not be null", name);
    if (m->type < 0 || m->type > BULLETOU_B200_TYPE_I32 || !(types >> m->type & 1u))
        return fail_messagef("%s has type %d, which this entry does not take", name, m->type);
    // (so that the kernels' 32-bit indexes may run past an extent by a CTA's work)
    constexpr size_t kMost = (static_cast<size_t>(1) << 31) - (static_cast<size_t>(1) << 16);
    if (m->rows > kMost || m->cols > kMost)
        return fail_messagef("%s is too large (%zu x %zu)", name, m->rows, m->cols);
    if (m->rows == 0 || m->cols == 0) return 0;
    if (m->data == nullptr) return fail_messagef("%s data must not be null", name);
    const size_t bytes = type_bytes(m->type);
    if (reinterpret_cast<uintptr_t>(m->data) % bytes != 0)
        return fail_messagef("%s data is not aligned to its %zu-byte elements", name, bytes);
    if (m->rows > 1) {
        if (m->row_stride < m->cols)
            return fail_messagef("%s row stride %zu is smaller than its %zu columns", name, m->row_stride, m->cols);
        if (m->row_stride > static_cast<size_t>(INT64_MAX) / bytes / m->rows)
            return fail_messagef("%s row stride %zu is too large", name, m->row_stride);
    }
    return 0;
}

int validate_matrix(const BulletOuB200Matrix* m, unsigned types, size_t rows, size_t cols, const char* name) {
    if (validate_matrix(m, types, name) != 0) return -1;
    if (m->rows != rows || m->cols != cols)
        return fail_messagef("%s is %zu x %zu, expected %zu x %zu", name, m->rows, m->cols, rows, cols);
    return 0;
}

int validate_disjoint(const BulletOuB200Matrix* out, const char* out_name, const BulletOuB200Matrix* in,
                      const char* in_name, bool same_ok) {
    if (out == nullptr || in == nullptr || out->rows * out->cols == 0 || in->rows * in->cols == 0) return 0;
    auto begin = [](const BulletOuB200Matrix* m) { return reinterpret_cast<uintptr_t>(m->data); };
    auto end = [&](const BulletOuB200Matrix* m) {
        return begin(m) + ((m->rows - 1) * (m->rows > 1 ? m->row_stride : 0) + m->cols) * type_bytes(m->type);
    };
    if (begin(out) >= end(in) || begin(in) >= end(out)) return 0;
    // columns of one wider matrix: rows of the same distance that interleave
    const size_t pitch = out->row_stride * type_bytes(out->type);
    if (out->rows > 1 && in->rows > 1 && pitch == in->row_stride * type_bytes(in->type)) {
        const size_t out_bytes = out->cols * type_bytes(out->type), in_bytes = in->cols * type_bytes(in->type);
        const size_t shift = begin(out) >= begin(in) ? (begin(out) - begin(in)) % pitch
                                                     : (pitch - (begin(in) - begin(out)) % pitch) % pitch;
        if (shift >= in_bytes && shift + out_bytes <= pitch) return 0;
    }
    if (same_ok && out->data == in->data && out->type == in->type &&
        (out->rows == 1 || out->row_stride == in->row_stride))
        return 0;
    return fail_messagef("%s must not overlap %s", out_name, in_name);
}

}  // namespace bou
