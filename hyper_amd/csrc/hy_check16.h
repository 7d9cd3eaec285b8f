// Argument checks that the C entries of the 16-bit calls share.
#pragma once
#include "hy_internal.h"

namespace hy {

inline bool type16(int t) { return t == HY_F16 || t == HY_BF16; }
inline bool misaligned(const void *p, size_t a) { return ((uintptr_t) p & (a - 1)) != 0; }

// a matrix of `rows` x `cols` elements of `bytes` each whose rows lie `ld` elements apart; out: written
inline int check_mat(const char *what, const char *name, const void *p, int64_t ld, int rows, int cols, int bytes, bool out) {
    if (!rows) return HY_OK;   // an empty matrix may have no address
    if (!p) { set_error("%s: %s is null", what, name); return HY_EINVAL; }
    if (misaligned(p, bytes)) { set_error("%s: %s is not aligned to its %d-byte values", what, name, bytes); return HY_EBAD_SHAPE; }
    if (ld < 0 || (out && rows > 1 && ld < cols)) { set_error("%s: %lld elements between the rows of %s (%d values)", what, (long long) ld, name, cols); return HY_EBAD_SHAPE; }
    return HY_OK;
}
inline int check_sizes(const char *what, int type, int m, int n, int k) {
    if (!type16(type)) { set_error("%s: type %d (HY_F16 or HY_BF16)", what, type); return HY_EUNSUPPORTED_TYPE; }
    if (m < 0) { set_error("%s: %d rows", what, m); return HY_EINVAL; }
    if (n <= 0 || k <= 0 || n > HY_MM_MAX || k > HY_MM_MAX || m > HY_MM_MAX) { set_error("%s: m %d, n %d, k %d (1 .. 2^30)", what, m, n, k); return HY_EBAD_SHAPE; }
    return HY_OK;
}
inline int check_out_type(const char *what, int type, int out_type) {
    if (out_type != HY_F32 && out_type != type) { set_error("%s: output type %d (HY_F32 or the operands' type)", what, out_type); return HY_EUNSUPPORTED_TYPE; }
    return HY_OK;
}
// eight neighbouring values at columns that are multiples of 8 start on 16 bytes
inline bool vec16(const void *p, int64_t ld, int bytes) { return !p || (ld % (16 / bytes) == 0 && !misaligned(p, 16)); }

#define HY_TRY(e) do { const int rc_ = (e); if (rc_ != HY_OK) return rc_; } while (0)

} // namespace hy
