// Checks of rows of values that the *_device calls share (element types: rk_npu_mx4.h).
#ifndef RK_VALUES_H
#define RK_VALUES_H

#include "rk_npu_mx4.h"
#include "rk_rows.h"

namespace rkhost {

inline bool valid_type(int type) { return type >= RK_NPU_MX4_F32 && type <= RK_NPU_MX4_BF16; }
inline int64_t type_bytes(int type) { return type == RK_NPU_MX4_F32 ? 4 : 2; }
inline bool valid_length(int K) { return K > 0 && K <= INT32_MAX / 1024; }

inline Span values(const void* p, int type, int64_t rows, int64_t ld, int64_t width) {
    return Span(p, rows, ld * type_bytes(type), width * type_bytes(type));
}
// Pointer and stride of rows of values: aligned to the type, no row on the next one, and all of it addressable.
inline bool valid_rows(const void* p, int type, int64_t rows, int64_t ld, int64_t width) {
    if (rows == 0) return valid_type(type); // (an empty tensor may have no address)
    return valid_type(type) && p && reinterpret_cast<uintptr_t>(p) % type_bytes(type) == 0 && ld >= width && ld <= (INT64_C(1) << 40) &&
           ld <= (INT64_C(1) << 56) / rows;
}

} // namespace rkhost

#endif // RK_VALUES_H
