// paged_check.h -- argument checks that every paged entry point makes.
#pragma once

#include "../../include/b200_paged.h"
#include "host_util.h"

namespace b200 {

inline int check_paged_kv(const b200_paged_kv* kv) {
    if (!kv || !kv->k || !kv->v || kv->n_head_kv <= 0 || kv->page_size <= 0 || kv->n_pages <= 0 ||
        kv->n_pages >= INT32_MAX / kv->page_size)
        return B200_EINVAL;
    if (kv->type != B200_TYPE_F16 && kv->type != B200_TYPE_BF16) return B200_EUNSUPPORTED;
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return B200_EUNSUPPORTED;
    const int64_t strides = kv->k_page | kv->k_row | kv->k_head | kv->v_page | kv->v_row | kv->v_head;
    if (!aligned16(kv->k) || !aligned16(kv->v) || (strides & 15) || strides < 0) return B200_EINVAL;
    // the last byte of K and of V: offsets are counted in 16-byte steps in 32 bits.
    // Each term is compared by division first, so the sums cannot wrap around
    const int64_t span = (int64_t)1 << 36;
    const int64_t last[3] = {kv->n_pages - 1, kv->page_size - 1, kv->n_head_kv - 1};
    const int64_t steps[2][3] = {{kv->k_page, kv->k_row, kv->k_head}, {kv->v_page, kv->v_row, kv->v_head}};
    for (const auto& step : steps) {
        int64_t end = 0;
        for (int i = 0; i < 3; ++i) {
            if (step[i] >= span || (step[i] > 0 && last[i] > span / step[i])) return B200_EUNSUPPORTED;
            end += last[i] * step[i];
        }
        if (end >= span) return B200_EUNSUPPORTED;
    }
    if ((kv->k_lo == nullptr) != (kv->k_hi == nullptr) || !aligned16(kv->k_lo) || !aligned16(kv->k_hi))
        return B200_EINVAL;
    return B200_OK;
}

// Whether `size` bytes at out meet one of n rows of `row` bytes, `stride` bytes
// apart from q on.
inline bool meets_rows(const void* out, int64_t size, const void* q, int64_t stride, int64_t row, int64_t n) {
    const int64_t ahead = reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(q);
    // the first row that ends behind out's first byte
    const int64_t s = ahead < row ? 0 : n == 1 || stride == 0 ? n : (ahead - row) / stride + 1;
    return s < n && s * stride < ahead + size;
}

}  // namespace b200
