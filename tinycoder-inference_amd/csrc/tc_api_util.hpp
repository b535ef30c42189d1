// tc_api_util.hpp -- argument checks that the entry points around attention share.
#pragma once

#include <string>

#include "tc_attention.h"
#include "tc_attn_common.hpp"
#include "tc_kernels.hpp"
#include "tc_qmatmul.h"

namespace tc {
namespace api {

inline int refuse(int code, const std::string &msg) { return tc::fail_code(code, msg.c_str()); }

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline int no_device() { return refuse(TC_E_UNSUPPORTED, "no gfx950 device"); }
inline bool row_type(int t) { return t == TC_F32 || t == TC_F16 || t == TC_BF16; }

// Cache and batch of a call checked and put together. Nothing of the batch's
// arrays is read here: they are the device's.
int kv_args(const tc_kv_cache *c, const tc_kv_batch *b, int xtype, tc::KvArgs *a);
// Rows of `width` elements of xtype at a stride.
int check_rows(const char *name, const void *p, uint32_t stride, uint64_t width, uint32_t n, int xtype);

inline int hip_rc(hipError_t e, const char *what) {
    if (e == hipSuccess) return TC_OK;
    return refuse(TC_E_LAUNCH, std::string(what) + ": " + hipGetErrorString(e));
}

}  // namespace api
}  // namespace tc
