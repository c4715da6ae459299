// What the C ABI's files share: error messages, sizes and the checks that outputs stand apart (internal to libsubq_b200).
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>
#include <string>

#include "kernels.hpp"
#include "overlap.h"

namespace subq {
namespace capi {

// (capi.cu) The calling thread's last error, which the functions return with its code; the last call's kernel launches.
int fail(int code, const std::string& msg);
int fail_cuda(cudaError_t err, const char* where);
void set_launches(int n);

inline size_t elem_size(int dtype) { return dtype == SUBQ_FP64 ? 8 : dtype == SUBQ_FP32 ? 4 : 2; }

constexpr size_t kAlign = 256;
inline size_t align_up(size_t x) { return (x + kAlign - 1) / kAlign * kAlign; }

inline int check_workspace(void* ws, size_t have, size_t need) {
    if (need == 0) return SUBQ_OK;
    if (!ws) return fail(SUBQ_ERR_WORKSPACE, "workspace required: " + std::to_string(need) + " bytes");
    if (have < need)
        return fail(SUBQ_ERR_WORKSPACE, "workspace too small: need " + std::to_string(need) +
                                            " bytes, got " + std::to_string(have));
    if (reinterpret_cast<uintptr_t>(ws) % kAlign != 0)
        return fail(SUBQ_ERR_WORKSPACE, "workspace must be 256-byte aligned");
    return SUBQ_OK;
}

struct Memory {
    const char* name;
    MemRows rows;
};
inline Memory of_bytes(const char* name, const void* at, int64_t bytes) { return {name, {reinterpret_cast<uintptr_t>(at), bytes}}; }

// An output's rows must be apart, from one another and from every input's and other output's.
inline int check_apart(std::initializer_list<Memory> out_list, std::initializer_list<Memory> in_list) {
    const Memory *outs = out_list.begin(), *ins = in_list.begin();
    const int no = (int)out_list.size(), ni = (int)in_list.size();
    for (int i = 0; i < no; ++i) {
        if (rows_overlap_themselves(outs[i].rows))
            return fail(SUBQ_ERR_INVALID_ARGUMENT, std::string("rows of ") + outs[i].name + " overlap");
        for (int j = 0; j < ni + i; ++j) {
            const Memory& other = j < ni ? ins[j] : outs[j - ni];
            if (rows_overlap(outs[i].rows, other.rows))
                return fail(SUBQ_ERR_ALIAS, std::string(outs[i].name) + " shares memory with " + other.name);
        }
    }
    return SUBQ_OK;
}

}  // namespace capi
}  // namespace subq
