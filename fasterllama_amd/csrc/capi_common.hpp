// Host helpers shared by the C-ABI source files: error capture, argument import and validation, kernel launches.
#pragma once

#include <hip/hip_runtime.h>

#include <atomic>
#include <cmath>
#include <cstddef>
#include <cstdint>
#include <cstring>

#include "../../include/fl_decode_attn.h"

namespace flhost {

inline thread_local int g_last_hip_error = 0;

constexpr int kMaxSplits = 1024;

inline bool check_hip(hipError_t e)
{
    if (e != hipSuccess) {
        g_last_hip_error = (int)e;
        return false;
    }
    return true;
}

// Compute units of the current device.  The only thing the library remembers between calls: an
// immutable property of the hardware, cached per device id (256 when no device can be queried).
inline int device_cus()
{
    static std::atomic<int> cached[64];
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess || dev < 0 || dev >= 64) return 256;
    int n = cached[dev].load(std::memory_order_relaxed);
    if (n == 0) {
        if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0)
            n = 256;
        cached[dev].store(n, std::memory_order_relaxed);
    }
    return n;
}

inline bool head_dim_ok(int D)
{
    // the reference's set: the multiples of 32 up to 128 (decoder_kernels.cu:564-571, :640, :960) and 256, 512, 1024
    return D == 32 || D == 64 || D == 96 || D == 128 || D == 256 || D == 512 || D == 1024;
}

// The caller's struct, struct_size bytes of it, copied into a zeroed struct of this build: members the caller's
// header did not have yet read as zero / NULL.  MIN is the size of the first layout that carried struct_size.
constexpr size_t kDescMinBytes = offsetof(fl_attn_desc, flags) + sizeof(int32_t);
constexpr size_t kIoMinBytes = offsetof(fl_attn_io, mask_tile_classes) + sizeof(void *);

template <typename S>
int import_struct(const S *in, S *out, size_t min_bytes)
{
    if (!in) return FL_ATTN_ERR_NULL_POINTER;
    uint32_t n;
    std::memcpy(&n, in, sizeof n); // struct_size is the first member of both structs
    if (n < min_bytes || n > sizeof(S)) return FL_ATTN_ERR_STRUCT_SIZE;
    std::memset(static_cast<void *>(out), 0, sizeof(S));
    std::memcpy(static_cast<void *>(out), in, n);
    return FL_ATTN_OK;
}

inline int validate_desc(const fl_attn_desc *d)
{
    if (d->dtype != FL_ATTN_F32 && d->dtype != FL_ATTN_F16) return FL_ATTN_ERR_DTYPE;
    if (d->batch_size <= 0 || d->head_num <= 0 || d->total_len <= 0) return FL_ATTN_ERR_SHAPE;
    if (d->batch_size > 65535 || d->head_num > 65535) return FL_ATTN_ERR_SHAPE;
    if (!head_dim_ok(d->size_per_head)) return FL_ATTN_ERR_HEAD_DIM;
    if (d->nsplit < 0 || d->nsplit > kMaxSplits || (d->flags & ~FL_ATTN_FLAG_FAST_PROMPT_QK) != 0) return FL_ATTN_ERR_ARGUMENT;
    if (!(d->softmax_scale >= 0.f) || std::isinf(d->softmax_scale)) return FL_ATTN_ERR_ARGUMENT;
    // Row offsets inside one (b,h) slice of a cache are 32-bit byte offsets in the kernels, and the buffer descriptors
    // of the streaming kernel span 2^31 bytes from the slice's base: a slice stays below that, with room for the whole
    // tiles the prompt-phase kernels address past the last row (up to 63 rows, which fail the range check and read as
    // zeros).
    if (((int64_t)d->total_len + 64) * d->size_per_head * (d->dtype == FL_ATTN_F16 ? 2 : 4) >= ((int64_t)1 << 31)) return FL_ATTN_ERR_SHAPE;
    // the streaming grid is one-dimensional: B*H*splits workgroups must fit the 2^31 limit
    if ((int64_t)d->batch_size * d->head_num > (int64_t)INT32_MAX / kMaxSplits) return FL_ATTN_ERR_SHAPE;
    return FL_ATTN_OK;
}

// Every entry point works on its own copy of the caller's descriptor (see import_struct).
inline int import_desc(const fl_attn_desc **desc, fl_attn_desc *copy)
{
    const int st = import_struct(*desc, copy, kDescMinBytes);
    if (st != FL_ATTN_OK) return st;
    *desc = copy;
    return validate_desc(copy);
}

inline size_t align_up(size_t x, size_t a) { return (x + a - 1) / a * a; }

// Row stride of the persistent mask tile class table: the 32-row blocks of one key tile, padded to whole words.
inline size_t class_table_ld(int total_len) { return align_up(((size_t)total_len + 31) / 32, 4); }

// Kernel launch that reports its own status: hipLaunchKernel returns the error of this launch,
// whereas hipGetLastError would also return (and clear) an error left behind by an earlier,
// unrelated HIP call of the calling thread.
template <typename T> struct same_type { typedef T type; };
template <typename... KArgs>
inline hipError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, hipStream_t stream, typename same_type<KArgs>::type... args)
{
    void *ptrs[] = {const_cast<void *>(static_cast<const void *>(&args))...};
    return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, block, ptrs, 0, stream);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

} // namespace flhost
