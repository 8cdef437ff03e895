// What the files of the C ABI share: error text, notes, the workspace object.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

struct vfkv_workspace {
    uint32_t n_heads, head_dim, max_tiles;
    int device;            // where the scratch is
    float* scratch_out;
    float* scratch_max;
    float* scratch_sum;
    float* q_rot;          // n_heads * head_dim floats: rotated queries of vfkv_qk_rope_kv_write_decode_attention when the caller
                           // does not want them and the shape takes the separate RoPE launch
};

namespace vfkv {

int fail(int status, const char* fmt, ...) __attribute__((format(printf, 2, 3)));   // sets the thread's error text, returns status
int hip_fail(hipError_t e, const char* what);
void clear_note();
void set_note(const char* fmt, ...) __attribute__((format(printf, 1, 2)));           // the thread's advisory (vfkv_last_note)

}  // namespace vfkv
