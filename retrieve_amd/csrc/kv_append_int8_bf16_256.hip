// Appending bf16 heads of more than 128 channels to the 8-bit paged cache (kv_append_int8.h).
#include "kv_append_int8.h"

int rt::append_int8_bf16_256(int64_t D, const WriteArgs& a, unsigned grid, unsigned lds,
                         bool interleaved, hipStream_t s) {
  switch (D) {
    case 192: return append_int8_launch<__bf16, 192>(a, grid, lds, interleaved, s);
    default: return append_int8_launch<__bf16, 256>(a, grid, lds, interleaved, s);
  }
}
