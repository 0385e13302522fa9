// Appending f16 heads of up to 128 channels to the 8-bit paged cache (kv_append_int8.h).
#include "kv_append_int8.h"

int rt::append_int8_f16_128(int64_t D, const WriteArgs& a, unsigned grid, unsigned lds,
                         bool interleaved, hipStream_t s) {
  switch (D) {
    case 64: return append_int8_launch<_Float16, 64>(a, grid, lds, interleaved, s);
    case 96: return append_int8_launch<_Float16, 96>(a, grid, lds, interleaved, s);
    default: return append_int8_launch<_Float16, 128>(a, grid, lds, interleaved, s);
  }
}
