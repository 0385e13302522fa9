// f16 attention over 8-bit pages of 16 and 32 slots (kv_attend_int8.h).
#include "kv_attend_int8.h"

int rt::attend_int8_f16_16(int64_t D, const AttendInt8Args& a, const AttendInt8Plan& p,
                           hipStream_t s) {
  return a.tok.shift == 4 ? attend_int8_dims<_Float16, 4>(D, a, p, s)
                          : attend_int8_dims<_Float16, 5>(D, a, p, s);
}
