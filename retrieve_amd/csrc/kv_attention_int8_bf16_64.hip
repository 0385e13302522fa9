// bf16 attention over 8-bit pages of 64 and 128 slots (kv_attend_int8.h).
#include "kv_attend_int8.h"

int rt::attend_int8_bf16_64(int64_t D, const AttendInt8Args& a, const AttendInt8Plan& p,
                            hipStream_t s) {
  return a.tok.shift == 6 ? attend_int8_dims<__bf16, 6>(D, a, p, s)
                          : attend_int8_dims<__bf16, 7>(D, a, p, s);
}
