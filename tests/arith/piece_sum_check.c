/* last_piece_sum / is_last_piece / piece_sum: every denominator a piece may have (zero, subnormals, every binade, the
   largest) comes back bit for bit, marked as the last piece's, and is not marked when it is stored as it is. */
#include <stdint.h>
#include <stdio.h>
#include <string.h>

#include "../../int8-kvcache_amd/csrc/piece_sum.h"

int main(void) {
  long bad = 0, n = 0;
  for (uint64_t b = 0; b <= 0x7f7fffffu; b += b < 64 ? 1 : 997) {
    const uint32_t w = (uint32_t)b;
    float l, back;
    memcpy(&l, &w, 4);
    const float s = last_piece_sum(l);
    back = piece_sum(s);
    bad += memcmp(&back, &l, 4) != 0;
    back = piece_sum(l);
    bad += memcmp(&back, &l, 4) != 0;
    bad += !is_last_piece(s) || is_last_piece(l);
    ++n;
  }
  bad += !is_last_piece(-1.f);   /* the mark of a row that was not cut */
  printf("checked %ld mismatched %ld\n", n, bad);
  return bad != 0;
}
