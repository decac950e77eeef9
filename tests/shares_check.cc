/* Checks csrc/shares.h against 128-bit arithmetic and against a walk over the shares; prints the number of mismatches. */
#include <stdio.h>

#include "shares.h"

using asterq::share_of;
using asterq::shares_up_to;
typedef unsigned long long u64;

static u64 state = 88172645463325252ull;
static u64 next() {
  state ^= state << 13;
  state ^= state >> 7;
  state ^= state << 17;
  return state;
}
// of up to `bits` bits, the length even
static long long value(int bits) { return (long long)(next() >> (64 - 1 - next() % bits)) + 1; }

int main() {
  long long bad = 0;
  for (int i = 0; i < 4000000; ++i) {
    const int n = 1 + (int)(next() % 256);
    const long long a = value(52) - 1, d = value(i & 1 ? 52 : 33);
    if (share_of(a, n, d) != (long long)((__int128)a * n / d)) ++bad;
    const long long total = value(52);
    long long end = i & 2 ? value(24) : value(52);
    if (end > total) end = 1 + end % total;
    const int got = shares_up_to(end, n, total, 0) - 1;
    // the share that has end - 1
    const long long from = (long long)((__int128)total * got / n), to = (long long)((__int128)total * (got + 1) / n);
    if (got < 0 || got >= n || !(from <= end - 1 && end - 1 < to)) ++bad;
    if (shares_up_to(end, n, total, got) != 1) ++bad;
  }
  // units of a few tiles at the front of 2^32 tiles and around
  for (long long total = (1ll << 31) - 3; total <= (1ll << 33); total += (1ll << 30) - 1)
    for (int n = 1; n <= 256; n += 51)
      for (long long end = 1; end < (1 << 23); end = end * 3 + 1)
        if (shares_up_to(end, n, total, 0) - 1 != (int)((__int128)(end * n - 1) / total)) ++bad;
  printf("%lld\n", bad);
  return 0;
}
