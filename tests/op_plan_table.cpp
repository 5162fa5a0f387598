// What the operators' launch shapes are at given sizes (vtc_amd/csrc/op_plan.h).  One question per line of standard input, one line of
// answer each:
//   gate M K F save | rows M N K | dgate M N F | weights M K F N   ->  "small" or "wide", tiles, K splits, blocks launched
//   rotary tokens pieces_per_token table                           ->  tokens per block, blocks
#include <cstdio>
#include <cstring>

#include "op_plan.h"

using namespace vtc;

static long long up8(long long n) { return (n + 7) / 8 * 8; }
static long long cover(long long a, long long b) { return (a + b - 1) / b; }
static void answer(const OgPlan& p, long long wide, long long small) {
  const long long tiles = p.small ? small : wide, units = tiles * p.splits;
  printf("%s %lld %d %lld\n", p.small ? "small" : "wide", tiles, p.splits, p.small ? units : (units < 256 ? units : 256));
}

int main() {
  char kind[16];
  long long a, b, c, d;
  while (scanf("%15s %lld %lld %lld", kind, &a, &b, &c) == 4) {
    if (!strcmp(kind, "rotary")) {
      const long long n = rotary_tokens_per_block(a, b, c);
      printf("%lld %lld\n", n, cover(a, n));
      continue;
    }
    if (!strcmp(kind, "gate")) {
      if (scanf("%lld", &d) != 1) return 1;
      answer(plan_gate(a, (int)b, (int)up8(c), d != 0), cover(a, 256) * cover(up8(c), 128), cover(a, 128) * cover(up8(c), 32));
    } else if (!strcmp(kind, "rows")) {
      answer(plan_rows(a, (int)b, (int)cover(c, 64)), cover(a, 256) * cover(b, 192), cover(a, 128) * cover(b, 64));
    } else if (!strcmp(kind, "dgate")) {
      answer(plan_dgate(a, (int)b, (int)up8(c)), cover(a, 256) * cover(up8(c), 192), cover(a, 128) * cover(up8(c), 64));
    } else if (!strcmp(kind, "weights")) {
      if (scanf("%lld", &d) != 1) return 1;
      answer(plan_weights(a, (int)b, (int)c, (int)d), 2 * cover(c, 256) * cover(up8(b), 256) + cover(d, 256) * cover(up8(c), 256),
             2 * cover(c, 128) * cover(up8(b), 64) + cover(d, 128) * cover(up8(c), 64));
    } else {
      return 1;
    }
  }
  return 0;
}
