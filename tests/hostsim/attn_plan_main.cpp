// Sweeps the choice of a forward attention kernel (csrc/attn_plan.hpp) over sizes, zeros among them, and checks what the kernels take
// for granted: the key tiles are divided without a gap or an empty part, every part fits the join's table, and sizes fit 32 bits.
#include <stdio.h>

#include "../../pstl_diffusion_policy_amd/csrc/attn_plan.hpp"

using namespace pstl::attn;

static int failures = 0;
#define CHECK(x)                                                                                                             \
  do {                                                                                                                       \
    if (!(x) && failures++ < 20) printf("%s: B %d Hk %d R %d Lk %d f32 %d cus %d -> kind %d tiles %d splits %d of %d\n", #x, B, Hk, R, Lk, \
                                        f32, cus, p.kind, p.n_tiles, p.splits, p.tiles_per_split);                            \
  } while (0)

int main() {
  const int Bs[] = {0, 1, 2, 3, 7, 64, 65, 255, 4096, 70000}, heads[] = {1, 2, 5, 8, 64};
  const int Rs[] = {0, 1, 2, 15, 16, 17, 31, 32, 33, 64, 127, 128, 129, 777, 4096, 1 << 20};
  const int Ls[] = {0, 1, 16, 17, 31, 32, 33, 64, 65, 100, 127, 128, 129, 255, 256, 257, 300, 511, 512, 513, 544, 545, 767, 1000, 1024, 1025, 4097,
                    20000, 32768, 100003, 1 << 20, (1 << 29) + 31, (1 << 30) - 1};
  const int cu[] = {1, 7, 8, 64, 256, 304};
  long n = 0, split = 0;
  for (int B : Bs) for (int Hk : heads) for (int R : Rs) for (int Lk : Ls) for (int cus : cu) for (int f32 = 0; f32 < 2; ++f32) {
    const FwdPlan p = plan_forward(B, Hk, R, Lk, f32 != 0, cus);
    const int64_t units = (int64_t)B * Hk;
    ++n, split += p.splits > 1;
    CHECK(p.cus_per_xcd >= 1 && p.splits >= 1 && p.splits <= kMaxSplits);
    if (units * R == 0) {
      CHECK(p.splits == 1 && (int64_t)p.n_tiles * units == 0);
      continue;
    }
    const int rows = p.kind == kManyRows ? 128 : 32;
    CHECK((int64_t)p.n_tiles * rows >= R && (int64_t)(p.n_tiles - 1) * rows < R);      // every row in one tile
    CHECK(Lk > 32 ? p.kind == kManyRows || p.kind == kFewRows : p.kind == kShort || p.kind == kShortPairs);
    CHECK(p.kind != kShortPairs || (Lk <= 16 && R <= 16));
    CHECK(p.splits == 1 || p.kind == kFewRows);
    if (p.kind == kFewRows) {
      const int64_t key_tiles = ((int64_t)Lk + 31) / 32;
      CHECK(p.tiles_per_split >= 4 && p.tiles_per_split % 4 == 0);                     // the four wavefronts' turns
      CHECK((int64_t)p.splits * p.tiles_per_split >= key_tiles);                       // no key without a part
      CHECK((int64_t)(p.splits - 1) * p.tiles_per_split < key_tiles);                  // no part without a key
      CHECK((int64_t)p.splits * p.tiles_per_split * 32 + 128 < (1ll << 31));           // 32-bit key indexes in the kernel
      CHECK(p.splits == 1 || units * p.n_tiles * p.splits <= cus);                     // divided only to fill the chip
    }
  }
  printf("%ld plans, %ld divided, %d failures\n", n, split, failures);
  return failures != 0;
}
