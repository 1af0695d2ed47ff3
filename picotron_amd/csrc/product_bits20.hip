// C = A B in 20 bits a value: the large product (product_large.h) for a gradient that the next kernel reads at once.  bf16 would lose what that kernel's own rounding loses once more, fp32
// takes 4 bytes written and read where this takes 2.5.
#include "product_large.h"

using namespace pico;

extern "C" int pico_product_large_bits20(const void* a, const void* b, void* c, void* left, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int tile_m, int tile_n, void* stream) {
  const char* fn = "pico_product_large_bits20";
  if (N % 16 != 0 || !pico_product_large_takes(M, N, K, lda, ldb, 0, 1, 1))
    return fail(PICO_ERR_SHAPE, "%s: M=%lld N=%lld K=%lld row pitches %lld, %lld (as pico_product_large, a b, rows of c of a multiple of 16 elements)", fn, (long long)M, (long long)N, (long long)K,
                (long long)lda, (long long)ldb);
  if (!a || !b || !c || !left) return fail(PICO_ERR_NULL, "%s: a, b, c and left are required", fn);
  if (!aligned16(a) || !aligned16(b) || !aligned16(c) || !aligned16(left)) return fail(PICO_ERR_ALIGN, "%s: pointers must be 16-byte aligned", fn);
  const LargeBits20Params p = {{static_cast<const __bf16*>(a), static_cast<const __bf16*>(b), c, (int)M, (int)N, (int)K, lda, ldb, 0, 0, 1, false}, static_cast<uint32_t*>(left)};
  return launch_tiles<false, true, StoreBits20>(p, false, tile_m, tile_n, static_cast<hipStream_t>(stream));
}
