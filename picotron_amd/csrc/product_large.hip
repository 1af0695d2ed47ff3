// Matrix products that fill the GPU: C = op(A) op(B) in bf16 with fp32 accumulation, in any of the three layouts of a linear
// layer (forward, input gradient, weight gradient).
//
// What bounds them is the matrix pipe and the power it draws: sustained products hold the clock at 1.6 .. 1.8 GHz, so an
// instruction that moves less through the registers per product is faster as well as cheaper.  Tiles of 256 x 256 (or one side
// 192 or 128, where that fills the CUs better) by eight waves, two per SIMD, one workgroup per CU that walks its tiles; 64 of
// contraction per step, two LDS buffers.  What the forms that were built reach, TFLOP/s at [8192 x 4096] @ [4096 x 8192]:
//   * products of 16 x 16 x 32 instead of 32 x 32 x 16: 1350 -> 1430 (half the accumulator traffic);
//   * one instruction between two products, whatever it is: a request of the next tile is one `buffer_load ... lds` (its place
//     in LDS goes into m0 one product earlier, the masks of a ragged contraction are made once per tile): 1290 -> 1350;
//   * operands go to LDS without passing the registers, 16 bytes per lane, all of them requested in the half step behind the
//     one that frees the buffer; fragments are read half a step ahead;
//   * a barrier whose two halves lie apart, with products between a wave's arrival and its wait: 102 -> 98 us at [4096 x 4096] @
//     [4096 x 4096], 423 -> 395 with a contraction of 16384, whose requests take longer;
//   * four waves of 128 x 128 (a third less LDS traffic): level with long contractions, 10 % behind with short ones; the two
//     waves of a SIMD in opposite phases of memory and products: 1300.
// LDS rows are swizzled so that neither the 16-byte reads down a column (fast contraction) nor the transposing reads (slow
// contraction) have bank conflicts; all three layouts run at the same rate (98 .. 103 us at 4096 cubed), where the GEMM library
// takes 91 in the forward's, 104 in the input gradient's and 137 in the weight gradient's.  The error against 64 bits is the
// library's (1.66e-3, the rounding to bf16).
#include "product_large.h"

namespace pico {
namespace {

template <bool kSlowA, bool kSlowB, bool kParts>
int launch_shape(const LargeParams& p, int tile_m, int tile_n, hipStream_t s) {
  return launch_tiles<kSlowA, kSlowB, StoreTile<kParts>>(p, kParts, tile_m, tile_n, s);
}

}  // namespace
}  // namespace pico

using namespace pico;

extern "C" int pico_product_large_takes(int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int a_slow, int b_slow, int parts) {
  constexpr int64_t kMost = 0x7fffffff;
  // (two steps per piece at least: the kernel requests one step ahead of the tile it works on)
  if (M < 1 || N < 1 || M > kMost / 2 || N > kMost / 256 || K > kMost - 4096 || N % 8 != 0 || (a_slow ? M : K) % 8 != 0 || (b_slow ? N : K) % 8 != 0 ||
      lda % 8 != 0 || ldb % 8 != 0 || lda < (a_slow ? M : K) || ldb < (b_slow ? N : K) || (a_slow && !b_slow) || parts < 1 || parts > 64 ||
      (K + kStep - 1) / kStep < 2 * parts)
    return 0;
  // the windows of the buffer loads: a tile's rows, or the whole contraction where that is the slow axis
  if (lda > kMost / 2 || ldb > kMost / 2 || ((a_slow ? K + kStep : 256) * lda + K) * 2 > kMost || ((b_slow ? K + kStep : 256) * ldb + K) * 2 > kMost)
    return 0;
  return ((M + 127) / 128) * ((N + 127) / 128) * parts <= kMost / 256;
}

namespace {
int product_large(const void* a, const void* b, void* c, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int a_slow, int b_slow, int tile_m, int tile_n, int parts, bool sums,
                  void* stream) {
  if (!pico_product_large_takes(M, N, K, lda, ldb, a_slow, b_slow, parts))
    return fail(PICO_ERR_SHAPE, "pico_product_large: M=%lld N=%lld K=%lld row pitches %lld, %lld, %d pieces (rows of a, b and c and the pitches must be multiples of 8 elements, two steps of 64 per piece, a tile's rows span less than 2 GiB, no a^T b^T)",
                (long long)M, (long long)N, (long long)K, (long long)lda, (long long)ldb, parts);
  if (!a || !b || !c) return fail(PICO_ERR_NULL, "pico_product_large: a, b and c are required");
  if (!aligned16(a) || !aligned16(b) || !aligned16(c)) return fail(PICO_ERR_ALIGN, "pico_product_large: pointers must be 16-byte aligned");
  const LargeParams p = {static_cast<const __bf16*>(a), static_cast<const __bf16*>(b), c, (int)M, (int)N, (int)K, lda, ldb, 0, 0, parts, false};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a_slow) return sums ? launch_shape<true, true, true>(p, tile_m, tile_n, s) : launch_shape<true, true, false>(p, tile_m, tile_n, s);
  if (b_slow) return sums ? launch_shape<false, true, true>(p, tile_m, tile_n, s) : launch_shape<false, true, false>(p, tile_m, tile_n, s);
  return sums ? launch_shape<false, false, true>(p, tile_m, tile_n, s) : launch_shape<false, false, false>(p, tile_m, tile_n, s);
}
}  // namespace

extern "C" int pico_product_large(const void* a, const void* b, void* c, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int a_slow,
                                  int b_slow, int tile_m, int tile_n, int parts, void* stream) {
  return product_large(a, b, c, M, N, K, lda, ldb, a_slow, b_slow, tile_m, tile_n, parts, parts > 1, stream);
}
extern "C" int pico_product_large_sums(const void* a, const void* b, float* sums, int64_t M, int64_t N, int64_t K, int64_t lda, int64_t ldb, int a_slow,
                                       int b_slow, int tile_m, int tile_n, int parts, void* stream) {
  return product_large(a, b, sums, M, N, K, lda, ldb, a_slow, b_slow, tile_m, tile_n, parts, true, stream);
}
