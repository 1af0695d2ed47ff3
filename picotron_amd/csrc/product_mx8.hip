// C = A B^T of rows in the 8-bit form (mx8.h) in bf16: the products of a layer whose activations and weights are held that way.
//
// The matrix instructions with scales multiply 32 e4m3 values of a row by 32 of another and apply both blocks' scales; four (16 x 16 x 128) or two
// (32 x 32 x 64) blocks to an instruction.  Where a lane's values lie: bytes 16 h .. + 15 of the row's 128 (64) and as many from the middle on, h the lane's quarter
// (half) of the wave; its scale is that of block h.  The sums are fp32 registers.  Within an instruction the products of eight neighbouring values of a row lose what lies 2^-13 under
// the largest of the eight (measured: 2^16 + 2^3 is whole, 2^16 + 2^2 is 2^16), others are added with 24 bits: over normal values 1.5e-5 of the result's root mean square
// (7e-5 with outliers of 20), without a bias and without growth from a contraction of 128 to one of 8192.  The rounding of the result to bf16 is 1.7e-3, so the result is bf16 only.
//
// What bounds it: few rows the weight's bytes, 1.03 of them a value and half of what bf16 takes ([1 x 2048] @ [16384 x 2048]^T 7.2 us, 4.8 TB/s, with its launch); many rows the matrix
// pipe and the power that it draws: [16384 x 4096] @ [4096 x 4096]^T 213 us (2.6 PFLOP/s), where the pipe is busy 69 % of the time at a clock of 1.8 GHz (as the large products in bf16
// are, at half the rate); [8192 x 8192] @ [8192 x 8192]^T 2.7, and 3.2 if all values are 0, which draw less.  A library's e4m3 product without block scales reaches 2.5 and 2.8.
#include <iterator>
#include "mx8.h"
#include "product_large.h"

namespace pico {
namespace {

typedef __attribute__((ext_vector_type(8))) int i32x8;

struct Mx8Params {
  const uint8_t *a, *b;        // [M, K], [N, K]
  const uint8_t *sa, *sb;      // their scales
  const __bf16* x;             // or a before it is rounded to 8 bits, with its pitch
  int64_t x_ld;
  void* c;                     // bf16 [M, N rounded up to 8]; fp32 [parts, M, N rounded up to 8] where the contraction goes in pieces
  int M, N, K, parts;
};

__device__ __forceinline__ i32x8 both(u32x4 low, u32x4 high) {
  return __builtin_bit_cast(i32x8, __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 16 values of each half of a row's 128, rounded to 8 bits as mx8.h has it, and the scale of block h of the four: a block lies in two lanes 16 apart, its scale goes to the lanes
// whose h it has.
__device__ __forceinline__ i32x8 encode_fragment(const u32x4 (&raw)[2][2], int lane, int& scale) {
  u32x4 code[2];
  uint32_t byte[2];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float v[16];
    uint32_t largest = 0;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const uint32_t pair = raw[half][e / 8][e % 8 / 2];
      v[e] = __uint_as_float(e % 2 ? pair & 0xffff0000u : pair << 16);
      largest = max(largest, __float_as_uint(v[e]) & 0x7fffffffu);
    }
    largest = max(largest, static_cast<uint32_t>(__shfl_xor(static_cast<int>(largest), 16, kWave)));
    byte[half] = scale_byte(largest);
    const float inverse = inverse_scale(byte[half]);
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const int low = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w] * inverse, v[4 * w + 1] * inverse, 0, false);
      code[half][w] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * w + 2] * inverse, v[4 * w + 3] * inverse, low, true));
    }
  }
  const int from = lane % 16 + lane / 16 % 2 * 32, first = __shfl(static_cast<int>(byte[0]), from, kWave), second = __shfl(static_cast<int>(byte[1]), from, kWave);
  scale = lane < 32 ? first : second;
  return both(code[0], code[1]);
}

// ---- few rows, and contractions under two steps: MT x NT tiles of 16 x 16 to a workgroup, whose W waves take every W-th 128 of the contraction straight from memory and join their sums in LDS.
// Bound by the weight's bytes or, where the tiles are few and long, by what one CU takes, 25 to 35 bytes a ns however much is on its way (four steps requested ahead instead of two: the same).
// A wave requests U steps before it uses the first.
// kRound: a is bf16 and every workgroup rounds it anew (MT 1): a launch less, us for rounding and product by two launches and by one, [1 x 2048] @ [16384 x 2048]^T 9.2, 8.0;
// [1 x 2048] @ [2048 x 2048]^T 7.1, 4.0; [1 x 11008] @ [4096 x 11008]^T 12.7, 13.5 (the same values rounded by 256 workgroups: rounding_form decides).
// kParts: the contraction goes in pieces over workgroups that leave fp32 sums, with larger tiles: [24 x 8192] @ [2048 x 8192]^T 10.1 us by 256 tiles of 16 x 16, of which each reads 256 KB, 8.8 by
// 64 tiles of 32 x 32 in four pieces, the sum's launch included.
template <int MT, int NT, int W, int U, bool kRound, bool kParts>
__global__ __launch_bounds__(W * kWave) void product_mx8_few_kernel(const Mx8Params p) {
  Arguments<0>().arrive();
  __shared__ f32x4 sums[W][MT * NT][kWave];
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), n = lane % 16, h = lane / 16;
  const int across = (p.N + 16 * NT - 1) / (16 * NT), tiles = across * ((p.M + 16 * MT - 1) / (16 * MT)), part = kParts ? static_cast<int>(blockIdx.x) / tiles : 0;
  const int tile_of = static_cast<int>(blockIdx.x) - part * tiles, m0 = tile_of / across * 16 * MT, n0 = tile_of % across * 16 * NT;
  const int steps = (p.K + kGroup - 1) / kGroup, first = kParts ? part * steps / p.parts : 0, end = kParts ? (part + 1) * steps / p.parts : steps;
  // rows past the matrix read its last one, and what they give is not written
  int64_t ra[MT], rb[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) ra[i] = min(m0 + 16 * i + n, p.M - 1);
#pragma unroll
  for (int j = 0; j < NT; ++j) rb[j] = min(n0 + 16 * j + n, p.N - 1);
  f32x4 acc[MT][NT];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int t0 = first + wave; t0 < end; t0 += U * W) {
    u32x4 a[kRound ? 1 : U][MT][2], b[U][NT][2], x[kRound ? U : 1][2][2];
    int sa[U][MT], sb[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // pieces past the contraction read their row's first ones, steps past this piece of it the next one's; b's are made 0 below (a's row is NaN as a whole or finite)
      const int t = min(t0 + u * W, steps - 1), k = (t0 + u * W) * kGroup + 16 * h;
      const int64_t low = k < p.K ? k : 0, high = k + 64 < p.K ? k + 64 : 0;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        b[u][j][0] = *reinterpret_cast<const u32x4*>(p.b + rb[j] * p.K + low);
        b[u][j][1] = *reinterpret_cast<const u32x4*>(p.b + rb[j] * p.K + high);
        sb[u][j] = p.sb[(static_cast<int64_t>(t) * p.N + rb[j]) * 4 + h];
      }
      if constexpr (kRound) {
        const __bf16* row = p.x + ra[0] * p.x_ld;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          x[u][0][q] = *reinterpret_cast<const u32x4*>(row + low + 8 * q);
          x[u][1][q] = *reinterpret_cast<const u32x4*>(row + high + 8 * q);
        }
      }
#pragma unroll
      for (int i = 0; i < (kRound ? 0 : MT); ++i) {
        a[u][i][0] = *reinterpret_cast<const u32x4*>(p.a + ra[i] * p.K + low);
        a[u][i][1] = *reinterpret_cast<const u32x4*>(p.a + ra[i] * p.K + high);
        sa[u][i] = p.sa[(static_cast<int64_t>(t) * p.M + ra[i]) * 4 + h];
      }
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = (t0 + u * W < end ? t0 + u * W : steps) * kGroup + 16 * h;
      const u32x4 zero = {0, 0, 0, 0};
      i32x8 fb[NT];
#pragma unroll
      for (int j = 0; j < NT; ++j) fb[j] = both(k < p.K ? b[u][j][0] : zero, k + 64 < p.K ? b[u][j][1] : zero);
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        i32x8 fa;
        if constexpr (kRound) fa = encode_fragment(x[u], lane, sa[u][i]);   // (past the contraction: whatever its first values give, times b's zeros)
        else fa = both(a[u][i][0], a[u][i][1]);
#pragma unroll
        for (int j = 0; j < NT; ++j)   // C^T: a lane holds four columns of a row of C
          acc[i][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa, acc[i][j], 0, 0, 0, sb[u][j], 0, sa[u][i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j) sums[wave][i * NT + j][lane] = acc[i][j];
  __syncthreads();
  const int ldc = (p.N + 7) / 8 * 8;
  for (int tile = wave; tile < MT * NT; tile += W) {
    f32x4 v = sums[0][tile][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += sums[w][tile][lane];
    const int row = m0 + 16 * (tile / NT) + n, col = n0 + 16 * (tile % NT) + 4 * h;
    if (row >= p.M || col >= ldc) continue;
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = col + e < p.N ? v[e] : 0.f;
    if constexpr (kParts) {
      *reinterpret_cast<f32x4*>(static_cast<float*>(p.c) + (static_cast<int64_t>(part) * p.M + row) * ldc + col) = v;
    } else {
      bf16x4 o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = static_cast<__bf16>(v[e]);
      *reinterpret_cast<bf16x4*>(static_cast<__bf16*>(p.c) + static_cast<int64_t>(row) * ldc + col) = o;
    }
  }
}

template <int MT, int NT, int W, int U, bool kRound, bool kParts>
int launch_few(const Mx8Params& p, hipStream_t s) {
  const int64_t tiles = ((p.N + INT64_C(16) * NT - 1) / (16 * NT)) * ((p.M + INT64_C(16) * MT - 1) / (16 * MT)) * p.parts;
  if (tiles * W * kWave > 0xffffffff) return fail(PICO_ERR_SHAPE, "pico_mx8_product: M=%d N=%d with K=%d has too many tiles (a launch has under 2^32 threads)", p.M, p.N, p.K);
  hipLaunchKernelGGL((product_mx8_few_kernel<MT, NT, W, U, kRound, kParts>), dim3(static_cast<unsigned>(tiles)), dim3(W * kWave), 0, s, p);
  return check_launch("pico_mx8_product");
}
// What can be asked for: tiles of 16 x 16 to a workgroup, its waves, steps that a wave requests at once (of the forms that round, two), and whether the contraction can go in pieces.  us of the
// best of the others and of each where it serves: 2048 columns and a contraction of 2048, 24 rows, 4.0 by the first, 4.6; [4096 x 4096], one row, 5.3 by the third (16 waves), 6.4;
// [16384 x 1280], 16 rows, 6.4 by the fourth, 7.1; [16384 x 2048], 24 rows, 9.3 by {2, 4}, 9.8; [4096 x 128], 4096 rows, 20.5 by the last, 39.5 by eight waves.
struct Few {
  int mt, nt, waves, ahead;
  bool parts;
};
constexpr Few kFew[] = {{1, 1, 4, 2, false}, {1, 1, 8, 2, false}, {1, 1, 16, 2, false}, {1, 2, 8, 1, true}, {2, 1, 8, 2, false}, {2, 2, 8, 2, true}, {2, 4, 8, 1, false}, {4, 4, 8, 1, false}, {4, 2, 2, 1, false}};
constexpr int kForms = static_cast<int>(std::size(kFew)), kRoundForms = 4;   // (the first ones have one tile of rows)
static_assert(kFew[kRoundForms - 1].mt == 1 && kFew[kRoundForms].mt > 1);
template <bool kRound, int... v>
int dispatch_few(const Mx8Params& p, int form, hipStream_t s, std::integer_sequence<int, v...>) {
  int rc = PICO_ERR_SHAPE;
  auto launch = [&](auto of) {
    constexpr Few f = kFew[decltype(of)::value];
    if constexpr (f.parts && !kRound) {
      if (p.parts > 1) return launch_few<f.mt, f.nt, f.waves, f.ahead, false, true>(p, s);
    }
    return launch_few<f.mt, f.nt, f.waves, kRound ? 2 : f.ahead, kRound, false>(p, s);
  };
  ((form == v ? static_cast<void>(rc = launch(std::integral_constant<int, v>())) : void()), ...);
  return rc;
}

// ---- many rows: the large products' workgroups (product_large.h) with 128 of contraction a step
//
// An e4m3 matrix [rows, K] is staged as a bf16 one [rows, K / 2] would be: a step is 128 bytes of every row of the tiles.  2 x 4 waves of 32 I x 32 J;
// each half of a step is one 32 x 32 x 64 product per pair of fragments.  The scales of a step's rows, four bytes a row, take one request more: 64 rows by each wave.
struct Mx8Large : LargeParams {   // (a, b, K and the pitches in pairs of values; N without the columns that round the output up)
  const uint8_t *sa, *sb;
  int cols;                       // of c
};
// wait_requests<kMore> where `but` is not 0, wait_requests<kLess> where it is.  The branch is inside: products ahead of one that the compiler sees would be moved behind it.
template <int kLess, int kMore>
__device__ __forceinline__ void wait_requests_but(int but) {
  static_assert(kLess <= kMore && kMore < 64);
  asm volatile("s_cmp_lg_u32 %0, 0\n\ts_cbranch_scc1 pico_but_%=\n\ts_waitcnt vmcnt(%1)\npico_but_%=:\n\ts_waitcnt vmcnt(%2)" ::"s"(but), "n"(kLess), "n"(kMore) : "scc", "memory");
}
// unit_at of product_large.h in 32 bits and scalar registers: pieces times steps stay under 2^21 here, and a division of 64 bits takes the sizes, and with them the loops' counts and the
// windows, through vector registers.
template <int TM, int TN>
__device__ __forceinline__ bool mx8_unit_at(const Mx8Large& p, int round, Unit& u) {
  const int tiles = p.tiles_m * p.tiles_n, grid = gridDim.x, start = round * grid, count = min(grid, tiles * p.parts - start);
  if (static_cast<int>(blockIdx.x) >= count) return false;
  const int xcd = blockIdx.x % 8, id = start + xcd * (count / 8) + min(xcd, count % 8) + blockIdx.x / 8;
  constexpr int kDeep = 8;
  u.part = __builtin_amdgcn_readfirstlane(id / tiles);
  const int t = id - u.part * tiles, block = __builtin_amdgcn_readfirstlane(t / (kDeep * p.tiles_n)), in = t - block * kDeep * p.tiles_n, deep = min(kDeep, p.tiles_m - block * kDeep);
  const int column = __builtin_amdgcn_readfirstlane(in / deep);
  u.m0 = (block * kDeep + in - column * deep) * TM;
  u.n0 = column * TN;
  const int steps = (p.K + kStep - 1) / kStep;
  u.first = __builtin_amdgcn_readfirstlane(u.part * steps / p.parts);
  u.steps = __builtin_amdgcn_readfirstlane((u.part + 1) * steps / p.parts) - u.first;
  return true;
}
// kWavesM x kWavesN waves of 32 I x 32 J, and as many buffers as kPerCu workgroups find place for in a CU's LDS (two of tiles of 256 x 256; four of 128 x 128, or two where two
// workgroups share a CU; six of 64 x 128).  Where there are fewer tiles than CUs nothing else hides what a request takes, about 0.5 us: us with two buffers and with four or six,
// [1003 x 11008] @ [4096 x 11008]^T in tiles of 128 x 128 70.3, 52.2; [512 x 2048] @ [2048 x 2048]^T in 64 x 128 11.6, 10.2.  Where there are more, a second workgroup does
// better: [4096 x 2048] @ [2048 x 2048]^T 19.3, and 23.5 with four buffers and one workgroup.
template <int kWavesM, int kWavesN, int I, int J, int kPerCu>
struct Mx8Shape {
  static constexpr int kWaves = kWavesM * kWavesN, kThreads = kWaves * kWave, TM = 32 * I * kWavesM, TN = 32 * J * kWavesN;
  using A = Tile<false, TM, kThreads>;
  using B = Tile<false, TN, kThreads>;
  static constexpr int kScales = A::kBytes + B::kBytes, kBuffer = kScales + kWaves * 256;   // (the scales of 64 rows by each wave)
  static constexpr int kRowRegion = 16 * 128, kMost = 160 * 1024 / kPerCu, kBuffers = (kMost - kWaves * kRowRegion) / kBuffer;   // (rows: per wave, where a tile's rows are put together)
  static constexpr int kRows = kBuffers * kBuffer, kLds = kRows + kWaves * kRowRegion;
  static_assert(kBuffers >= 2 && kLds <= kMost && (TM + TN) / 64 <= kWaves && TM % 64 == 0);
};
template <int kPlus>
__device__ __forceinline__ void request16_along(uint32_t lds_off, u32x4 window, uint32_t off, uint32_t along) {   // request16_to with a scalar offset
  uint32_t aim;
  asm volatile("s_add_u32 %0, %1, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %3, %4, %5 offen lds"
               : "=&{m0}"(aim) : "s"(lds_off), "n"(kPlus), "v"(off), "s"(window), "s"(along) : "scc", "memory");
}
template <int kPlus>
__device__ __forceinline__ void request4_to(uint32_t lds_off, u32x4 window, uint32_t off) {   // request16_to of 4 bytes per lane
  uint32_t aim;
  asm volatile("s_add_u32 %0, %1, %2\n\ts_nop 0\n\tbuffer_load_dword %3, %4, 0 offen lds" : "=&{m0}"(aim) : "s"(lds_off), "n"(kPlus), "v"(off), "s"(window) : "scc", "memory");
}

// The tile leaves as in product_large.h, 16 rows and 128 bytes of columns at a time through LDS.  A lane holds, of row lane % 32 of a 32 x 32 block, columns 8 q + 4 h .. + 3:
// two q change places between the two 16 rows, so that all lanes write each time (branches on lanes would cost the kernel its scalar registers).
template <typename Out, int I, int J>
__device__ __forceinline__ void store_tile32(Out* c, int64_t first_row, int M, int cols, bool streaming, int row0, int col0, int lane, unsigned char* rows, const f32x16 (&acc)[I][J]) {
  constexpr int kBlocks = 128 / 32 / static_cast<int>(sizeof(Out)) < J ? 128 / 32 / static_cast<int>(sizeof(Out)) : J;   // of 32 columns at a time
  constexpr int kWords = sizeof(Out);   // of four columns
  const int n = lane % 16, odd = lane / 16 % 2, h = lane / 32, left = cols - col0;
  const uint32_t pitch = static_cast<uint32_t>(cols) * sizeof(Out), back = lane / 8 * pitch + lane % 8 * 16;
#pragma unroll
  for (int i = 0; i < I; ++i) {
#pragma unroll
    for (int j0 = 0; j0 < J; j0 += kBlocks) {
      uint32_t word[2][kBlocks][2][kWords];   // of the first and the second 16 rows: column blocks 2 k + odd
#pragma unroll
      for (int j = 0; j < kBlocks; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
          for (int w = 0; w < kWords; ++w) {
            auto packed = [&](int q) {
              if constexpr (sizeof(Out) == 4) return __float_as_uint(acc[i][j0 + j][4 * q + w]);
              else return pack_bf16x2(acc[i][j0 + j][4 * q + 2 * w], acc[i][j0 + j][4 * q + 2 * w + 1]);
            };
            const auto swapped = __builtin_amdgcn_permlane16_swap(packed(2 * k), packed(2 * k + 1), false, false);
            word[0][j][k][w] = swapped[0];
            word[1][j][k][w] = swapped[1];
          }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int j = 0; j < kBlocks; ++j)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            unsigned char* to = rows + n * 128;
            const int q = 2 * k + odd;
            if constexpr (sizeof(Out) == 4)
              *reinterpret_cast<u32x4*>(to + ((j * 8 + 2 * q + h) ^ (n / 2)) * 16) = u32x4{word[half][j][k][0], word[half][j][k][1], word[half][j][k][2], word[half][j][k][3]};
            else
              *reinterpret_cast<u32x2*>(to + ((j * 4 + q) ^ (n / 2)) * 16 + h * 8) = u32x2{word[half][j][k][0], word[half][j][k][1]};
          }
        const int first = row0 + 32 * i + 16 * half, live = min(16, M - first);
        const u32x4 r = request_window(reinterpret_cast<uint64_t>(c + (first_row + first) * cols + col0),
                                       live > 0 && left > 0 ? static_cast<uint32_t>(((live - 1) * static_cast<int64_t>(cols) + left) * sizeof(Out)) : 0u);
        const buffer_rsrc window = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(r[0] | static_cast<uint64_t>(r[1]) << 32), 0, static_cast<int>(r[2]), static_cast<int>(r[3]));
        const int col = lane % 8 * (16 / static_cast<int>(sizeof(Out)));
        const bool in = col < kBlocks * 32 && 32 * j0 + col < left;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int row = 8 * q + lane / 8;
          const u32x4 v = *reinterpret_cast<const u32x4*>(rows + row * 128 + ((lane % 8) ^ (row / 2)) * 16);
          const int to = in ? static_cast<int>(back + 8 * q * pitch + 32 * j0 * sizeof(Out)) : static_cast<int>(0xfffffff0u);
          constexpr int kStreaming = 2;
          if (streaming) __builtin_amdgcn_raw_buffer_store_b128(v, window, to, 0, kStreaming);
          else __builtin_amdgcn_raw_buffer_store_b128(v, window, to, 0, 0);
        }
      }
    }
  }
}

template <int kWavesM, int kWavesN, int I, int J, int kPerCu, bool kParts>
__global__ __launch_bounds__(kWavesM * kWavesN * kWave, 2) void product_mx8_kernel(const Mx8Large p) {
  using S = Mx8Shape<kWavesM, kWavesN, I, J, kPerCu>;
  using A = typename S::A;
  using B = typename S::B;
  constexpr int TM = S::TM, TN = S::TN, kPA = A::kPieces, kPB = B::kPieces, kPieces = kPA + kPB;
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds[];
  const int tid = threadIdx.x, lane = tid % kWave, wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int wm = wave / kWavesN * 32 * I, wn = wave % kWavesN * 32 * J, n = lane % 32, h = lane / 32;

  // ---- requests (as in product_large_kernel; both operands have one pitch, and a thread's pieces lie kThreads / 8 rows apart)
  const uint32_t piece_bytes = static_cast<uint32_t>(p.lda) * (S::kThreads / 8 * 2);
  uint32_t first_piece = A::offset(p.lda, tid, 0);
  const int k_piece = (tid % 8 ^ (tid / 16 & 7)) * 8;
  const bool ragged = p.K % kStep != 0;
  Unit load;   // where the requests stand
  int load_round = 0, load_step = 0;
  mx8_unit_at<TM, TN>(p, 0, load);
  // A tile's windows stay where they are and the contraction goes on in the requests' scalar offset, with which a piece in the window stays in its row (a piece of a row past the
  // matrix lies past the window without it).  The scales of the steps lie as far apart as the matrix has rows: their window moves.
  u32x4 ra, rb, rs;
  uint32_t along = 0;
  uint64_t s_base;
  // the scales of this wave's 64 rows: of a for the first TM / 64 waves, of b for the others
  constexpr int kOfA = TM / 64;
  const bool of_a = wave < kOfA;
  const int s_rows = of_a ? p.M : p.N, s_first = (of_a ? wave : wave - kOfA) * 64;
  auto open = [&](uint32_t whole) __attribute__((always_inline)) {   // (whole 0: requests past the work's end read no memory)
    const Window wa = open_window<false>(p.a, p.lda, load.m0, TM, p.M, load.first * kStep, p.K), wb = open_window<false>(p.b, p.ldb, load.n0, TN, p.N, load.first * kStep, p.K);
    const int first = (of_a ? load.m0 : load.n0) + s_first;
    s_base = reinterpret_cast<uint64_t>(of_a ? p.sa : p.sb) + (static_cast<int64_t>(load.first) * s_rows + first) * 4;
    ra = request_window(wa.base, wa.bytes * whole);
    rb = request_window(wb.base, wb.bytes * whole);
    rs = request_window(s_base, first < s_rows ? static_cast<uint32_t>(min(s_rows - first, 64)) * 4 * whole : 0u);
    along = 0;
  };
  open(1);
  auto go_on = [&]() __attribute__((always_inline)) {
    ++load_step;
    along += kStep * 2;
    s_base += static_cast<uint32_t>(s_rows) * 4u;
    rs[0] = static_cast<uint32_t>(s_base);
    rs[1] = static_cast<uint32_t>(s_base >> 32);
    if (load_step >= load.steps - 1) {
      if (load_step == load.steps) {
        load_step = 0;
        open(mx8_unit_at<TM, TN>(p, ++load_round, load) ? 1 : 0);
      }
      if (ragged)   // pieces past the contraction's end read as zeros (their scales are bytes of 0, no NaN); a window is under 2^31 bytes, and so is a row's end past this
        first_piece = k_piece < p.K - (load.first + load_step) * kStep ? A::offset(p.lda, tid, 0) : 0x80000000u;
    }
    along = __builtin_amdgcn_readfirstlane(along);   // (they are scalars; the compiler does not see it behind the branch)
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      ra[i] = __builtin_amdgcn_readfirstlane(ra[i]);
      rb[i] = __builtin_amdgcn_readfirstlane(rb[i]);
      rs[i] = __builtin_amdgcn_readfirstlane(rs[i]);
    }
  };
  const uint32_t lds_wave = wave * 1024, lds_scales = S::kScales + wave * 256;   // (dynamic LDS starts at 0: the build looks)
  auto request = [&](auto piece, uint32_t buffer) __attribute__((always_inline)) {
    constexpr int i = decltype(piece)::value;
    if constexpr (i < kPA) request16_along<i * S::kThreads * 16>(lds_wave + buffer, ra, first_piece + i * piece_bytes, along);
    else if constexpr (i < kPieces) request16_along<A::kBytes + (i - kPA) * S::kThreads * 16>(lds_wave + buffer, rb, first_piece + (i - kPA) * piece_bytes, along);
    else request4_to<0>(lds_scales + buffer, rs, static_cast<uint32_t>(lane) * 4);
  };
  constexpr int kRequests = kPieces + 1, kAhead = (S::kBuffers - 2) * kRequests;   // of a step; of the steps behind the one that is waited for
  using Out = std::conditional_t<kParts, float, __bf16>;
  constexpr int kAtOnce = 128 / 32 / static_cast<int>(sizeof(Out)), kStores = 2 * I * ((J + kAtOnce - 1) / kAtOnce) * 2;   // of a wave, at a tile's end

  // ---- half a step: its products, row by row of the wave's tile.  A fragment of a is read anew, for the half step that follows, as soon as its row is done, those of b are
  // held twice.  The workgroup meets once a step, behind the first product of the second half: a wave's reads of the buffer in use are complete there, and so are its
  // requests for the next; from there on it reads the next buffer and requests into the one that was in use.  (A barrier in two halves over a count in LDS, as product_large.h
  // has it, is slower here: [4096 x 2048] @ [16384 x 2048]^T 119.7 us against 116.4, tiles of 128 x 128 27.4 against 23.8 at [1024 x 4096] @ [4096 x 4096]^T.)
  constexpr int kProducts = I * J;
  i32x8 fa[I], fb[2][J];
  int sca[I], scb[2][J];
  f32x16 acc[I][J];
  // row `first` + n, bytes 64 s + 16 h and 32 further, and the scale of bytes 64 s + 32 h .. + 31
  auto fragment = [&](const unsigned char* tile, int first, int s) __attribute__((always_inline)) {
    const unsigned char* row = tile + first * 128 + n * 128;
    return both(*reinterpret_cast<const u32x4*>(row + ((4 * s + h) ^ (n / 2 & 7)) * 16), *reinterpret_cast<const u32x4*>(row + ((4 * s + 2 + h) ^ (n / 2 & 7)) * 16));
  };
  auto scale = [&](uint32_t buffer, int first, int s) __attribute__((always_inline)) { return lds[S::kScales + buffer + (first + n) * 4 + 2 * s + h]; };
  auto fetch_a = [&](uint32_t buffer, int s, int i) __attribute__((always_inline)) {
    fa[i] = fragment(lds + buffer, wm + 32 * i, s);
    sca[i] = scale(buffer, wm + 32 * i, s);
  };
  auto fetch_b = [&](uint32_t buffer, int s, int j) __attribute__((always_inline)) {
    fb[s][j] = fragment(lds + buffer + A::kBytes, wn + 32 * j, s);
    scb[s][j] = scale(buffer, TM + wn + 32 * j, s);
  };
  auto half_step = [&](auto half, uint32_t next, uint32_t free, int stores) __attribute__((always_inline)) {
    constexpr int s = decltype(half)::value;
    each(std::make_integer_sequence<int, kProducts>(), [&](auto product) __attribute__((always_inline)) {
      constexpr int m = decltype(product)::value, i = m / J, j = i % 2 ? J - 1 - m % J : m % J;
      __builtin_amdgcn_sched_barrier(0);
      // C^T: a lane holds columns of a row of C
      acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(fb[s][j], fa[i], acc[i][j], 0, 0, 0, scb[s][j], 0, sca[i]);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (s == 1 && m == 0) {
        // the next step's requests, behind which lie those of kBuffers - 2 steps more and, in a tile's first steps, the stores of the tile before
        wait_requests_but<kAhead, kAhead + kStores>(stores);
        wait_lds();
        __builtin_amdgcn_s_barrier();
      }
#pragma unroll
      for (int f = 0; f < J; ++f)
        if ((f < kProducts ? f : kProducts - 1) == m) fetch_b(next, 1 - s, f);
#pragma unroll
      for (int f = 0; f < I; ++f)
        if (f * J + J - 1 == m) fetch_a(next, 1 - s, f);
      if constexpr (s == 1)
        each(std::make_integer_sequence<int, kRequests>(), [&](auto piece) __attribute__((always_inline)) {
          if constexpr (decltype(piece)::value * kProducts / kRequests == m) request(piece, free);
        });
      __builtin_amdgcn_sched_barrier(0);
    });
  };

  auto all_requests = [&](uint32_t buffer) __attribute__((always_inline)) {
    each(std::make_integer_sequence<int, kRequests>(), [&](auto piece) __attribute__((always_inline)) { request(piece, buffer); });
  };
#pragma unroll
  for (int b = 0; b < S::kBuffers; ++b) {
    if (b > 0) go_on();
    all_requests(b * S::kBuffer);
  }
  wait_requests<kAhead + kRequests>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < I; ++i) fetch_a(0, 0, i);
#pragma unroll
  for (int j = 0; j < J; ++j) fetch_b(0, 0, j);

  unsigned char* rows = lds + S::kRows + wave * S::kRowRegion;
  uint32_t now = 0;   // the buffer of this step
  Unit u;
  for (int round = 0; mx8_unit_at<TM, TN>(p, round, u); ++round) {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.f;
#pragma unroll 1
    for (int t = 0; t < u.steps; ++t) {
      const uint32_t then = now == (S::kBuffers - 1) * S::kBuffer ? 0 : now + S::kBuffer;
      __builtin_amdgcn_s_setprio(0);
      go_on();   // (its branch ahead of the products: the compiler would move those before a branch behind it)
      half_step(std::integral_constant<int, 0>(), now, 0, 0);
      __builtin_amdgcn_s_setprio(1);
      half_step(std::integral_constant<int, 1>(), then, now, t < S::kBuffers - 1 ? round : 0);   // (requests a step that comes kBuffers later into `now`)
      now = then;
    }
    store_tile32<Out, I, J>(static_cast<Out*>(p.c), static_cast<int64_t>(u.part) * p.M, p.M, p.cols, p.streaming, u.m0 + wm, u.n0 + wn, lane, rows, acc);
  }
  wait_requests<0>();   // (requests past the work's end still write zeros to LDS)
}

template <int kWavesM, int kWavesN, int I, int J, int kPerCu, bool kParts>
int launch_large(const Mx8Params& q, void* c, int parts, hipStream_t s) {
  using S = Mx8Shape<kWavesM, kWavesN, I, J, kPerCu>;
  static LdsOnce reserved;
  if (!reserve_lds_once(reserved, reinterpret_cast<const void*>(&product_mx8_kernel<kWavesM, kWavesN, I, J, kPerCu, kParts>), S::kLds))
    return fail(PICO_ERR_LAUNCH, "pico_mx8_product: cannot reserve %d bytes of LDS", S::kLds);
  Mx8Large p;
  p.a = reinterpret_cast<const __bf16*>(q.a);
  p.b = reinterpret_cast<const __bf16*>(q.b);
  p.c = c;
  p.M = q.M;
  p.N = q.N;
  p.K = q.K / 2;
  p.lda = p.ldb = p.K;
  p.tiles_m = (q.M + S::TM - 1) / S::TM;
  p.tiles_n = (q.N + S::TN - 1) / S::TN;
  p.parts = parts;
  p.sa = q.sa;
  p.sb = q.sb;
  p.cols = (q.N + 7) / 8 * 8;
  const int64_t units = static_cast<int64_t>(p.tiles_m) * p.tiles_n * parts;
  constexpr int kGrid = 256 * kPerCu;
  p.streaming = !kParts && units > kGrid;   // (as for the large products in bf16)
  hipLaunchKernelGGL((product_mx8_kernel<kWavesM, kWavesN, I, J, kPerCu, kParts>), dim3(static_cast<unsigned>(std::min<int64_t>(units, kGrid))), dim3(S::kThreads), S::kLds, s, p);
  return check_launch("pico_mx8_product");
}
// What can be asked for: the sides of a tile, workgroups to a CU.
struct Tiling {
  int tile_m, tile_n, per_cu;
  float step, step_full, end;   // us a step with few tiles and with every CU taken, us a tile beside them (for route)
};
constexpr Tiling kTilings[] = {{256, 256, 1, 1.03f, 1.60f, 2.0f}, {128, 256, 1, 0.72f, 0.93f, 1.5f}, {256, 128, 1, 0.72f, 0.93f, 1.5f}, {128, 128, 2, 0.55f, 0.93f, 1.5f}, {128, 128, 1, 0.44f, 0.53f, 1.2f},
                               {64, 128, 1, 0.35f, 0.38f, 1.0f}};
template <bool kParts>
int launch_shape(const Mx8Params& p, void* c, int tile_m, int tile_n, int per_cu, int parts, hipStream_t s) {
  if (tile_m == 256 && tile_n == 256 && per_cu == 1) return launch_large<2, 4, 4, 2, 1, kParts>(p, c, parts, s);
  if (tile_m == 128 && tile_n == 256 && per_cu == 1) return launch_large<2, 4, 2, 2, 1, kParts>(p, c, parts, s);
  if (tile_m == 256 && tile_n == 128 && per_cu == 1) return launch_large<4, 2, 2, 2, 1, kParts>(p, c, parts, s);
  if (tile_m == 128 && tile_n == 128 && per_cu == 2) return launch_large<2, 2, 2, 2, 2, kParts>(p, c, parts, s);
  if (tile_m == 128 && tile_n == 128 && per_cu == 1) return launch_large<2, 2, 2, 2, 1, kParts>(p, c, parts, s);
  if (tile_m == 64 && tile_n == 128 && per_cu == 1) return launch_large<2, 2, 1, 2, 1, kParts>(p, c, parts, s);
  return fail(PICO_ERR_SHAPE, "pico_mx8_product: tiles of %d x %d, %d workgroups to a CU (64 x 128, or sides of 128 or 256; 2 for 128 x 128)", tile_m, tile_n, per_cu);
}

// Which kernel, tiles and pieces of the contraction a product of these sizes goes to.  tile_m 0: the kernel of few rows, in form tile_n.
struct Route {
  int tile_m, tile_n, per_cu, parts;
};
bool large_takes(int64_t M, int64_t N, int64_t K, int parts) {
  return parts >= 1 && parts <= 64 && (K + 127) / 128 >= 2 * parts && K <= (1 << 22) && ((M + 63) / 64) * ((N + 127) / 128) * parts <= 0x7fffffff / 256 && N <= 0x7fffffff / 256 && M <= 0x7fffffff / 2;
}
// us that the sum of the pieces takes: a launch, and the sums again at 4 TB/s
float join_us(int64_t M, int64_t N, int parts) { return parts > 1 ? 3.3f + 0.2f * parts + (4.f * parts + 2.f) * M * ((N + 7) / 8 * 8) * 2.5e-7f : 0.f; }
// A form of the kernel of few rows, its pieces, and its time: the longer of what a CU takes from memory and the caches (about 25 bytes a ns) and the weight's bytes, and the waits for one
// request after the other.
struct FewRoute {
  int form, parts;
  float us;
};
// `waves` not 0: of the forms that round, among those whose sums go over as many waves
FewRoute few_route(int64_t M, int64_t N, int64_t K, int waves) {
  const bool rounding = waves != 0;
  FewRoute best = {0, 1, 1e30f};
  for (int v = 0; v < (rounding ? kRoundForms : kForms); ++v) {
    const Few& f = kFew[v];
    if ((rounding && f.waves != waves) || (f.mt > 1 && M <= 8 * f.mt)) continue;   // (half a tile of rows would be empty)
    const int ahead = rounding ? 2 : f.ahead;
    for (int parts : {1, 4, 8}) {
      const int64_t steps = ((K + 127) / 128 + parts - 1) / parts;
      if (parts > 1 && (rounding || !f.parts || (K + 127) / 128 < parts)) break;
      const int64_t blocks = (M + 16 * f.mt - 1) / (16 * f.mt), per_cu = (blocks * ((N + 16 * f.nt - 1) / (16 * f.nt)) * parts + 255) / 256, turns = (steps + f.waves * ahead - 1) / (f.waves * ahead);
      const float rows = static_cast<float>(M) / (16 * blocks);   // (rows past the matrix cost no memory)
      const float a = rounding ? 1.1f * rows + 0.18f : 0.7f * rows;   // (bf16, and the rounding)
      const float asked = steps + 0.5f * (turns * f.waves * ahead - steps);   // (steps past the end are requested too)
      const float us = 2.6f + std::max(0.09f * per_cu * asked * (f.nt + a), 1.3e-7f * N * K) + 0.17f * (turns - 1) / per_cu + join_us(M, N, parts);
      if (us < best.us) best = {v, parts, us};
    }
  }
  return best;
}
Route route(int64_t M, int64_t N, int64_t K, float& least) {
  const int64_t steps = (K + 127) / 128;
  const FewRoute few = few_route(M, N, K, 0);
  Route best = {0, few.form, 1, few.parts};
  least = few.us;
  if (M <= 8 || !large_takes(M, N, K, 1)) return best;
  for (const Tiling& t : kTilings)
    for (int parts = 1; parts <= 16 && large_takes(M, N, K, parts); parts *= 2) {
      const int64_t units = ((M + t.tile_m - 1) / t.tile_m) * ((N + t.tile_n - 1) / t.tile_n) * parts, slots = 256 * t.per_cu, rounds = (units + slots - 1) / slots;
      const float taken = static_cast<float>(units < slots ? units : slots) / slots, step = std::max(t.step, t.step_full * taken);
      const float us = 5.4f + rounds * ((steps + parts - 1) / parts * step + t.end) + join_us(M, N, parts);
      if (us < least) {
        least = us;
        best = {t.tile_m, t.tile_n, t.per_cu, parts};
      }
    }
  return best;
}

}  // namespace
}  // namespace pico

using namespace pico;

namespace {
int check_product(const char* fn, const pico_mx8* a, const pico_mx8* b, const void* c, int64_t M, int64_t N, int64_t K) {
  if (int rc = check_mx8_shape(fn, M, K)) return rc;
  if (int rc = check_mx8_shape(fn, N, K)) return rc;
  if (M == 0 || N == 0) return PICO_OK;
  if (int rc = check_mx8(fn, "a", a)) return rc;
  if (int rc = check_mx8(fn, "b", b)) return rc;
  if (!c) return fail(PICO_ERR_NULL, "%s: c is required", fn);
  if (!aligned16(c)) return fail(PICO_ERR_ALIGN, "%s: c must be 16-byte aligned", fn);
  return PICO_OK;
}
int64_t parts_bytes(int64_t M, int64_t N, int parts) { return parts > 1 ? parts * M * ((N + 7) / 8 * 8) * 4 : 0; }
}  // namespace

extern "C" int64_t pico_mx8_product_workspace_bytes(int64_t M, int64_t N, int64_t K) {
  if (M < 1 || N < 1 || K < 1) return 0;
  float us;
  return parts_bytes(M, N, route(M, N, K, us).parts);
}

extern "C" int pico_mx8_product_tiled(const pico_mx8* a, const pico_mx8* b, void* c, int64_t M, int64_t N, int64_t K, int tile_m, int tile_n, int per_cu, int parts, void* workspace,
                                      int64_t workspace_bytes, void* stream) {
  const char* fn = "pico_mx8_product";
  if (int rc = check_product(fn, a, b, c, M, N, K)) return rc;
  if (M == 0 || N == 0) return PICO_OK;
  Mx8Params p = {static_cast<const uint8_t*>(a->data), static_cast<const uint8_t*>(b->data), static_cast<const uint8_t*>(a->scales), static_cast<const uint8_t*>(b->scales),
                       nullptr, 0, c, (int)M, (int)N, (int)K, parts};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (tile_m == 0) {
    if (tile_n < 0 || tile_n >= kForms) return fail(PICO_ERR_SHAPE, "%s: no form %d of the kernel of few rows", fn, tile_n);
    if (parts < 1 || parts > 64 || (parts > 1 && (!kFew[tile_n].parts || (K + 127) / 128 < parts)))
      return fail(PICO_ERR_SHAPE, "%s: K=%lld in %d pieces by form %d of the kernel of few rows (a step of 128 a piece at least)", fn, (long long)K, parts, tile_n);
  } else if (!large_takes(M, N, K, parts)) {
    return fail(PICO_ERR_SHAPE, "%s: M=%lld N=%lld K=%lld in %d pieces (two steps of 128 a piece at least)", fn, (long long)M, (long long)N, (long long)K, parts);
  }
  if (parts > 1) {
    if (!workspace || workspace_bytes < parts_bytes(M, N, parts))
      return fail(PICO_ERR_WORKSPACE, "%s: the workspace has %lld bytes, needs %lld", fn, (long long)workspace_bytes, (long long)parts_bytes(M, N, parts));
    if (!aligned16(workspace)) return fail(PICO_ERR_ALIGN, "%s: the workspace must be 16-byte aligned", fn);
    p.c = workspace;
  }
  int rc;
  if (tile_m == 0) rc = dispatch_few<false>(p, tile_n, s, std::make_integer_sequence<int, kForms>());
  else rc = parts > 1 ? launch_shape<true>(p, workspace, tile_m, tile_n, per_cu, parts, s) : launch_shape<false>(p, c, tile_m, tile_n, per_cu, 1, s);
  if (rc || parts == 1) return rc;
  return pico_sum_parts(static_cast<const float*>(workspace), c, parts, M * ((N + 7) / 8 * 8), PICO_BF16, stream);
}

extern "C" int pico_mx8_product(const pico_mx8* a, const pico_mx8* b, void* c, int64_t M, int64_t N, int64_t K, void* workspace, int64_t workspace_bytes, void* stream) {
  if (int rc = check_product("pico_mx8_product", a, b, c, M, N, K)) return rc;
  if (M == 0 || N == 0) return PICO_OK;
  float us;
  const Route r = route(M, N, K, us);
  return pico_mx8_product_tiled(a, b, c, M, N, K, r.tile_m, r.tile_n, r.per_cu, r.parts, workspace, workspace_bytes, stream);
}

namespace {
// The form in which a's rounding costs less than a launch of its own, or -1.  It adds in the order of the form that pico_mx8_product goes to, so the results are the same to the bit.
int rounding_form(int64_t M, int64_t N, int64_t K) {
  float two;
  const Route r = route(M, N, K, two);
  if (M > 16 || r.tile_m != 0 || r.parts > 1) return -1;
  const FewRoute one = few_route(M, N, K, kFew[r.tile_n].waves);
  return one.us < two + 2.f ? one.form : -1;
}
}  // namespace

extern "C" int pico_mx8_product_rounding_pays(int64_t M, int64_t N, int64_t K) { return M >= 1 && N >= 1 && K >= 1 && rounding_form(M, N, K) >= 0; }

extern "C" int pico_mx8_product_rounding(const void* x, const pico_mx8* b, void* c, int64_t M, int64_t N, int64_t K, int64_t x_ld, void* stream) {
  const char* fn = "pico_mx8_product_rounding";
  const pico_mx8 a = {const_cast<void*>(x), const_cast<void*>(x)};
  if (int rc = check_product(fn, &a, b, c, M, N, K)) return rc;
  if (M == 0 || N == 0) return PICO_OK;
  if (x_ld < K) return fail(PICO_ERR_STRIDE, "%s: x has a row pitch under its columns", fn);
  if (x_ld % 8 != 0) return fail(PICO_ERR_ALIGN, "%s: the row pitch of x must be a multiple of 8", fn);
  Mx8Params p = {nullptr, static_cast<const uint8_t*>(b->data), nullptr, static_cast<const uint8_t*>(b->scales), static_cast<const __bf16*>(x), x_ld, c, (int)M, (int)N, (int)K, 1};
  const int form = rounding_form(M, N, K);
  if (form < 0) return fail(PICO_ERR_SHAPE, "%s: M=%lld N=%lld K=%lld (sizes for which pico_mx8_product_rounding_pays)", fn, (long long)M, (long long)N, (long long)K);
  return dispatch_few<true>(p, form, static_cast<hipStream_t>(stream), std::make_integer_sequence<int, kRoundForms>());
}
