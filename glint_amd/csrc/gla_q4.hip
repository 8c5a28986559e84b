// gla_q4.hip -- projections with 4-bit weights: GGML's Q4_0 (groups of 32 with
// an f16 scale) and Q4_K (groups of 32 with a 6-bit scale and minimum, eight of
// them under an f16 scale of each kind).
//
// Weights are repacked once, on upload, into pieces of 16 rows x 128 columns (a
// row tile and a quad of groups), in the operand order of
// v_mfma_f32_16x16x32_f16: lane l of a wave holds row l % 16, and of each of the
// four groups elements (l / 16) * 8 .. +8 as one dword, so a wave reads a piece
// as one contiguous kilobyte. Element 2i of the eight sits at bits 4i of its
// dword and element 2i + 1 at bits 16 + 4i: two masks give both as halves.
//   quants [tile][quad][64 lanes][4 groups] u32
//   aux    [tile][quad][16 rows] 8 bytes: Q4_0 four f16 scales; Q4_K four scale
//          bytes, then four minimum bytes
//   super  Q4_K: [tile][superblock][16 rows] {f16 d, f16 dmin}
// Groups and rows past the matrix have scale (and minimum) 0.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "gla_internal.h"

struct gla_q4w {
    gla_ctx *ctx = nullptr;
    gla_q4_format format = GLA_Q4_0;
    int rows = 0;
    int cols = 0;
    int n_tiles = 0;  // ceil(rows / 16)
    int n_quads = 0;  // ceil(cols / 128)
    uint8_t *quants = nullptr;
    uint8_t *aux = nullptr;
    uint32_t *super = nullptr;
};

namespace gla {

void detach_q4w(gla_q4w *w) {
    if (w->quants) (void)hipFree(w->quants);
    if (w->aux) (void)hipFree(w->aux);
    if (w->super) (void)hipFree(w->super);
    w->quants = w->aux = nullptr;
    w->super = nullptr;
    w->ctx = nullptr;
}

namespace {

struct Weights {
    const uint8_t *quants;
    const uint8_t *aux;
    const uint32_t *super;
    int rows, cols, n_tiles, n_quads;
};

// ---- repack ----------------------------------------------------------------------

// One thread per (tile, quad, lane): the lane's four dwords and, of lanes 0..15,
// the 8 aux bytes of row tile * 16 + lane and the superblock's word.
template <bool K>
__global__ __launch_bounds__(256) void q4_repack_kernel(const uint8_t *ggml, int rows, int n_groups, int n_quads,
                                                        int64_t n_units, uint8_t *quants, uint8_t *aux,
                                                        uint32_t *super) {
    const int64_t u = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (u >= n_units) return;
    const int lane = (int)(u & 63);
    const int64_t tq = u >> 6;
    const int quad = (int)(tq % n_quads);
    const int tile = (int)(tq / n_quads);
    const int row = tile * 16 + (lane & 15);
    const int k8 = (lane >> 4) * 8;  // first of the lane's elements in a group
    uint32_t w[4];
    uint32_t lo = 0, hi = 0;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int g = quad * 4 + j;
        w[j] = 0;
        if (row >= rows || g >= n_groups) continue;
        const uint8_t *blk;  // the group's nibbles: 16 bytes low then high (Q4_0), 32 bytes low or high (Q4_K)
        if (K)
            blk = ggml + ((int64_t)row * (n_groups / 8) + g / 8) * 144;
        else
            blk = ggml + ((int64_t)row * n_groups + g) * 18;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const int k = k8 + e;
            uint32_t q;
            if (K)
                q = (blk[16 + (g % 8 / 2) * 32 + k] >> (g % 2 * 4)) & 15u;
            else
                q = (blk[2 + k % 16] >> (k / 16 * 4)) & 15u;
            w[j] |= q << (e / 2 * 4 + e % 2 * 16);
        }
        if (K) {
            const uint8_t *b = blk + 4;
            const int i = g % 8;
            const uint32_t sc = i < 4 ? b[i] & 63u : (b[i + 4] & 15u) | (uint32_t)(b[i - 4] >> 6) << 4;
            const uint32_t mn = i < 4 ? b[i + 4] & 63u : (uint32_t)(b[i + 4] >> 4) | (uint32_t)(b[i] >> 6) << 4;
            lo |= sc << (8 * j);
            hi |= mn << (8 * j);
            if (lane < 16 && g % 8 == 0)
                super[((int64_t)tile * (n_quads / 2) + g / 8) * 16 + lane] =
                    blk[0] | (uint32_t)blk[1] << 8 | (uint32_t)blk[2] << 16 | (uint32_t)blk[3] << 24;
        } else {
            const uint32_t d = blk[0] | (uint32_t)blk[1] << 8;
            (j < 2 ? lo : hi) |= d << (j % 2 * 16);
        }
    }
    *reinterpret_cast<uint4 *>(quants + u * 16) = make_uint4(w[0], w[1], w[2], w[3]);
    if (lane < 16) {
        *reinterpret_cast<uint2 *>(aux + (tq * 16 + lane) * 8) = make_uint2(lo, hi);
        if (K && row >= rows && quad % 2 == 0) super[((int64_t)tile * (n_quads / 2) + quad / 2) * 16 + lane] = 0;
    }
}

// ---- operands ----------------------------------------------------------------------

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ half2v h2(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ half2v both(float x) { return half2v{(_Float16)x, (_Float16)x}; }
__device__ __forceinline__ float lo_of(uint32_t w) { return (float)h2(w)[0]; }
__device__ __forceinline__ float hi_of(uint32_t w) { return (float)h2(w)[1]; }

// (u & mask) | 0x64006400 in one instruction, which needs the constant in a register
__device__ __forceinline__ half2v under_1024(uint32_t u, uint32_t mask) {
    uint32_t o, k = 0x64006400u;
    asm("" : "+v"(k));
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(o) : "v"(u), "s"(mask), "v"(k));
    return h2(o);
}
// Q4_0: n - 8 of the 8 nibbles of a dword. A nibble under the bits of 1024 is 1024 + n,
// four bits further up 1024 + 16 n; every result is exact.
__device__ __forceinline__ half8 nibbles_q4_0(uint32_t w) {
    half8 o;
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const uint32_t u = w >> (8 * i);
        const half2v a = under_1024(u, 0x000f000fu) - both(1032.0f);
        const half2v b = __builtin_elementwise_fma(under_1024(u, 0x00f000f0u), both(0.0625f), both(-72.0f));
        o[4 * i] = a[0];
        o[4 * i + 1] = a[1];
        o[4 * i + 2] = b[0];
        o[4 * i + 3] = b[1];
    }
    return o;
}
// An integer up to 2047 as the bits of a half is that many times 2^-24 (subnormals and
// the binade above them), and the MFMA takes it so: Q4_K's A operands are integers, its
// products 2^-24 of their value, which kUnscale takes back. A mask and a product a pair
// of nibbles instead of a mask, a conversion and its constants: 14336 x 4096, 1 vector
// 12.2 -> 10.2 us; 6144 x 4096, 1 vector 6.5 -> 6.1, 1,999 vectors 2% less (194).
constexpr float kUnscale = 0x1p24f;
// Q4_K: n * (scale byte j of sc), at most 15 * 63; one 24-bit product for a pair
__device__ __forceinline__ half8 nibbles_q4_k(uint32_t w, uint32_t sc, int j) {
    uint32_t mask = 0x000f000fu;
    asm("" : "+v"(mask));
    const uint32_t s = (sc >> (8 * j)) & 255u;
    u32x4 o;
#pragma unroll
    for (int i = 0; i < 4; i++) o[i] = __umul24((w >> (4 * i)) & mask, s);
    return __builtin_bit_cast(half8, o);
}
// Q4_K: 32 times the four minimum bytes
__device__ __forceinline__ half4 minima(uint32_t mn) {
    const u32x2 o = {__builtin_amdgcn_perm(0u, mn, 0x0c010c00u) << 5, __builtin_amdgcn_perm(0u, mn, 0x0c030c02u) << 5};
    return __builtin_bit_cast(half4, o);
}

// x enters the products as two halves, hi = f16(x 2^s) and lo = f16(x 2^s - hi),
// s bringing the largest finite |x| of a range into [2^13, 2^14): off by 2^-22 of x
// (half a step of 11 bits, twice) or, where lo is subnormal, by 2^-25 and so 2^-38 of the
// largest. A NaN is both its pieces. An infinity is its own hi piece (lo 0)
// in Q4_0; in Q4_K, where a weight's nibble and minimum multiply x in sums of their own and
// an infinity would end as inf - inf, it is 0 and infinite_terms adds its products.
// The range's largest |x| is kept as bits, which order as the values do.
constexpr uint32_t kInf = 0x7f800000u;
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ int shift_of(uint32_t mx) { return min(140 - (int)(mx >> 23), 120); }
__device__ __forceinline__ float exp2_of(int n) { return __uint_as_float((uint32_t)(n + 127) << 23); }
// the largest of a row of 16 lanes, by rotation
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, true));
    return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, true));
}
// ... of the wave: then rows 0/1 and 2/3, then the halves
__device__ __forceinline__ uint32_t wave_max(uint32_t x) {
    x = row_max(x);
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(b[0], b[1]);
}
// ... of the lanes that are equal mod 4
__device__ __forceinline__ uint32_t wave_max4(uint32_t x) {
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true));
    x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true));
    const auto a = __builtin_amdgcn_permlane16_swap(x, x, false, false);
    x = max(a[0], a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(x, x, false, false);
    return max(b[0], b[1]);
}
// Sums of four neighbouring lanes; of the four lanes of a row that are equal mod 4.
__device__ __forceinline__ float quad_sum(float x) {
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0xB1, 0xf, 0xf, true));
    return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x4E, 0xf, 0xf, true));
}
__device__ __forceinline__ float apart_sum(float x) {
    x += __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x124, 0xf, 0xf, true));
    return x + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), 0x128, 0xf, 0xf, true));
}
// Pieces of x * mul (a power of two); `odd`: the range has an infinity or a NaN.
__device__ __forceinline__ void pieces(float x, float mul, bool odd, _Float16 &hi, _Float16 &lo) {
    hi = (_Float16)(x * mul);
    lo = (_Float16)fmaf(x, mul, -(float)hi);
    if (odd && abs_bits(x) == kInf) lo = (_Float16)0.0f;
}
// Q4_K: x as it enters the pieces and the sums
template <bool K>
__device__ __forceinline__ float without_inf(float x, bool odd) {
    return K && odd && abs_bits(x) == kInf ? 0.0f : x;
}
// 8 floats from byte `at` of a row's `bytes` (wave-uniform), zeros past them: the
// bounds check of the buffer loads, which also take rows at any 4-byte address.
__device__ __forceinline__ void load_row(float (&e)[8], const float *row, int bytes, int at) {
    const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(row), 0, bytes, 0x00027000);
    const u32x4 a = __builtin_amdgcn_raw_buffer_load_b128(r, at, 0, 0), b = __builtin_amdgcn_raw_buffer_load_b128(r, at + 16, 0, 0);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        e[j] = __uint_as_float(a[j]);
        e[4 + j] = __uint_as_float(b[j]);
    }
}

// Q4_K: the products of row `row` with the infinite elements of x, each with the whole
// weight, as the definition has it: an infinity by the weight's sign, NaN for a weight of
// 0 and for infinities of both signs. Only outputs of vectors that hold an infinity come
// here. d * scale * nibble and dmin * minimum are exact in f32, so their difference is 0
// where the weight is. A walk through x by each output's thread: 6144 x 4096, 1 vector 6 ->
// 105 us, 1,999 vectors with an infinity each 0.2 -> 21 ms.
__device__ float infinite_terms(const Weights &w, const float *x, int row) {
    const int64_t tile = row >> 4, r = row & 15;
    float sum = 0.0f;
    for (int c0 = 0; c0 < w.cols && sum == sum; c0 += 8) {  // a NaN stays one
        uint32_t any = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) any |= abs_bits(x[c0 + k]) == kInf ? 1u << k : 0u;
        if (!any) continue;
        const int64_t tq = tile * w.n_quads + (c0 >> 7);
        const int j = (c0 >> 5) & 3;
        const uint32_t q = reinterpret_cast<const uint32_t *>(w.quants)[(tq * 64 + ((c0 >> 3) & 3) * 16 + r) * 4 + j];
        const uint8_t *a = w.aux + (tq * 16 + r) * 8;
        const uint32_t d = w.super[(tile * (w.n_quads / 2) + (c0 >> 8)) * 16 + r];
        const float scale = lo_of(d) * (float)a[j], low = hi_of(d) * (float)a[4 + j];
        for (int k = 0; k < 8; k++)
            if (any >> k & 1) sum += fmaf(scale, (float)((q >> (k / 2 * 4 + k % 2 * 16)) & 15u), -low) * x[c0 + k];
    }
    return sum;
}

// ---- up to 8 vectors ------------------------------------------------------------------

// y[v][row] for up to NV vectors, RT row tiles a workgroup. The eight waves split
// K; a wave takes its quads CH at a time (a chunk; four, or one where that is all
// there is, four vectors side by side then): its lanes load 8 elements of each
// vector, find the chunk's largest |x| of each vector, and put the pieces into the
// wave's LDS in the order of the B operand, whose 16 columns are the hi pieces of the
// vectors and then their lo pieces: one MFMA multiplies 16 rows x 32 columns of
// weights with all of them. No wave waits for another until the sums are merged.
//   Q4_0: a group's product times its rows' scales goes into the sum (C = A B is
//   16 rows x 16 columns, lane (column l % 16, rows l / 16 * 4 + r)).
//   Q4_K: A holds nibble * scale, exact, so a quad's four groups add up in the
//   MFMA; the rows' d multiplies once a quad. The minima are a product of their
//   own: four minima of a row with the sums of x over the four groups (in pieces,
//   scaled by 2^-5; the minima carry 2^5).
// Columns past the vectors multiply what the first ones do, and their sums are not used:
// zeros there cost 16 instructions a quad. A chunk's weights are loaded for CH quads
// whether or not the wave has so many: where columns are no multiple of 4,096 a wave
// loads some of the next one's as well.
// Bound: one chain of launch (2.7 us), loads from HBM, unpacking and the merge; the
// vector unit is busy a third of it (about 85 instructions for 16 rows x 128 columns of
// Q4_0, 100 of Q4_K). us: Q4_0 4096 x 4096, 1 / 2 / 4 / 8 vectors 4.3 / 4.6 / 5.5 / 7.2;
// 4096 x 2048, 1 / 4 3.9 / 4.8; 5120 x 5120 8.0 / 9.9; 49152 x 576 15.8 / 23.8;
// 14336 x 4096, 1 vector 10.9, Q4_K 10.3 (33 MB, 3.2 TB/s).
constexpr int kFewWaves = 8;
template <bool K, int NV, int RT, int CH>
__global__ __launch_bounds__(kFewWaves * 64) void matvec_q4_few_kernel(const Weights w, const float *x, int n_vec, float *y) {
    constexpr int COLS = 2 * NV;
    constexpr int LANES = 16 * CH;                // of a vector's chunk, 8 elements each
    constexpr int VP = 64 / LANES;                // vectors at a time
    constexpr int NI = (NV + VP - 1) / VP;
    constexpr int PITCH = LANES + 1;              // half8 from column to column: [group][kg], and one for the banks
    constexpr int PIECES = COLS * PITCH;          // of a wave's chunk
    constexpr int SUMS = K ? CH * COLS : 0;       // half4: [quad][column]
    constexpr int WAVE = (PIECES * 16 + SUMS * 8 + NV * 4 + 15) / 16 * 16;
    constexpr int RED = kFewWaves * RT * 64 * 16;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kFewWaves * WAVE > RED ? kFewWaves * WAVE : RED];
    __shared__ uint32_t inf_of[K ? kFewWaves : 1];  // Q4_K: bit v, the wave's columns of vector v may hold an infinity
    uint32_t inf = 0;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, kg = lane >> 4;
    const int vg = lane / LANES, vl = lane % LANES;  // the vector of a pass, and the lane's eight of its chunk
    half8 *px = reinterpret_cast<half8 *>(lds + wave * WAVE);
    half4 *ps = reinterpret_cast<half4 *>(lds + wave * WAVE + PIECES * 16);
    float *pu = reinterpret_cast<float *>(lds + wave * WAVE + PIECES * 16 + SUMS * 8);
    constexpr int UNIT = K ? 2 : 1;  // whole superblocks a wave
    const int per = (w.n_quads / UNIT + kFewWaves - 1) / kFewWaves * UNIT;
    const int q0 = min(w.n_quads, wave * per), q1 = min(w.n_quads, q0 + per);
    const int tile0 = blockIdx.x * RT;

    floatx4 total[RT];
#pragma unroll
    for (int t = 0; t < RT; t++) total[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int c0 = q0; c0 < q1; c0 += CH) {
        // x first: loads return in order, so the pieces do not wait for weights
        float e[NI][8];
        const int bytes = (min(w.cols, q1 * 128) - c0 * 128) * 4;  // of the wave's columns from here on
#pragma unroll
        for (int i = 0; i < NI; i++) {
            if constexpr (VP == 1) {
                load_row(e[i], x + (int64_t)min(i, n_vec - 1) * w.cols + c0 * 128, i < n_vec ? bytes : 0, lane * 32);
            } else {
                const int v = i * VP + vg;
                const bool in = v < n_vec && vl * 32 < bytes;
                load_row(e[i], x + c0 * 128, ((n_vec - 1) * w.cols + w.cols - c0 * 128) * 4, in ? v * w.cols * 4 + vl * 32 : -32);
            }
        }
        u32x4 qw[RT][CH];
        u32x4 sc[RT][CH][2];            // Q4_0: the 32 bytes of rows kg * 4 .. +3
        u32x2 am[RT][CH];               // Q4_K: the lane's row's scales and minima
        u32x4 sup[RT][(CH + 1) / 2];    // Q4_K: d and dmin of rows kg * 4 .. +3
#pragma unroll
        for (int i = 0; i < CH; i++)
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int64_t tile = min(tile0 + t, w.n_tiles - 1);
                const int64_t tq = tile * w.n_quads + min(c0 + i, w.n_quads - 1);
                qw[t][i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(w.quants + (tq * 64 + lane) * 16));
                if constexpr (K) {
                    am[t][i] = *reinterpret_cast<const u32x2 *>(w.aux + (tq * 16 + col) * 8);
                    if (i % 2 == 0) {
                        const int sb = min((c0 >> 1) + i / 2, w.n_quads / 2 - 1);
                        sup[t][i >> 1] = *reinterpret_cast<const u32x4 *>(w.super + (tile * (w.n_quads / 2) + sb) * 16 + kg * 4);
                    }
                } else {
                    const u32x4 *s = reinterpret_cast<const u32x4 *>(w.aux + (tq * 16 + kg * 4) * 8);
                    sc[t][i][0] = s[0];
                    sc[t][i][1] = s[1];
                }
            }
        uint32_t mx[NI];
#pragma unroll
        for (int i = 0; i < NI; i++) {
            mx[i] = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) mx[i] = max(mx[i], abs_bits(e[i][j]));
            mx[i] = VP == 1 ? wave_max(mx[i]) : row_max(mx[i]);
        }
#pragma unroll
        for (int i = 0; i < NI; i++) {
            uint32_t top = VP == 1 ? __builtin_amdgcn_readfirstlane(mx[i]) : mx[i];
            const bool odd = VP == 1 ? top >= kInf : __any(top >= kInf);
            if (odd) {  // scaled by what is finite
                inf |= ((1u << VP) - 1) << (i * VP);
                mx[i] = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) mx[i] = max(mx[i], abs_bits(e[i][j]) < kInf ? abs_bits(e[i][j]) : 0);
                top = VP == 1 ? __builtin_amdgcn_readfirstlane(wave_max(mx[i])) : row_max(mx[i]);
            }
            const int sh = shift_of(top);
            const float mul = exp2_of(sh);
            half8 hi, lo;
            float sum = 0.0f;
            const auto split = [&](bool odd) {
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float t = without_inf<K>(e[i][j], odd);
                    _Float16 a, b;
                    pieces(t, mul, odd, a, b);
                    hi[j] = a;
                    lo[j] = b;
                    sum = fmaf(t, mul, sum);
                }
            };
            if (odd)
                split(true);
            else
                split(false);
            const int v = i * VP + vg;
            if (v >= NV) continue;  // (more lanes than vectors)
            if (vl == 0) pu[v] = exp2_of(-sh);
            px[v * PITCH + vl] = hi;  // vl = group * 4 + kg of the chunk
            px[(NV + v) * PITCH + vl] = lo;
            if constexpr (K) {
                _Float16 a, b;
                pieces(quad_sum(sum), 0.03125f, false, a, b);
                if ((vl & 3) == 0) {
                    _Float16 *to = reinterpret_cast<_Float16 *>(ps + (vl >> 4) * COLS) + ((vl >> 2) & 3);
                    to[v * 4] = a;
                    to[(NV + v) * 4] = b;
                }
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        const float undo = pu[col % NV];  // 2^-s of the lane's column (of the first 2 NV)
        floatx4 acc[RT];
#pragma unroll
        for (int t = 0; t < RT; t++) acc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < CH; i++) {
            if (c0 + i >= q1) break;
            half8 bx[4];
#pragma unroll
            for (int j = 0; j < 4; j++) bx[j] = px[col % COLS * PITCH + (i * 4 + j) * 4 + kg];
            if constexpr (K) {
                const half4 bs = ps[i * COLS + col % COLS];
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    floatx4 c = zero;
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        c = __builtin_amdgcn_mfma_f32_16x16x32_f16(nibbles_q4_k(qw[t][i][j], am[t][i][0], j), bx[j], c, 0, 0, 0);
                    half4 mn = minima(am[t][i][1]);
                    if (kg) mn = half4{};
                    const floatx4 m = __builtin_amdgcn_mfma_f32_16x16x16f16(mn, bs, zero, 0, 0, 0);
                    const u32x4 dd = sup[t][i >> 1];
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        acc[t][r] = fmaf(c[r], lo_of(dd[r]), acc[t][r]);
                        acc[t][r] = fmaf(-m[r], hi_of(dd[r]), acc[t][r]);
                    }
                }
            } else {
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    floatx4 c[4];
#pragma unroll
                    for (int j = 0; j < 4; j++)
                        c[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(nibbles_q4_0(qw[t][i][j]), bx[j], zero, 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 4; j++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const uint32_t s = sc[t][i][r >> 1][(r & 1) * 2 + (j >> 1)];
                            acc[t][r] = fmaf(c[j][r], (j & 1) ? hi_of(s) : lo_of(s), acc[t][r]);
                        }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < RT; t++) total[t] += (K ? acc[t] * kUnscale : acc[t]) * undo;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // the pieces are read before the next chunk's are written
        __builtin_amdgcn_wave_barrier();
    }

    // the waves in order, the hi and then the lo column of a vector
    __syncthreads();
    floatx4 *red = reinterpret_cast<floatx4 *>(lds);
#pragma unroll
    for (int t = 0; t < RT; t++) red[(wave * RT + t) * 64 + lane] = total[t];
    if (K && lane == 0) inf_of[wave] = inf;
    __syncthreads();
    for (int i = threadIdx.x; i < RT * 16 * NV; i += kFewWaves * 64) {
        const int rr = i & 15, t = (i >> 4) % RT, v = (i >> 4) / RT;
        const float *f = reinterpret_cast<const float *>(red) + (t * 64 + (rr >> 2) * 16) * 4 + (rr & 3);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kFewWaves; k++) sum += f[k * RT * 256 + v * 4] + f[k * RT * 256 + (NV + v) * 4];
        const int row = (tile0 + t) * 16 + rr;
        if (v < n_vec && row < w.rows) y[(int64_t)v * w.rows + row] = sum;
    }
    if constexpr (K) {
        for (int k = 0; k < kFewWaves; k++) inf |= inf_of[k];
        if (inf)  // the thread's own outputs again
            for (int i = threadIdx.x; i < RT * 16 * NV; i += kFewWaves * 64) {
                const int row = (tile0 + (i >> 4) % RT) * 16 + (i & 15), v = (i >> 4) / RT;
                if (v < n_vec && row < w.rows && (inf >> v & 1))
                    y[(int64_t)v * w.rows + row] += infinite_terms(w, x + (int64_t)v * w.cols, row);
            }
    }
}

// ---- more vectors: the pieces of x, once per call ----------------------------------

// A workgroup per VQ vectors (thread t: vector t % VQ): their scales from the largest
// finite |x| of a row, then the pieces in B-operand order, xp[v / 16][group][piece]
// [lane = kg * 16 + v % 16] = 8 halves, zeros past the columns, and undo[v] = 2^-s.
// Q4_K: the sums of each group, times 2^-5 and in pieces, xm[v / 16][superblock][piece]
// [v % 16] = the eight groups' halves, and undo[v] < 0 of a vector that holds an infinity
// and no NaN. Vectors up to the next 16 are left as they are:
// a column of the product is its vector's alone. Many vectors go four a workgroup, so
// that 64 bytes are written together (1,999 x 4,096: 29 us at one, whose 16-byte
// pieces met in memory). Up to 64 take a workgroup each, for the chip's sake, twice:
// both find the scale, each writes every other of the thread's units (4,096 columns, 16
// vectors with their product 12.1 -> 11.4 us; 576 8.1 -> 6.5).
constexpr int kSplitThreads = 512;
constexpr int kSplitUnits = 4;  // units of 8 elements a thread keeps; a wider row is read twice
template <bool K, int VQ>
__global__ __launch_bounds__(kSplitThreads) void split_q4_kernel(const float *x, int n_vec, int cols, int n_quads,
                                                                 _Float16 *xp, _Float16 *xm, float *undo) {
    constexpr int PASS = kSplitThreads / VQ;  // units of a vector a pass
    const int t = threadIdx.x, vq = t % VQ, ut = t / VQ;
    const int v = blockIdx.x * VQ + vq;
    const int units = n_quads * 16, in = cols / 8;
    float e[kSplitUnits][8];
    const float *row = x + (int64_t)min(v, n_vec - 1) * cols;
    const bool aligned = ((uintptr_t)x & 15) == 0;  // rows are 128-byte multiples apart
    const auto fetch = [&](float (&d)[8], int u) {
        const float *p = row + (int64_t)min(u, in - 1) * 8;
        if (aligned) {
            const floatx4 a = reinterpret_cast<const floatx4 *>(p)[0], b = reinterpret_cast<const floatx4 *>(p)[1];
#pragma unroll
            for (int j = 0; j < 4; j++) d[j] = a[j], d[4 + j] = b[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) d[j] = p[j];
        }
        if (u >= in)
#pragma unroll
            for (int j = 0; j < 8; j++) d[j] = 0.0f;
    };
    const auto bits_of = [](const float (&d)[8], bool finite) {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const uint32_t a = abs_bits(d[j]);
            m = max(m, finite && a >= kInf ? 0u : a);
        }
        return m;
    };
    __shared__ uint32_t red[2][kSplitThreads / 64][VQ];
    const auto group_max = [&](bool finite, int at) {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < kSplitUnits; i++) m = max(m, bits_of(e[i], finite));
        for (int u = kSplitUnits * PASS + ut; u < in; u += PASS) {
            float d[8];
            fetch(d, u);
            m = max(m, bits_of(d, finite));
        }
        m = VQ == 1 ? wave_max(m) : wave_max4(m);
        if ((t & 63) < VQ) red[at][t >> 6][vq] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kSplitThreads / 64; i++) m = max(m, red[at][i][vq]);
        return m;
    };
#pragma unroll
    for (int i = 0; i < kSplitUnits; i++) fetch(e[i], i * PASS + ut);
    uint32_t top = group_max(false, 0);
    const bool odd = top >= kInf, inf = top == kInf;
    if (__syncthreads_or(odd)) {
        const uint32_t fin = group_max(true, 1);
        if (odd) top = fin;
    }
    const int sh = shift_of(top);
    const float mul = exp2_of(sh);
    if (v >= n_vec) return;
    if (ut == 0) undo[v] = K && inf ? -exp2_of(-sh) : exp2_of(-sh);
    const auto put = [&](const float (&d)[8], int u) {
        half8 hi, lo;
        float sum = 0.0f;
        const auto split = [&](bool odd) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float t = without_inf<K>(d[j], odd);
                _Float16 a, b;
                pieces(t, mul, odd, a, b);
                hi[j] = a;
                lo[j] = b;
                sum = fmaf(t, mul, sum);
            }
        };
        if (odd)
            split(true);
        else
            split(false);
        _Float16 *to = xp + (((int64_t)(v >> 4) * n_quads * 4 + (u >> 2)) * 128 + (u & 3) * 16 + (v & 15)) * 8;
        *reinterpret_cast<half8 *>(to) = hi;
        *reinterpret_cast<half8 *>(to + 512) = lo;
        if constexpr (K) {
            _Float16 a, b;
            // units of a group are four threads, neighbours or VQ apart
            pieces(VQ == 1 ? quad_sum(sum) : apart_sum(sum), 0.03125f, false, a, b);
            if ((u & 3) == 0) {
                _Float16 *m = xm + (((int64_t)(v >> 4) * (n_quads / 2) + (u >> 5)) * 32 + (v & 15)) * 8 + ((u >> 2) & 7);
                m[0] = a;
                m[128] = b;
            }
        }
    };
    const int seg = blockIdx.y, segs = gridDim.y;
#pragma unroll
    for (int i = 0; i < kSplitUnits; i++)
        if (i % segs == seg && i * PASS + ut < units) put(e[i], i * PASS + ut);
    for (int i = kSplitUnits + seg; i * PASS + ut < units; i += segs) {
        const int u = i * PASS + ut;
        float d[8];
        fetch(d, u);
        put(d, u);
    }
}

struct Pieces {
    const _Float16 *xp;
    const _Float16 *xm;
    const float *undo;
    const float *x;  // the vectors themselves, for the infinities among them
};

// ---- some vectors -------------------------------------------------------------------

constexpr int kMidWaves = 8;

// y[v][row] for RT row tiles x up to 16 NVT VH vectors a workgroup: the eight waves
// are VH ranges of vectors x 8 / VH ranges of K. Every fragment of x that a wave reads
// serves RT row tiles, every fragment of weights NVT vector tiles; x comes D groups
// ahead, the weights a quad ahead, and the waves are merged in LDS in order. Bound: a
// short wave's latencies (launch, the first weights, the merge: 10 of 16.7 us at 4096 x
// 4096 and 64 vectors), then the vector unit, whose 11 instructions to unpack a dword
// of nibbles serve NVT tiles. Workgroups for other vectors read the same weights again
// from L2, which costs less than slices of K that have to be joined through memory
// (64 vectors, Q4_0 4096 x 4096 19.4 -> 16.7 us, 1024 x 4096 17.4 -> 11.9, Q4_K 6144 x
// 4096 25.5 -> 20.8).
template <bool K, int NVT, int RT, int VH>
__global__ __launch_bounds__(kMidWaves * 64) void matvec_q4_mid_kernel(const Weights w, const Pieces px, int n_vec, float *y) {
    constexpr int UNIT = K ? 2 : 1, D = NVT * RT <= 4 && NVT <= 2 ? 4 : 2, KW = kMidWaves / VH;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, kg = lane >> 4;
    const int tile0 = blockIdx.x * RT;
    const int vb = blockIdx.y * (NVT * VH), vt0 = wave / KW * NVT, last_vt = (n_vec - 1) >> 4;
    const int units = w.n_quads / UNIT;
    const int per = (units + KW - 1) / KW;
    const int q0 = min(units, wave % KW * per) * UNIT, q1 = min(units, (wave % KW + 1) * per) * UNIT;
    const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};

    floatx4 acc[RT][NVT];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int v = 0; v < NVT; v++) acc[t][v] = zero;

    half8 bh[D][NVT], bl[D][NVT];
    const auto load_x = [&](half8 (&h)[NVT], half8 (&l)[NVT], int group) {
#pragma unroll
        for (int v = 0; v < NVT; v++) {
            const _Float16 *src = px.xp + (((int64_t)min(vb + vt0 + v, last_vt) * w.n_quads * 4 + group) * 128 + lane) * 8;
            h[v] = *reinterpret_cast<const half8 *>(src);
            l[v] = *reinterpret_cast<const half8 *>(src + 512);
        }
    };
    // sc: Q4_0 the 32 bytes of the C rows' scales; Q4_K [0] the A row's scales and
    // minima, [1] the C rows' d and dmin. bm: Q4_K the sums of x.
    u32x4 qw[RT], sc[RT][2];
    half8 bm[NVT];
    const auto load_w = [&](u32x4 (&q)[RT], u32x4 (&s)[RT][2], half8 (&m)[NVT], int quad) {
#pragma unroll
        for (int t = 0; t < RT; t++) {
            const int64_t tile = min(tile0 + t, w.n_tiles - 1);
            const int64_t tq = tile * w.n_quads + quad;
            q[t] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(w.quants + (tq * 64 + lane) * 16));
            if constexpr (K) {
                const u32x2 a = *reinterpret_cast<const u32x2 *>(w.aux + (tq * 16 + col) * 8);
                s[t][0] = u32x4{a[0], a[1], 0, 0};
                s[t][1] = *reinterpret_cast<const u32x4 *>(w.super + (tile * (w.n_quads / 2) + (quad >> 1)) * 16 + kg * 4);
            } else {
                const u32x4 *p = reinterpret_cast<const u32x4 *>(w.aux + (tq * 16 + kg * 4) * 8);
                s[t][0] = p[0];
                s[t][1] = p[1];
            }
        }
        if constexpr (K)
#pragma unroll
            for (int v = 0; v < NVT; v++)
                m[v] = *reinterpret_cast<const half8 *>(
                    px.xm + (((int64_t)min(vb + vt0 + v, last_vt) * (w.n_quads / 2) + (quad >> 1)) * 32 + (kg & 1) * 16 + col) * 8);
    };
    if (q0 < q1) {
        load_w(qw, sc, bm, q0);
#pragma unroll
        for (int i = 0; i < D; i++) load_x(bh[i], bl[i], q0 * 4 + i);
        __builtin_amdgcn_sched_barrier(0);
        for (int q = q0; q < q1; q++) {
            u32x4 qn[RT], sn[RT][2];
            half8 mn[NVT];
            load_w(qn, sn, mn, min(q + 1, q1 - 1));
            __builtin_amdgcn_sched_barrier(0);
            floatx4 c[RT][NVT];
#pragma unroll
            for (int j = 0; j < 4; j++) {
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    const half8 a = K ? nibbles_q4_k(qw[t][j], sc[t][0][0], j) : nibbles_q4_0(qw[t][j]);
#pragma unroll
                    for (int v = 0; v < NVT; v++)
                        c[t][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh[j % D][v], K && j ? c[t][v] : zero, 0, 0, 0);
#pragma unroll
                    for (int v = 0; v < NVT; v++)
                        c[t][v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl[j % D][v], c[t][v], 0, 0, 0);
                    if constexpr (!K)
#pragma unroll
                        for (int v = 0; v < NVT; v++)
#pragma unroll
                            for (int r = 0; r < 4; r++) {
                                const uint32_t s = sc[t][r >> 1][(r & 1) * 2 + (j >> 1)];
                                acc[t][v][r] = fmaf(c[t][v][r], (j & 1) ? hi_of(s) : lo_of(s), acc[t][v][r]);
                            }
                }
                load_x(bh[j % D], bl[j % D], min(q * 4 + j + D, q1 * 4 - 1));
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (K)
#pragma unroll
                for (int t = 0; t < RT; t++) {
                    // k = 0..7 this quad's minima, zeros at the other's places, with the sums'
                    // hi pieces, 8..15 with their lo ones; the other lanes zeros
                    const half4 m4 = minima(sc[t][0][1]);
                    const half8 am = kg > 1  ? half8{}
                                     : q & 1 ? half8{0, 0, 0, 0, m4[0], m4[1], m4[2], m4[3]}
                                             : half8{m4[0], m4[1], m4[2], m4[3], 0, 0, 0, 0};
#pragma unroll
                    for (int v = 0; v < NVT; v++) {
                        const floatx4 m = __builtin_amdgcn_mfma_f32_16x16x32_f16(am, kg > 1 ? half8{} : bm[v], zero, 0, 0, 0);
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            acc[t][v][r] = fmaf(c[t][v][r], lo_of(sc[t][1][r]), acc[t][v][r]);
                            acc[t][v][r] = fmaf(-m[r], hi_of(sc[t][1][r]), acc[t][v][r]);
                        }
                    }
                }
#pragma unroll
            for (int t = 0; t < RT; t++) qw[t] = qn[t], sc[t][0] = sn[t][0], sc[t][1] = sn[t][1];
#pragma unroll
            for (int v = 0; v < NVT; v++) bm[v] = mn[v];
        }
    }

    // merge the waves through LDS, in order: 4 floats after every 16 lanes, so that
    // a wave's reads of 16 rows x 4 vectors fall in distinct banks
    constexpr int S = 272, VT = NVT * VH;
    __shared__ __attribute__((aligned(16))) float red[KW * RT * VT * S];
    const auto at = [&](int kw, int t, int v, int ln) { return ((kw * RT + t) * VT + v) * S + 4 * ln + 4 * (ln >> 4); };
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int v = 0; v < NVT; v++) *reinterpret_cast<floatx4 *>(&red[at(wave % KW, t, vt0 + v, lane)]) = acc[t][v];
    __syncthreads();
    bool inf = false;  // Q4_K: of a vector with an infinity
    for (int i = threadIdx.x; i < RT * 16 * VT * 16; i += kMidWaves * 64) {
        const int rl = i % (RT * 16), vl = i / (RT * 16);  // consecutive threads, consecutive rows
        const int from = at(0, rl >> 4, vl >> 4, ((rl & 15) >> 2) * 16 + (vl & 15)) + (rl & 3);
        float sum = red[from];
#pragma unroll
        for (int k = 1; k < KW; k++) sum += red[from + k * RT * VT * S];
        const int row = tile0 * 16 + rl, v = vb * 16 + vl;
        if (row < w.rows && v < n_vec) {
            const float undo = px.undo[v];
            y[(int64_t)v * w.rows + row] = K ? sum * kUnscale * fabsf(undo) : sum * undo;
            inf |= K && undo < 0;
        }
    }
    if (inf)  // the thread's own outputs again
        for (int i = threadIdx.x; i < RT * 16 * VT * 16; i += kMidWaves * 64) {
            const int row = tile0 * 16 + i % (RT * 16), v = vb * 16 + i / (RT * 16);
            if (row < w.rows && v < n_vec && px.undo[v] < 0)
                y[(int64_t)v * w.rows + row] += infinite_terms(w, px.x + (int64_t)v * w.cols, row);
        }
}

// ---- many vectors ----------------------------------------------------------------------

__device__ __forceinline__ floatx4 load_agent4(const float *p) {
    uint64_t *q = reinterpret_cast<uint64_t *>(const_cast<float *>(p));
    const uint64_t a = __hip_atomic_load(q, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const uint64_t b = __hip_atomic_load(q + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    return floatx4{__uint_as_float((uint32_t)a), __uint_as_float((uint32_t)(a >> 32)), __uint_as_float((uint32_t)b),
                   __uint_as_float((uint32_t)(b >> 32))};
}

__device__ __forceinline__ void store_agent2(float *p, float a, float b) {
    __hip_atomic_store(reinterpret_cast<uint64_t *>(p), (uint64_t)__float_as_uint(b) << 32 | __float_as_uint(a),
                       __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// y[v][row] for 128 rows x 32 VT vectors a workgroup, and one of `slices` (one or two) slices
// of K, slice0 + blockIdx.z: two workgroups of one launch, whose last to arrive adds the
// slices, or two launches, whose second adds to y (undo and kUnscale are powers of two: the
// same bits). Four waves of 4 row tiles x VT vector tiles, 2 x 2 of them, which share weights
// and pieces of x through LDS. A step is a group of 32 columns: the pieces come by
// LDS copies two steps ahead into a ring of three, the weights of a quad of groups
// (with scales, and for Q4_K the sums of x) during the quad before, each wave issuing
// the same number of copies at the same step, so that the waits can count them. The
// copies of steps past the end repeat the last ones. Bound: matrix and vector issue;
// the scales of a row tile's products are applied, and the next tile's nibbles
// unpacked, between the MFMAs of this one.
template <bool K, int VT>
__global__ __launch_bounds__(256, 2) void matvec_q4_gemm_kernel(const Weights w, const Pieces px, int n_vec, float *y,
                                                                int slices, int slice0, float *part, int64_t slice_stride,
                                                                int32_t *arrivals) {
    constexpr int RT = 4, UNIT = K ? 2 : 1;
    constexpr int XS = 2 * VT * 2048;  // a ring slot of x: the pieces of 2 VT tiles
    constexpr int AUX = 2 * RT * 1024, SUP = AUX + 1024, XM = SUP + 1024, WS = K ? XM + 4096 : SUP;
    constexpr int RING = VT == 2 && !K ? 4 : 3;
    __shared__ __attribute__((aligned(16))) uint8_t lds[RING * XS + 2 * WS];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, kg = lane >> 4;
    const int tile_wg = blockIdx.x * 2 * RT, vt_wg = blockIdx.y * 2 * VT;
    const int rt0 = (wave & 1) * RT, vt0 = (wave >> 1) * VT;
    const int last_tile = w.n_tiles - 1, last_vt = (n_vec - 1) >> 4;
    const uint32_t base = __builtin_amdgcn_readfirstlane(
        (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) void *)&lds[0]);

    const int units = w.n_quads / UNIT;
    const int ps = (units + slices - 1) / slices, slice = slice0 + (int)blockIdx.z;
    const int q0 = min(units, slice * ps) * UNIT, q1 = min(units, (slice + 1) * ps) * UNIT;

    // the wave's copies: VT of 2 VT x 2 pieces, two row tiles and their scales, and
    // (Q4_K, a superblock at a time) the sums of VT / 2 vector tiles
    const uint8_t *xsrc[VT];
#pragma unroll
    for (int c = 0; c < VT; c++) {
        const int i = wave * VT + c;
        xsrc[c] = reinterpret_cast<const uint8_t *>(px.xp) +
                  (int64_t)min(vt_wg + (i >> 1), last_vt) * w.n_quads * 8192 + (i & 1) * 1024;
    }
    const int ta = min(tile_wg + 2 * wave, last_tile), tb = min(ta + 1, last_tile);
    const uint8_t *qa = w.quants + (int64_t)ta * w.n_quads * 1024, *qb = w.quants + (int64_t)tb * w.n_quads * 1024;
    const uint8_t *as = w.aux + (int64_t)ta * w.n_quads * 128;
    const uint32_t aoff = (uint32_t)((lane >> 5) * (tb - ta)) * (uint32_t)w.n_quads * 128 + (lane & 31) * 4;
    const uint8_t *ss = reinterpret_cast<const uint8_t *>(w.super) + (int64_t)ta * (w.n_quads / 2) * 64;
    const uint32_t soff = (uint32_t)(((lane >> 4) & 1) * (tb - ta)) * (uint32_t)(w.n_quads / 2) * 64 + (lane & 15) * 4;
    const int va = min(vt_wg + wave * (VT / 2), last_vt), vb = min(va + 1, last_vt);
    const uint8_t *ms = reinterpret_cast<const uint8_t *>(px.xm) + (int64_t)va * (w.n_quads / 2) * 512;
    const uint32_t moff = (VT == 4 ? (uint32_t)((lane >> 5) * (vb - va)) * (uint32_t)(w.n_quads / 2) * 512 : 0u) + (lane & 31) * 16;
    const auto copy_x = [&](int s, int slot) {
#pragma unroll
        for (int c = 0; c < VT; c++) lds_copy16(xsrc[c] + (int64_t)s * 2048, lane * 16, base + slot * XS + (wave * VT + c) * 1024);
    };
    const auto copy_w = [&](int as_quad, int q, int j) {  // part j of quad q's weights, where quad as_quad's go
        const uint32_t to = base + RING * XS + (as_quad & 1) * WS;
        if (j == 0) {
            lds_copy16(qa + (int64_t)q * 1024, lane * 16, to + 2 * wave * 1024);
            if (K) lds_copy16(ms + (int64_t)(q >> 1) * 512, moff, to + XM + wave * 1024);
        } else if (j == 1) {
            lds_copy16(qb + (int64_t)q * 1024, lane * 16, to + (2 * wave + 1) * 1024);
        } else if (j == 2) {
            lds_copy4(as + (int64_t)q * 128, aoff, to + AUX + wave * 256);
            if (K) lds_copy4(ss + (int64_t)(q >> 1) * 64, soff, to + SUP + wave * 256);
        }
    };

    const floatx4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
    floatx4 acc[RT][VT];
#pragma unroll
    for (int t = 0; t < RT; t++)
#pragma unroll
        for (int v = 0; v < VT; v++) acc[t][v] = zero;

    if (q0 < q1) {
        const int s_last = q1 * 4 - 1;
#pragma unroll
        for (int j = 0; j < 3; j++) copy_w(q0, q0, j);
        copy_x(q0 * 4, 0);
#pragma unroll
        for (int i = 1; i < RING - 1; i++) copy_x(q0 * 4 + i, i);  // a quad has four groups
        int slot = 0;           // of the step
        for (int q = q0; q < q1; q += UNIT) {
            floatx4 c[K ? RT : 2][VT];  // Q4_0: this tile's products and the last one's
            uint32_t mins[RT];          // Q4_K: the first quad's minima
#pragma unroll
            for (int h = 0; h < UNIT; h++) {
                const uint8_t *ws = lds + RING * XS + ((q + h) & 1) * WS;
                u32x4 qw[RT], sc[RT][2];
                u32x2 am[RT];
                const auto unpack = [&](int t, int j) { return K ? nibbles_q4_k(qw[t][j], am[t][0], j) : nibbles_q4_0(qw[t][j]); };
                const auto scale = [&](int t, int j) {  // Q4_0: the products of tile t, group j
#pragma unroll
                    for (int v = 0; v < VT; v++)
#pragma unroll
                        for (int r = 0; r < 4; r++) {
                            const uint32_t f = sc[t][r >> 1][(r & 1) * 2 + (j >> 1)];
                            acc[t][v][r] = fmaf(c[t & 1][v][r], (j & 1) ? hi_of(f) : lo_of(f), acc[t][v][r]);
                        }
                };
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    // step s's x has landed once only the copies of the step before are in
                    // flight; every wave is past step s - 1, whose slot is free
                    if (j == 0)
                        wait_vm<VT>();
                    else if (j == 1)
                        wait_vm<(RING == 4 ? VT : 0) + VT + 1 + K>();
                    else if (j == 2)
                        wait_vm<(RING == 4 ? VT + 1 + K : 0) + VT + 1>();
                    else
                        wait_vm<(RING == 4 ? VT + 1 : 0) + VT + 1 + K>();
                    __syncthreads();
                    const int qn = min(q + h + 1, q1 - 1);
                    copy_x(min((q + h) * 4 + j + RING - 1, s_last), slot == 0 ? RING - 1 : slot - 1);
                    copy_w(q + h + 1, qn, j);
                    const uint8_t *xl = lds + slot * XS + vt0 * 2048 + lane * 16;
                    slot = slot == RING - 1 ? 0 : slot + 1;
                    if (j == 0) {
#pragma unroll
                        for (int t = 0; t < RT; t++) {
                            const int i = rt0 + t;
                            qw[t] = *reinterpret_cast<const u32x4 *>(ws + i * 1024 + lane * 16);
                            const uint8_t *a = ws + AUX + (i >> 1) * 256 + (i & 1) * 128;
                            if constexpr (K) {
                                am[t] = *reinterpret_cast<const u32x2 *>(a + col * 8);
                            } else {
                                sc[t][0] = *reinterpret_cast<const u32x4 *>(a + kg * 32);
                                sc[t][1] = *reinterpret_cast<const u32x4 *>(a + kg * 32 + 16);
                            }
                        }
                    }
                    half8 bh[VT], bl[VT];
#pragma unroll
                    for (int v = 0; v < VT; v++) {
                        bh[v] = *reinterpret_cast<const half8 *>(xl + v * 2048);
                        bl[v] = *reinterpret_cast<const half8 *>(xl + v * 2048 + 1024);
                    }
                    half8 a = unpack(0, j);
#pragma unroll
                    for (int t = 0; t < RT; t++) {
                        floatx4(&ct)[VT] = c[K ? t : t & 1];
#pragma unroll
                        for (int v = 0; v < VT; v++)
                            ct[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bh[v], K && (h || j) ? ct[v] : zero, 0, 0, 0);
#pragma unroll
                        for (int v = 0; v < VT; v++) ct[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bl[v], ct[v], 0, 0, 0);
                        if (!K && t) scale(t - 1, j);
                        if (!K && !t && j) scale(RT - 1, j - 1);
                        if (t + 1 < RT) a = unpack(t + 1, j);
#pragma unroll
                        for (int i = 0; i < 2 * VT; i++) {
                            __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);                // MFMA
                            __builtin_amdgcn_sched_group_barrier(0x2, K ? 16 / (2 * VT) : (11 + 4 * VT) / (2 * VT), 0);  // VALU
                        }
                    }
                }
                if constexpr (K) {
#pragma unroll
                    for (int t = 0; t < RT; t++) {
                        if (h == 0) mins[t] = am[t][1];
                    }
                    if (h) {
                        // the superblock's minima with its sums of x: k = 0..7 their hi pieces,
                        // 8..15 their lo ones, the other lanes zeros
                        half8 bm[VT];
#pragma unroll
                        for (int v = 0; v < VT; v++) {
                            const int i = vt0 + v;
                            bm[v] = *reinterpret_cast<const half8 *>(ws + XM + i / (VT / 2) * 1024 + i % (VT / 2) * 512 +
                                                                     ((kg & 1) * 16 + col) * 16);
                            if (kg > 1) bm[v] = half8{};
                        }
#pragma unroll
                        for (int t = 0; t < RT; t++) {
                            const int i = rt0 + t;
                            const u32x4 dd = *reinterpret_cast<const u32x4 *>(ws + SUP + (i >> 1) * 256 + (i & 1) * 64 + kg * 16);
                            const half4 m0 = minima(mins[t]), m1 = minima(am[t][1]);
                            const half8 a = kg > 1 ? half8{} : half8{m0[0], m0[1], m0[2], m0[3], m1[0], m1[1], m1[2], m1[3]};
#pragma unroll
                            for (int v = 0; v < VT; v++) {
                                const floatx4 m = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, bm[v], zero, 0, 0, 0);
#pragma unroll
                                for (int r = 0; r < 4; r++) {
                                    acc[t][v][r] = fmaf(c[t][v][r], lo_of(dd[r]), acc[t][v][r]);
                                    acc[t][v][r] = fmaf(-m[r], hi_of(dd[r]), acc[t][v][r]);
                                }
                            }
                        }
                    }
                } else {
                    scale(RT - 1, 3);
                }
            }
        }
        wait_vm<0>();  // no copy outlives the workgroup's LDS
    }

    // the lane's outputs: of vector (vt_wg + vt0 + v) * 16 + col the rows
    // (tile_wg + rt0 + t) * 16 + 4 kg .. +3
    const bool quads = w.rows % 4 == 0 && ((uintptr_t)y & 15) == 0;
    const auto each = [&](auto f) {
#pragma unroll
        for (int v = 0; v < VT; v++) {
            const int vec = (vt_wg + vt0 + v) * 16 + col;
            if (vec >= n_vec) continue;
#pragma unroll
            for (int t = 0; t < RT; t++) {
                const int row = (tile_wg + rt0 + t) * 16 + kg * 4;
                if (row < w.rows) f((int64_t)vec * w.rows + row, w.rows - row, acc[t][v], vec);
            }
        }
    };
    if (gridDim.z > 1) {
        float *o = part + blockIdx.z * slice_stride;
        each([&](int64_t at, int left, const floatx4 &t, int) {
            if (quads) {
                store_agent2(o + at, t[0], t[1]);
                store_agent2(o + at + 2, t[2], t[3]);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (r < left) store_agent(o + at + r, t[r]);
            }
        });
        __shared__ int last;
        if (!arrive_last(arrivals + blockIdx.y * gridDim.x + blockIdx.x, gridDim.z, &last)) return;
        o = part + (1 - (int)blockIdx.z) * slice_stride;
        each([&](int64_t at, int left, floatx4 &t, int) {
            if (quads) {
                t += load_agent4(o + at);
            } else {
#pragma unroll
                for (int r = 0; r < 4; r++)
                    if (r < left) t[r] += load_agent(o + at + r);
            }
        });
    }
    bool inf = false;  // Q4_K: of a vector with an infinity
    const bool add = gridDim.z < (unsigned)slices && slice > 0;
    each([&](int64_t at, int left, const floatx4 &t, int vec) {
        const float undo = px.undo[vec];
        floatx4 o = K ? t * kUnscale * fabsf(undo) : t * undo;
        inf |= K && undo < 0;
        if (quads) {
            if (add) o += *reinterpret_cast<const floatx4 *>(y + at);
            *reinterpret_cast<floatx4 *>(y + at) = o;
        } else {
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (r < left) y[at + r] = add ? o[r] + y[at + r] : o[r];
        }
    });
    if (inf && slice0 + (int)gridDim.z == slices)  // the lane's own outputs again
        for (int v = 0; v < VT; v++) {
            const int vec = (vt_wg + vt0 + v) * 16 + col;
            if (vec >= n_vec || !(px.undo[vec] < 0)) continue;
            for (int t = 0; t < RT * 4; t++) {
                const int row = (tile_wg + rt0 + t / 4) * 16 + kg * 4 + t % 4;
                if (row < w.rows) y[(int64_t)vec * w.rows + row] += infinite_terms(w, px.x + (int64_t)vec * w.cols, row);
            }
        }
}

constexpr int kMaxVec = 262128;
constexpr int kMaxCols = 1 << 26;  // a row of x is addressed by 32 bits of bytes
// A launch has fewer than 2^32 threads: 512 a row tile, and 64 a piece to repack.
constexpr int kMaxRows = 1 << 26;
constexpr int64_t kMaxPieces = (1 << 26) - 4;

int launched(const char *what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GLA_OK : set_error(GLA_ERR_KERNEL, "%s launch: %s", what, hipGetErrorString(e));
}

template <bool K, int NV>
int launch_few(gla_ctx *ctx, const gla_q4w *w, const Weights &p, const float *x, int n, float *y) {
    // Two row tiles a workgroup share the pieces of x where a tile each would be more
    // than one workgroup per CU. us, two tiles / one: 6144 x 4096 Q4_0, 2 vectors
    // 6.5 / 6.2, 4 7.4 / 9.1, 8 10.8 / 12.9; Q4_K 6.5 / 6.7, 7.8 / 10.1, 10.4 / 14.3.
    // Below that one each is faster (4096 x 4096 Q4_0, 2 vectors 6.2 / 4.6). One vector,
    // whose pieces are cheap, from three workgroups per CU on (6144 x 4096 6.0 / 5.7, Q4_K
    // 6.5 / 6.2; 14336 x 4096 10.8 / 9.6, Q4_K 10.2 / 10.4).
    const auto go = [&](auto kernel, int tiles) {
        hipLaunchKernelGGL(kernel, dim3((w->n_tiles + tiles - 1) / tiles), dim3(kFewWaves * 64), 0, ctx->stream, p, x, n, y);
    };
    if (w->n_tiles > (NV == 1 ? 2 : 1) * ctx->n_cu)
        go(matvec_q4_few_kernel<K, NV, 2, 4>, 2);
    else if (w->n_quads > kFewWaves)
        go(matvec_q4_few_kernel<K, NV, 1, 4>, 1);
    else
        go(matvec_q4_few_kernel<K, NV, 1, 1>, 1);
    return launched("matvec_q4_few_kernel");
}

int few(gla_ctx *ctx, const gla_q4w *w, const Weights &p, const float *x, int n, float *y) {
    const auto of = [&](auto k) {
        constexpr bool K = decltype(k)::value;
        return n == 1 ? launch_few<K, 1>(ctx, w, p, x, n, y) : n == 2 ? launch_few<K, 2>(ctx, w, p, x, n, y)
             : n <= 4 ? launch_few<K, 4>(ctx, w, p, x, n, y) : launch_few<K, 8>(ctx, w, p, x, n, y);
    };
    return w->format == GLA_Q4_K ? of(std::true_type()) : of(std::false_type());
}

constexpr int kFewVec = 8;

// Bytes of the pieces, the sums and the scales of n vectors.
struct PieceBytes {
    size_t xp, xm, undo;
    size_t all() const { return xp + xm + undo; }
};
PieceBytes piece_bytes(const gla_q4w *w, int n) {
    const size_t tiles = (size_t)(n + 15) / 16;
    return {tiles * w->n_quads * 4 * 2048, w->format == GLA_Q4_K ? tiles * (w->n_quads / 2) * 512 : 0,
            ((size_t)n * sizeof(float) + 255) / 256 * 256};
}

// Makes them in the stream's scratch.
int make_pieces(gla_ctx *ctx, const gla_q4w *w, const float *x, int n, Pieces *px) {
    const bool k = w->format == GLA_Q4_K;
    const PieceBytes b = piece_bytes(w, n);
    void *scr = nullptr;
    if (int rc = ensure_scratch(ctx, b.all(), &scr)) return rc;
    uint8_t *base = (uint8_t *)scr;
    px->xp = (const _Float16 *)base;
    px->xm = (const _Float16 *)(base + b.xp);
    px->undo = (const float *)(base + b.xp + b.xm);
    px->x = x;
    const bool four = n > 64;
    auto kernel = k ? (four ? split_q4_kernel<true, 4> : split_q4_kernel<true, 1>)
                    : (four ? split_q4_kernel<false, 4> : split_q4_kernel<false, 1>);
    hipLaunchKernelGGL(kernel, dim3(four ? (n + 3) / 4 : n, four ? 1 : 2), dim3(kSplitThreads), 0, ctx->stream, x, n, w->cols, w->n_quads,
                       (_Float16 *)px->xp, (_Float16 *)px->xm, (float *)px->undo);
    return launched("split_q4_kernel");
}

struct Tile {
    int nv, rt;  // of 16 vectors, of 16 rows
};
// The mid kernel's tiles, and its cost: rounds of a workgroup per CU, each the tile's
// products and two for what comes before and after them. (A call of 4,096 columns
// takes about 8 us + 1.33 a unit of cost, Q4_K 8 + 1.5. The two are fitted there: of
// 16,384 columns they are half a unit, of 576 some fourteen.)
constexpr int kMidCost = 34;
constexpr Tile kMidTiles[] = {{1, 1}, {1, 2}, {1, 3}, {1, 4}, {2, 3}, {2, 4}, {4, 4}, {8, 4}};
Tile mid_tile(const gla_ctx *ctx, const gla_q4w *w, int n, int64_t *cost) {
    Tile best = kMidTiles[0];
    *cost = INT64_MAX;
    for (const Tile &t : kMidTiles) {
        const int64_t wgs = (int64_t)((w->n_tiles + t.rt - 1) / t.rt) * (((n + 15) / 16 + t.nv - 1) / t.nv);
        const int64_t c = (wgs + ctx->n_cu - 1) / ctx->n_cu * (t.nv * t.rt + 2);
        if (c < *cost) best = t, *cost = c;
    }
    return best;
}

int mid(gla_ctx *ctx, const gla_q4w *w, const Weights &p, const float *x, int n, float *y, Tile t) {
    Pieces px;
    if (int rc = make_pieces(ctx, w, x, n, &px)) return rc;
    const auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((w->n_tiles + t.rt - 1) / t.rt, ((n + 15) / 16 + t.nv - 1) / t.nv), dim3(kMidWaves * 64),
                           0, ctx->stream, p, px, n, y);
        return launched("matvec_q4_mid_kernel");
    };
    const auto of = [&](auto kk) {
        constexpr bool K = decltype(kk)::value;
        switch (t.nv * 8 + t.rt) {
        case 1 * 8 + 1: return go(matvec_q4_mid_kernel<K, 1, 1, 1>);
        case 1 * 8 + 2: return go(matvec_q4_mid_kernel<K, 1, 2, 1>);
        case 1 * 8 + 3: return go(matvec_q4_mid_kernel<K, 1, 3, 1>);
        case 1 * 8 + 4: return go(matvec_q4_mid_kernel<K, 1, 4, 1>);
        case 2 * 8 + 3: return go(matvec_q4_mid_kernel<K, 2, 3, 1>);
        case 2 * 8 + 4: return go(matvec_q4_mid_kernel<K, 2, 4, 1>);
        case 4 * 8 + 4: return go(matvec_q4_mid_kernel<K, 2, 4, 2>);
        default: return go(matvec_q4_mid_kernel<K, 2, 4, 4>);
        }
    };
    return w->format == GLA_Q4_K ? of(std::true_type()) : of(std::false_type());
}

int many(gla_ctx *ctx, const gla_q4w *w, const Weights &p, const float *x, int n, float *y) {
    const bool k = w->format == GLA_Q4_K;
    // Workgroups of 128 vectors where they fill two on every CU, else of 64. us, 64 wide
    // / 128: 6144 x 4096, 1,024 vectors 117 / 118, 1,999 216 / 210; Q4_K 1,999 222 / 193.
    // Fewer than 384 of 64 are two slices of K (of eight quads or more), as long as
    // their partial sums stay within 28 MB: 6144 x 4096, 400 vectors 79.5 -> 71.2.
    const int vec_tiles = (n + 15) / 16, row_blocks = (w->n_tiles + 7) / 8;
    const int vt = (int64_t)row_blocks * ((vec_tiles + 7) / 8) >= 2 * ctx->n_cu ? 4 : 2;
    const int vec_blocks = (vec_tiles + 2 * vt - 1) / (2 * vt);
    const int64_t wgs = (int64_t)row_blocks * vec_blocks, stride = (int64_t)n * w->rows;
    const size_t partials = (size_t)(2 * stride) * sizeof(float);
    const int slices = vt == 2 && 2 * wgs <= 3 * ctx->n_cu && w->n_quads >= 16 && partials <= ((size_t)28 << 20) ? 2 : 1;
    const size_t behind = piece_bytes(w, n).all();
    void *scr = nullptr;
    int32_t *arrivals = nullptr;
    bool at_once = true;
    if (slices > 1 && (ensure_scratch(ctx, behind + partials, &scr) != GLA_OK || ensure_arrivals(ctx, (size_t)wgs, &arrivals) != GLA_OK)) {
        // the partial sums or their counters cannot be had (a capture in which they would
        // have to grow, a full device): a slice after the other
        clear_error();
        (void)hipGetLastError();
        at_once = false;
    }
    Pieces px;
    if (int rc = make_pieces(ctx, w, x, n, &px)) return rc;
    float *part = at_once && slices > 1 ? (float *)((uint8_t *)scr + behind) : nullptr;
    const auto go = [&](auto kernel) {
        for (int slice = 0; slice < (at_once ? 1 : slices); slice++) {
            hipLaunchKernelGGL(kernel, dim3(row_blocks, vec_blocks, at_once ? slices : 1), dim3(256), 0, ctx->stream, p, px, n, y,
                               slices, slice, part, stride, arrivals);
            if (int rc = launched("matvec_q4_gemm_kernel")) return rc;
        }
        return (int)GLA_OK;
    };
    if (vt == 4) return k ? go(matvec_q4_gemm_kernel<true, 4>) : go(matvec_q4_gemm_kernel<false, 4>);
    return k ? go(matvec_q4_gemm_kernel<true, 2>) : go(matvec_q4_gemm_kernel<false, 2>);
}

}  // namespace
}  // namespace gla

using namespace gla;

extern "C" {

int gla_q4w_create(gla_ctx *ctx, gla_q4_format format, const uint8_t *ggml_host, int rows, int cols, gla_q4w **out) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && ggml_host && out, "gla_q4w_create: NULL argument");
    *out = nullptr;
    GLA_REQUIRE(format == GLA_Q4_0 || format == GLA_Q4_K, "gla_q4w_create: bad format %d", (int)format);
    const bool k = format == GLA_Q4_K;
    GLA_REQUIRE(rows > 0 && cols > 0 && cols % (k ? 256 : 32) == 0,
                "gla_q4w_create: rows %d, cols %d (cols must be a positive multiple of %d)", rows, cols, k ? 256 : 32);
    GLA_REQUIRE(cols <= kMaxCols, "gla_q4w_create: %d columns (at most %d)", cols, kMaxCols);
    GLA_REQUIRE(rows <= kMaxRows && ((int64_t)rows + 15) / 16 * ((cols + 127) / 128) <= kMaxPieces,
                "gla_q4w_create: %d x %d is too large for one launch", rows, cols);
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    ctx->q4ws.reserve(ctx->q4ws.size() + 1);
    gla_q4w *w = new gla_q4w();
    w->ctx = ctx;
    w->format = format;
    w->rows = rows;
    w->cols = cols;
    w->n_tiles = (rows + 15) / 16;
    w->n_quads = (cols + 127) / 128;
    const int n_groups = cols / 32;
    const int64_t pieces = (int64_t)w->n_tiles * w->n_quads;
    const size_t raw_bytes = (size_t)rows * (k ? (size_t)(cols / 256) * 144 : (size_t)n_groups * 18);
    uint8_t *raw = nullptr;
    hipError_t e = hipMalloc(&w->quants, (size_t)pieces * 1024);
    if (e == hipSuccess) e = hipMalloc(&w->aux, (size_t)pieces * 128);
    if (e == hipSuccess && k) e = hipMalloc(&w->super, (size_t)pieces / 2 * 64);
    if (e == hipSuccess) e = hipMalloc(&raw, raw_bytes);
    if (e == hipSuccess) e = hipMemcpyAsync(raw, ggml_host, raw_bytes, hipMemcpyHostToDevice, ctx->stream);
    if (e == hipSuccess) {
        const int64_t n_units = pieces * 64;
        auto kernel = k ? q4_repack_kernel<true> : q4_repack_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3((unsigned)((n_units + 255) / 256)), dim3(256), 0, ctx->stream, raw, rows, n_groups,
                           w->n_quads, n_units, w->quants, w->aux, w->super);
        e = hipGetLastError();
    }
    const hipError_t done = hipStreamSynchronize(ctx->stream);
    if (e == hipSuccess) e = done;
    if (raw) (void)hipFree(raw);
    if (e != hipSuccess) {
        (void)hipGetLastError();  // not the next launch's
        detach_q4w(w);
        delete w;
        return set_error(GLA_ERR_BUFFER, "gla_q4w_create: %s", hipGetErrorString(e));
    }
    ctx->q4ws.push_back(w);
    *out = w;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_q4w_destroy(gla_q4w *w) {
    GLA_GUARD_BEGIN
    if (!w) return GLA_OK;
    if (gla_ctx *ctx = w->ctx) {  // else its context already freed the weights
        (void)hipSetDevice(ctx->device);
        (void)hipStreamSynchronize(ctx->stream);
        ctx->q4ws.erase(std::remove(ctx->q4ws.begin(), ctx->q4ws.end(), w), ctx->q4ws.end());
        detach_q4w(w);
    }
    delete w;
    return GLA_OK;
    GLA_GUARD_END
}

int gla_q4w_rows(const gla_q4w *w) { return w ? w->rows : -1; }
int gla_q4w_cols(const gla_q4w *w) { return w ? w->cols : -1; }

int gla_matvec_q4(gla_ctx *ctx, const gla_q4w *w, const float *x, int n_vec, float *y) {
    GLA_GUARD_BEGIN
    GLA_REQUIRE(ctx && w, "gla_matvec_q4: NULL argument");
    GLA_REQUIRE(w->ctx == ctx, "gla_matvec_q4: the weights belong to %s",
                w->ctx ? "another context" : "a destroyed context");
    GLA_REQUIRE(n_vec >= 0 && n_vec <= kMaxVec, "gla_matvec_q4: n_vec %d (0 to %d; split the call)", n_vec, kMaxVec);
    if (n_vec == 0) return GLA_OK;
    GLA_REQUIRE(x && y, "gla_matvec_q4: NULL buffer");
    GLA_CHECK_HIP(hipSetDevice(ctx->device), GLA_ERR_DEVICE);
    const Weights p{w->quants, w->aux, w->super, w->rows, w->cols, w->n_tiles, w->n_quads};
    if (n_vec <= kFewVec) return few(ctx, w, p, x, n_vec, y);
    // The mid kernel's small tiles while their products are few, then the other's large
    // ones (us, mid / many: Q4_0 4096 x 4096, 128 vectors 22.6 / 41.6, 400 52.7 / 52.8, 512
    // 53.5 / 57.7; 1024 x 4096, 1,500 54.4 / 56.7; Q4_K 6144 x 4096, 128 34.4 / 39.2, 192
    // 48.1 / 51.1, 256 56.4 / 51.7, 320 61.8 / 55.1; 14336 x 4096, 64 34.6 / 38.8, 160 91.1 /
    // 74.9; other widths: Q4_0 4096 x 16384, 64 40.4 / 113, 256 108 / 128, 512 194 / 175; 960
    // x 576, 256 11.3 / 17.5, 1,024 17.1 / 19.9; 49152 x 576, 32 19.4 / 19.6, 64 28.1 / 20.5).
    // The rule takes the slower one of Q4_K 6144 x 4096, 256, and 4096 x 16384, 512 vectors.
    int64_t cost;
    const Tile t = mid_tile(ctx, w, n_vec, &cost);
    if (cost <= kMidCost) return mid(ctx, w, p, x, n_vec, y, t);
    return many(ctx, w, p, x, n_vec, y);
    GLA_GUARD_END
}

}  // extern "C"
