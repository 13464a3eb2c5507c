// Shared state and helpers of libgen9blas_llm.so: errors, operands, work buffers, and the layout of MX4 matrices.
//
// MX4 layout. A tile is 16 rows × 128 k: 1024 bytes of codes, lane l = 16·g + r of a wave holding the 16 bytes (32 codes,
// low half first) of row r, k = 32g .. 32g+31: one block, so one scale. That is an operand of
// v_mfma_scale_f32_16x16x128_f8f6f4 as it lies, and after a conversion eight consecutive k for each of four FP16 or BF16
// 16x16x32 MFMAs (a sum over k in any order). A matrix is its row tiles, each its kc = ⌈K/128⌉ tiles in k order, so a
// wave that walks k streams consecutive KiB. Scales: for each row tile and group of 512 k a word per lane, byte j the
// scale of tile 4·group + j. Codes past K and past the last row are zero, their scales 0.
//
// Row exponents. A block of zeros has scale 0 (or 255: a NaN block, whatever its codes). `top`: for each row and group of
// 512 k the largest scale byte, so no scale of a row but NaN's lies above its largest, e. FP16 products scale a row's weights
// by it: code · 2^(s−e+13) is exact in FP16 (49152 at most, and down to s = e − 36), and the sums are multiplied by 2^(e−140)
// at the end.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>
#include "gen9blas.h"
#include "gen9blas_hip.h"
#include "gen9blas_llm.h"

#define G9_HIDDEN __attribute__((visibility("hidden")))

struct gen9blas_mx4 {
    int count, rows, K;
    int rt, kc, kg, kt;        // row tiles, tiles and groups along k, bytes of `top` a row (kg rounded up to 16)
    uint8_t *codes;            // [count][rt][kc][64][16]
    uint8_t *scales;           // [count][rt][kg][64][4]
    uint8_t *top;              // [count][rt][16][kt]
};

namespace g9llm {

// ---- errors: as in libgen9blas.so, in a text of this library's own ----
G9_HIDDEN int fail(int code, const char *fmt, ...) __attribute__((format(printf, 2, 3)));
G9_HIDDEN int hip_fail(hipError_t e, const char *what, const char *file, int line);
#define G9_FAIL(code, ...) return ::g9llm::fail((code), __VA_ARGS__)
#define G9_HIP(x) do { hipError_t e_ = (x); if (e_ != hipSuccess) return ::g9llm::hip_fail(e_, #x, __FILE__, __LINE__); } while (0)
#define G9_TRY(x) do { int r_ = (x); if (r_) return r_; } while (0)

G9_HIDDEN extern hipStream_t stream;   // libgen9blas.so's
G9_HIDDEN extern int num_cus;
// Start of every entry point: clears the status, opens the device, makes it current. 0 or an error.
G9_HIDDEN int begin();
// 0 if [p, p + bytes) is device memory of one allocation, else INVALID_ARG naming `what`.
G9_HIDDEN int need_device(const void *p, size_t bytes, const char *what);
// Device scratch, grown on demand and kept; growing waits for queued work.
enum Slot { SLOT_A = 0, SLOT_PART, SLOT_PLAN, SLOT_SLOTS, SLOT_X, SLOT_W, SLOT_DZ, SLOT_SUMS, SLOT_SORT, NSLOTS };
G9_HIDDEN int scratch(int slot, size_t bytes, void **p);
// 0, or UNSUPPORTED while the stream is being captured into a graph: for calls that queue more than kernels on their operands.
G9_HIDDEN int not_captured(const char *who);
// scratch(), refused while captured: a graph would go on using a buffer that later calls write, and free as they outgrow it.
inline int work_buffer(const char *who, int slot, size_t bytes, void **p) {
    G9_TRY(not_captured(who));
    return scratch(slot, bytes, p);
}
// Clears `rows` rows of `bytes` bytes (a multiple of 2), `ld` bytes apart.
G9_HIDDEN int zero_rows(void *p, long long ld, long long rows, long long bytes);
// The longest rows: kernels count k in an int, up to the end of the last 128-k chunk.
constexpr int MAX_COLS = 0x7fffff80;
inline int elem_size(int type) { return type == GEN9BLAS_S ? 4 : 2; }
inline long long cdiv(long long a, long long b) { return (a + b - 1) / b; }

// One MX4 matrix (or the matrices of the experts) as kernels see it.
struct Mx4View {
    const uint8_t *codes, *scales, *top;
    int rows, K, rt, kc, kg, kt;
};
inline Mx4View view(const gen9blas_mx4 *q) { return {q->codes, q->scales, q->top, q->rows, q->K, q->rt, q->kc, q->kg, q->kt}; }

// A dense product whose k is split among `parts` workgroups: each leaves its FP32 sums in a plane of rows × ld, and a second kernel
// adds the planes in their order. (The experts' have enough workgroups: parts = 1.)
struct Split {
    int parts;
    float *sums;
    long long rows, ld;
};

typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

}  // namespace g9llm
