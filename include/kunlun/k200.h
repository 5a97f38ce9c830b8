// KunlunK200 matmul surface, implemented for AMD Instinct MI355X (gfx950).
//
// This header keeps the declarations, argument meaning, defaults and class
// layouts of the matmul subset of the reference library's public header
// (reference include/kunlun/k200.h:10-37, 40-41, 62-107, 127-132, 185-335, 345-350)
// so a consumer of that subset rebuilds against this library unchanged.
// Declarations of the reference that are not on the matmul path (attention,
// Q6_K, KV caches, row gathers) are not
// declared here. matmul_swiglu, the paged key-value cache with its attention and
// process_logits have no reference counterpart (see below).
//
// Device numbering: the reference drives the two processing dies of one
// Kunlun card as devices 0 and 1. Here a device is one HIP device (one GPU);
// valid ids are [0, device_count()), at most kunlun::max_devices.
#pragma once

#include <cstddef>
#include <cstdint>
#include <mutex>

namespace kunlun {

constexpr int max_devices = 8;

// Process-wide lock around device selection, allocation and submission
// (reference k200.h:10). Callers hold it around raw select/copy/wait runs.
std::recursive_mutex & runtime_mutex();
// Fail fast: print the diagnostic context and abort when status != 0
// (reference k200.h:11).
void check(int status);
// Optional borrowed tensor name; dimensions are copied (reference k200.h:13).
void diagnostic_tensor(const char * name, const int64_t * dimensions = nullptr);
// Fail fast when the condition is false (reference k200.h:14).
void require(bool condition);
int device_count(int * count);                       // reference k200.h:15
void select(int device);                             // reference k200.h:16
// Completes every operation on the selected device, the library's and any
// other HIP work of the process (hipDeviceSynchronize; reference k200.h:17).
int wait();
enum CopyKind { host_to_device, device_to_host, device_to_device };
// Copies on the selected device after the library's submitted work there and
// completes before returning, in every direction (reference k200.h:18-19).
int copy(void * dst, const void * src, size_t bytes, CopyKind kind);
// Device-to-device copy between GPUs; completes before returning (reference k200.h:20).
void peer(int dst_device, void * dst, int src_device, const void * src, size_t bytes);
void * allocate(int device, size_t bytes);           // reference k200.h:21, nullptr on failure
void release(int device, void * ptr, size_t bytes);  // reference k200.h:22
size_t allocated_bytes(int device);                  // reference k200.h:23

// RAII device allocation (reference k200.h:25-37).
class Buffer {
public:
    Buffer(int device, size_t bytes);
    ~Buffer();
    Buffer(const Buffer &) = delete;
    Buffer & operator=(const Buffer &) = delete;
    void * data() const { return ptr_; }
    size_t size() const { return bytes_; }
private:
    int device_;
    size_t bytes_;
    void * ptr_;
};

// Values match the reference enumeration (reference k200.h:40). q6_k is not
// accepted by matmul, as in the reference.
enum class WeightType { f32 = 0, f16 = 1, q4_0 = 2, rowwise_i8 = 3, q6_k = 4 };
// Elementwise operations (reference k200.h:41).
enum class ElementwiseOp { add = 0, multiply = 1, silu = 2, rms_norm = 3, scale = 4 };

struct SwiGLULayout;
struct KVCacheLayout;
struct KVPagesLayout;
struct KVAppendLayout;
struct PagedAttentionLayout;
struct LogitsLayout;
struct KVCacheF8Layout;
struct KVReadLayout;

// Per-call state owner: binds to the first device it is used on and owns
// lazily grown device workspaces (reference k200.h:62-88).
class Kernel {
public:
    Kernel();
    ~Kernel();
    Kernel(const Kernel &) = delete;
    Kernel & operator=(const Kernel &) = delete;
    struct Impl;
private:
    Impl * impl_;
    friend void matmul(Kernel &, int, void *, const void *, const void *, int, int, int,
                       WeightType, const float *, const float *, int);
    friend bool swiglu(Kernel &, int, void *, size_t, const void *, size_t, const void *, size_t,
                       const SwiGLULayout &);
    friend void matmul_swiglu(Kernel &, int, void *, const void *, const void *, const void *, int, int, int,
                              WeightType);
    friend void elementwise(Kernel &, int, void *, const void *, const void *, int, int, int, ElementwiseOp,
                            float);
    friend bool paged_attention(Kernel &, int, void *, const void *, const void *, const void *, const int *,
                                const int *, const KVCacheLayout &, const PagedAttentionLayout &);
    friend bool kv_append(Kernel &, int, void *, void *, void *, const void *, const void *, const void *,
                          const int *, const int *, const int *, const int *, const float *, const float *,
                          const KVCacheLayout &, const KVAppendLayout &);
    friend bool kv_reserve(Kernel &, int, int *, int *, int *, const int *, const int *, int,
                           const KVCacheLayout &, const KVPagesLayout &);
    friend bool kv_fork(Kernel &, int, void *, void *, int *, int *, int *, const int *, const int *, int,
                        const KVCacheLayout &, const KVPagesLayout &);
    friend bool kv_free(Kernel &, int, int *, int *, int *, const int *, int, const KVCacheLayout &,
                        const KVPagesLayout &);
    friend bool kv_compact(Kernel &, int, void *, void *, int *, int *, int *, const int *, const int *,
                           const int *, const KVCacheLayout &, const KVPagesLayout &);
    friend bool kv_copy_pages(Kernel &, int, void *, void *, const int *, const int *, int, const KVCacheLayout &,
                              const KVPagesLayout &);
    friend bool paged_attention_f8(Kernel &, int, void *, const void *, const void *, const void *, const float *,
                                   const float *, const int *, const int *, const KVCacheF8Layout &,
                                   const PagedAttentionLayout &);
    friend bool kv_append_f8(Kernel &, int, void *, void *, float *, float *, void *, const void *, const void *,
                             const void *, const int *, const int *, const int *, const int *, const float *,
                             const float *, const KVCacheF8Layout &, const KVAppendLayout &);
    friend bool kv_read_f8(Kernel &, int, void *, void *, const void *, const void *, const float *, const float *,
                           const int *, const int *, const int *, const int *, const KVCacheF8Layout &,
                           const KVReadLayout &);
    friend bool kv_fork_f8(Kernel &, int, void *, void *, float *, float *, int *, int *, int *, const int *, const int *,
                           int, const KVCacheF8Layout &, const KVPagesLayout &);
    friend bool kv_compact_f8(Kernel &, int, void *, void *, float *, float *, int *, int *, int *, const int *,
                              const int *, const int *, const KVCacheF8Layout &, const KVPagesLayout &);
    friend bool kv_copy_pages_f8(Kernel &, int, void *, void *, float *, float *, const int *, const int *, int,
                                 const KVCacheF8Layout &, const KVPagesLayout &);
    friend bool process_logits(Kernel &, int, void *, const void *, const float *, const int *, const int *,
                               const int *, const float *, const int *, const uint32_t *, const LogitsLayout &);
};

// Packed rowwise INT8 weight layout (reference k200.h:90-96):
// [aligned(k*rows) int8 codes][aligned(4*rows) f32 row scales][256 B maxima].
size_t aligned(size_t bytes);
size_t packed_i8_size(int k, int rows);
float * packed_i8_scales(void * weights, int k, int rows);
float * packed_i8_maxima(void * weights, int k, int rows);
// Quantizes F32 host rows and uploads them to a caller-owned
// packed_i8_size(k, rows) device allocation. Completes before returning.
void upload_i8_rows(int device, void * weights, int k, int rows,
                    int first_row, int count, const float * input);

// W: [n,k], X: [batch,k], Y: [batch,n]. All pointers refer to device memory.
// Q4_0: 18-byte blocks (little-endian F16 scale + 16 paired 4-bit values).
// rowwise_i8 requires scales[n] and maxima[6], also in device memory.
// matmul submits work; select(device) + check(wait()) completes it.
// K must be divisible by 32, K <= 16384 (reference k200.h:98-105).
void matmul(Kernel &, int device, void * y, const void * w, const void * x,
            int k, int n, int batch, WeightType type,
            const float * scales = nullptr, const float * maxima = nullptr, int tile = 16);

// Element type of SwiGLU inputs and outputs (reference k200.h:132).
enum class InputType { f32, f16 };

// SiLU(gate) * up over `rows` rows of `width` contiguous values
// (reference k200.h:185-199). Strides are bytes between rows.
struct SwiGLULayout {
    int width, rows;
    int gate_stride, up_stride, output_stride;
    InputType type;
};
// Empty string: the layout is supported; otherwise "type", "shape", "stride"
// or "byte extent" names the first rule it breaks.
const char * swiglu_reason(const SwiGLULayout &);
// Computes SiLU(gate)*up with F32 intermediates and one final output
// rounding, and completes before returning. y may alias gate or up element
// for element (equal row strides), or hold rows disjoint from them; any other
// overlap, a span beyond the given byte sizes, misalignment, a bad device or
// a Kernel bound to another device returns false with no work submitted.
bool swiglu(Kernel &, int device, void * y, size_t y_bytes,
            const void * gate, size_t gate_bytes, const void * up, size_t up_bytes,
            const SwiGLULayout &);

// No counterpart in the reference, which computes this as two matmul calls
// followed by swiglu (or common_q4_matmul_pair then swiglu, reference
// src/q4-pair.inc:9-80): Y[batch,n] = SiLU(X W_gate^T) * (X W_up^T), F32 Y.
// w_gate and w_up are [n,k] weights of one type (f32, f16 or q4_0) and the
// arguments follow matmul's rules. At batch >= 64 (Q4_0, F16) both products
// run in one fp16-MFMA GEMM with SiLU * up in its last step; Q4_0 below that
// runs both matrices in one GEMV pass likewise (33..63 columns: per 32
// columns); others run two GEMVs and the SwiGLU kernel. Submits; select + wait
// completes it.
void matmul_swiglu(Kernel &, int device, void * y, const void * w_gate, const void * w_up, const void * x,
                   int k, int n, int batch, WeightType type);

// F32 elementwise op over `count` values, completed before returning
// (reference k200.h:106-107): add and multiply take b of b_count == count
// values or of b_count == width values repeated every row; silu, scale
// (a * parameter) and rms_norm (each `width` row scaled by
// 1 / sqrt(mean(a^2) + parameter)) ignore b. count % width == 0,
// width <= 16384; y may equal a or b.
void elementwise(Kernel &, int device, void * y, const void * a, const void * b,
                 int count, int width, int b_count, ElementwiseOp op, float parameter = 0);

// Native Q4 layout (reference k200.h:127-131): the Q4_0 values and FP16
// block scales of an [n,k] matrix repacked as [N32 tile][K32 block][16 K
// pairs][32 rows] signed 4-bit values, then the scales [N32 tile][K32
// block][32 rows]; N is padded to 32 with zeros. Supported for
// 0 < k <= 16384, k % 32 == 0, 0 < n <= 90000000 / k.
bool native_q4_layout_supported(int k, int n);
// Bytes of the layout, 0 when unsupported.
size_t native_q4_size(int k, int n);
// Host repack of n rows of Q4_0 blocks into `destination` (bytes >=
// native_q4_size); false for an unsupported shape, a short or null buffer or
// overlapping ranges.
bool pack_native_q4(void * destination, size_t bytes, const void * q4, int k, int n);
// Packs on the host and copies to device memory `weights`; completes before
// returning. Invalid arguments abort.
void upload_native_q4(int device, void * weights, const void * q4, int k, int n);

// Empty string when the reference would take its accelerated route for this
// shape, otherwise the reference's reason (reference k200.h:200-203).
const char * native_q4_reason(int k, int n, int batch, InputType type);
// Reference k200.h:204-207. Here every call runs the same exact kernels, and
// no HBM or L3 workspace is held (both sizes are 0).
struct NativeQ4Statistics {
    size_t accelerated, fallback;
    size_t hbm_workspace_bytes, l3_workspace_bytes;
};
class NativeQ4Workspace {                            // reference k200.h:208-219
public:
    NativeQ4Workspace();
    ~NativeQ4Workspace();
    NativeQ4Workspace(const NativeQ4Workspace &) = delete;
    NativeQ4Workspace & operator=(const NativeQ4Workspace &) = delete;
    NativeQ4Statistics statistics() const;
    struct Impl;
private:
    Impl * impl_;
    friend bool native_q4_matmul(NativeQ4Workspace &, int, void *, const void *, const void *, int, int, int,
                                 InputType);
};
// Y[batch,n] = X[batch,k] W^T for W in the native layout (256-byte aligned),
// X F32 or F16, Y F32; completes before returning (reference k200.h:220-224).
// The result is exact up to a 23-bit fixed-point view of each 32-value
// activation block, on every route. Returns true where the reference returns
// true (native_q4_reason is empty and y and input are 64-byte aligned) and
// counts the call as accelerated, else false and counts a fallback. The
// workspace binds to the first device it is used on; invalid arguments or
// overlapping ranges abort.
bool native_q4_matmul(NativeQ4Workspace &, int device, void * y, const void * weights,
                      const void * input, int k, int n, int batch = 1, InputType type = InputType::f32);

// ---------------------------------------------------------------------------
// Common Q4 ABI v1 (reference k200.h:226-335): the persistent weight format
// K200_Q4_0_MICRO32_BANK16_KMAJOR (layout 1, scale order 1) of an [n,k] Q4_0
// matrix, padded to Kp = k rounded up to 512 (k < 512) or 256 and Np = n
// rounded up to 256. For output column c and K block b, the 16 bytes of
// signed nibble pairs (K 2p low, 2p+1 high) sit at
// ((c/32) * Kp/32 + b) * 512 + (c%16) * 32 + ((c%32)/16) * 16; the FP16 scales
// follow at scale_offset = Np*Kp/2 as [b][Np]. Payload Np*Kp*9/16 bytes.
struct CommonQ4Info {
    uint32_t abi_version, quant_type, layout, scale_order;
    int k, n, kp, np, device;
    size_t scale_offset, payload_bytes;
};
bool common_q4_supported(int k, int n);               // 0 < k <= 16384, 0 < n <= 32000
size_t common_q4_size(int k, int n);                  // payload bytes, 0 when unsupported

struct CommonQ4ActivationStatistics {
    size_t prepare_calls, quantized_chunks, quant_kernel_launches;
    size_t prepared_matmuls, prepared_chunks, invalidations, rejected_calls;
    size_t hbm_activation_bytes;
    uint64_t quantization_ns, preparation_ns;
};
struct CommonQ4ActivationChunk {
    const void * values; const void * scales;
    int first, rows, padded_rows, kp, components;
    size_t values_bytes, scales_bytes;
};
class CommonQ4ActivationLease;
class CommonQ4Workspace;

struct CommonQ4WeightStatistics { size_t uploads, upload_bytes; double pack_ms, upload_ms; };
class CommonQ4Weight {
public:
    // Borrowed storage must be 256-byte aligned, hold common_q4_size bytes and
    // outlive this handle and its calls; null storage allocates it here.
    CommonQ4Weight(int device, int k, int n, void * storage = nullptr, size_t bytes = 0);
    ~CommonQ4Weight();
    CommonQ4Weight(const CommonQ4Weight &) = delete;
    CommonQ4Weight & operator=(const CommonQ4Weight &) = delete;
    CommonQ4Info info() const;
    CommonQ4WeightStatistics statistics() const;
    void * data() const;
    // Packs n rows of ceil(k/32) Q4_0 blocks on the host and uploads them;
    // completes before returning.
    void upload(const void * q4, size_t bytes);
    struct Impl;
private:
    Impl * impl_;
    friend bool common_q4_matmul_pair(CommonQ4Workspace &, int, void *, void *, const CommonQ4Weight &,
                                      const CommonQ4Weight &, const CommonQ4ActivationLease &, uint64_t);
    friend void common_q4_matmul(CommonQ4Workspace &, int, void *, const CommonQ4Weight &, const void *, int,
                                 InputType);
    friend bool common_q4_matmul_shared(CommonQ4Workspace &, int, void *, const CommonQ4Weight &,
                                        const CommonQ4ActivationLease &, uint64_t);
};
struct CommonQ4Statistics {
    // Calls by route, as the reference counts them: GEMV (M = 1, two-component
    // A8), then M > 1 chunks by padded rows (8, 32, 64 with Kp <= 8192, 128
    // with Kp <= 4096, 64 above, 128 above), then the exact M = 1 route.
    size_t paths[8], calls, chunks;
    size_t hbm_workspace_bytes, l3_workspace_bytes, slice_bytes;
};
// Counters of the reference's SD engine schedules; always zero here.
struct CommonQ4MacStatistics {
    size_t baseline_sd_calls, stream_sd_calls, shape_fallbacks, resident_l1d_bytes;
};
// Device view of the last call's quantized activations (components 0: none).
// components 2 (M = 1): code of K index j at values[(j/32)*64 + j%32], the
// residual code at values[2*kp + (j/32)*64 + j%32], F32 scales[0] and [1].
// components 1 (M > 1): row r's codes at values[r*kp + j], scale scales[r*16].
struct CommonQ4Quantization { const void * values; const void * scales; int rows, kp, components; };
struct CommonQ4PairStatistics { size_t calls, declined, l3_partial_bytes; };
enum class CommonQ4PairStatus { NotAttempted, Success, Disabled, InvalidInput, Configuration, WeightAbi, Lease, Alias,
                                Workspace };
class CommonQ4Workspace {
public:
    CommonQ4Workspace();
    ~CommonQ4Workspace();
    CommonQ4Workspace(const CommonQ4Workspace &) = delete;
    CommonQ4Workspace & operator=(const CommonQ4Workspace &) = delete;
    CommonQ4Statistics statistics() const;
    CommonQ4ActivationStatistics activation_statistics() const;
    CommonQ4MacStatistics mac_statistics() const;
    // Borrowed device buffers, valid until the next call or workspace destruction.
    CommonQ4Quantization quantization() const;
    struct Impl;
private:
    Impl * impl_;
    friend CommonQ4PairStatistics common_q4_pair_statistics(const CommonQ4Workspace &);
    friend CommonQ4PairStatus common_q4_pair_last_status(const CommonQ4Workspace &);
    friend bool common_q4_matmul_pair(CommonQ4Workspace &, int, void *, void *, const CommonQ4Weight &,
                                      const CommonQ4Weight &, const CommonQ4ActivationLease &, uint64_t);
    friend void common_q4_matmul(CommonQ4Workspace &, int, void *, const CommonQ4Weight &, const void *, int,
                                 InputType);
    friend bool common_q4_prepare(CommonQ4Workspace &, int, const void *, int, int, InputType, uint64_t,
                                  CommonQ4ActivationLease &);
    friend bool common_q4_matmul_shared(CommonQ4Workspace &, int, void *, const CommonQ4Weight &,
                                        const CommonQ4ActivationLease &, uint64_t);
};
// Y[m,n] = X[m,k] W^T, X F32 or F16 contiguous, Y F32; completes before
// returning (reference k200.h:300-302). M = 1 quantizes X per tensor into two
// int8 components (the exact F32 product when Np * Kp > 2^27, as the
// reference's exact route); M > 1 quantizes each row to int8 (Row A8). The
// original weight scales are exact. Invalid arguments, another device's
// weight, overlap or misalignment abort before any launch.
void common_q4_matmul(CommonQ4Workspace &, int device, void * y, const CommonQ4Weight &,
                      const void * input, int m, InputType type = InputType::f32);

// A quantized snapshot of X for later common_q4_matmul_shared and
// common_q4_matmul_pair calls (reference k200.h:306-322). The owner passes a
// new nonzero generation after writing X; any other workspace call retires it.
class CommonQ4ActivationLease {
public:
    CommonQ4ActivationLease();
    ~CommonQ4ActivationLease();
    CommonQ4ActivationLease(const CommonQ4ActivationLease &) = delete;
    CommonQ4ActivationLease & operator=(const CommonQ4ActivationLease &) = delete;
    void reset();
    bool matches(int device, int k, int rows, InputType, uint64_t generation) const;
    size_t chunks() const;
    CommonQ4ActivationChunk chunk(size_t index) const;
    struct Impl;
private:
    Impl * impl_;
    friend bool common_q4_matmul_pair(CommonQ4Workspace &, int, void *, void *, const CommonQ4Weight &,
                                      const CommonQ4Weight &, const CommonQ4ActivationLease &, uint64_t);
    friend bool common_q4_prepare(CommonQ4Workspace &, int, const void *, int, int, InputType, uint64_t,
                                  CommonQ4ActivationLease &);
    friend bool common_q4_matmul_shared(CommonQ4Workspace &, int, void *, const CommonQ4Weight &,
                                        const CommonQ4ActivationLease &, uint64_t);
};
// False (and a rejected call counted) for an unsupported descriptor; no launch.
bool common_q4_prepare(CommonQ4Workspace &, int device, const void * input, int k, int rows,
                       InputType, uint64_t generation, CommonQ4ActivationLease &);
// False means no output was written (stale lease, wrong weight or overlap).
bool common_q4_matmul_shared(CommonQ4Workspace &, int device, void * y, const CommonQ4Weight &,
                             const CommonQ4ActivationLease &, uint64_t generation);
// Gate/up pair over one prepared M = 1 F32 lease (reference k200.h:381-383,
// src/q4-pair.inc:9-80):
// y0 = X W0^T, y1 = X W1^T for the shapes the reference accepts (K4096 x
// N11008, K2048 x N5632, unpadded); false with a status otherwise.
bool common_q4_matmul_pair(CommonQ4Workspace &, int device, void * y0, void * y1, const CommonQ4Weight & w0,
                           const CommonQ4Weight & w1, const CommonQ4ActivationLease &, uint64_t generation);
CommonQ4PairStatistics common_q4_pair_statistics(const CommonQ4Workspace &);
CommonQ4PairStatus common_q4_pair_last_status(const CommonQ4Workspace &);

// ---------------------------------------------------------------------------
// Paged key-value cache and the operators on it and on logits (declared by this
// library; the reference's own cache entry points are not). All of them submit
// like matmul: select(device) + check(wait()) completes them. They return false,
// with no work submitted, for arguments that break the rules stated here or
// (the layouts' own rules) named by the *_reason functions, for a bad device, a
// Kernel bound to another one, overlapping ranges where none are allowed, and
// when a workspace cannot be allocated. Pointers are device memory.
//
// A pool holds F16 values of `pages` pages: value i of token t of head h of
// page p is element p * page_stride + h * head_stride + t * token_stride + i.
// Keys and values have a pool each, of the same layout. Either order within a
// page (a head's tokens together, or a token's heads together) and any padding
// may be given by the strides (in elements, multiples of 8); pools are 16-byte
// aligned. Sequence s of a table holds its tokens in the pages
// table[s * row_pages + token / page_tokens].
struct KVCacheLayout {
    int pages, page_tokens, heads, width;       // width: values of a head, a multiple of 8 up to 256
    int64_t page_stride, head_stride, token_stride;
};
// "" or the first rule broken: "shape", "stride", "byte extent".
const char * kv_cache_reason(const KVCacheLayout &);

// What the kernels met on `device` since the last call, completing its work
// first: 0, or a sum of 1 (a page id outside the pool; its tokens were left out),
// 2 (a sequence, position or length out of range, or a second entry for one sequence; left out or cut; or a block's tokens
// apart in a list of kv_append_f8) and 4 (no free page: the sequence kept its length, a fork's child is empty). -1: no such
// device.
int kv_cache_status(int device);

// One new token per sequence: y[s][h] = sum over tokens t of
// softmax_t(scale * q[s][h] . k[s][t]) v[s][t], query heads sharing key-value
// heads in equal groups (query head h uses head h / (query_heads / heads)).
// t runs over the sequence's lengths[s] tokens, or the last `window` of them
// (window 0: all); a sequence of length 0, and a row of which every weight is 0, give zeros. Pages before
// the window and past the length are not read. `longest` bounds the lengths
// (up to row_pages * page_tokens). q and y have rows of [query_heads][width] values of
// `type`, q_stride and y_stride elements apart. F32 q and y get sums and
// statistics in F32; queries and weights are factors of two F16 parts, which hold a query value to 2^-22 of itself or
// 2^-34 of its row's largest and a weight to 2^-22 of itself or 2^-39 of the largest, whichever is more. Infinities
// and what is not a number follow F32 products: an infinite value gives its infinity wherever its weight is above
// 2^-126 of the largest, an infinite key wherever the query's value is not 0. scale * log2(e) has to be finite.
struct PagedAttentionLayout {
    int sequences, query_heads, longest, window, row_pages;
    int64_t q_stride, y_stride;
    float scale;
    InputType type;
};
// "" or the first rule broken of the two layouts: those of kv_cache_reason,
// "type", "shape", "heads", "length", "scale", "stride".
const char * paged_attention_reason(const KVCacheLayout &, const PagedAttentionLayout &);
bool paged_attention(Kernel &, int device, void * y, const void * q, const void * k, const void * v,
                     const int * table, const int * lengths, const KVCacheLayout &, const PagedAttentionLayout &);

// Stores `tokens` new tokens: token i becomes token position[i] of sequence
// sequence[i], whose table row already holds the page. With rotary > 0 the first `rotary`
// values of each head of q and k are turned by the angle whose cosine and sine
// stand in row position[i] of two [positions][rotary / 2] F32 tables: pair j is
// values (2j, 2j + 1) (adjacent) or (j, j + rotary / 2) (halves). k, v rows of
// [heads][width] and q rows of [query_heads][width] values of `type` are
// *_stride elements apart, so that they may lie in one product's rows. Turned q
// goes to q_out (q may be null, then query_heads and the strides of q are ignored; q_out may be q with
// equal strides). k and v are rounded to F16 once. position null: token i is the
// newest, lengths[i] - 1, of sequence i (sequence null too, tokens <= sequences). A
// negative position or sequence marks a token that is left out; one out of range, or without a page
// in the pool, is left out whole and reported: nothing is stored and its row of q_out stays as it was. Two tokens of
// one call must not name one place.
enum class RotaryPairs { adjacent, halves };
struct KVAppendLayout {
    int tokens, sequences, row_pages, query_heads;
    int64_t q_stride, k_stride, v_stride, q_out_stride;
    int rotary, positions;
    RotaryPairs pairs;
    InputType type;
};
const char * kv_append_reason(const KVCacheLayout &, const KVAppendLayout &);
bool kv_append(Kernel &, int device, void * k_pool, void * v_pool, void * q_out, const void * q, const void * k,
               const void * v, const int * sequence, const int * position, const int * lengths, const int * table,
               const float * cosine, const float * sine, const KVCacheLayout &, const KVAppendLayout &);

// The pages of `sequences` sequences: table [sequences][row_pages] (-1 past a
// sequence's last page), lengths [sequences] in tokens, references [pages]
// (how many rows hold a page; 0: free). `layers` pools stand layer_stride
// elements apart and share the table. Lists are distinct sequences; entries out
// of range are left out and reported. New pages are the lowest free ones, in list order. Up to 2^30
// pages and sequences; kv_fork takes up to 65535 entries.
struct KVPagesLayout {
    int sequences, row_pages, layers;
    int64_t layer_stride;
};
const char * kv_pages_reason(const KVCacheLayout &, const KVPagesLayout &);
// Makes room for added[i] more tokens of sequence rows[i] and adds them to its length (of a sequence that is listed
// twice, by the first entry in range; the others are left out and reported). In list order: an entry whose pages are
// not there is refused and reported, and takes none from those after it.
bool kv_reserve(Kernel &, int device, int * table, int * lengths, int * references, const int * rows,
                const int * added, int count, const KVCacheLayout &, const KVPagesLayout &);
// children[i] continues parents[i] as it stood before the call: full pages are
// shared, a last page that is not full is copied to a page that was free before
// the call. What a child held is released. A sequence may be parent of several
// children, and a parent may itself be a child; of forks to one
// child the first in range is made, the others are left out and reported.
bool kv_fork(Kernel &, int device, void * k, void * v, int * table, int * lengths, int * references,
             const int * parents, const int * children, int count, const KVCacheLayout &, const KVPagesLayout &);
// Releases what the listed sequences hold: rows -1, lengths 0.
bool kv_free(Kernel &, int device, int * table, int * lengths, int * references, const int * rows, int count,
             const KVCacheLayout &, const KVPagesLayout &);
// Moves pages so that the U used ones are pages 0..U-1: the i-th free page below
// U takes the i-th used page from U up. Writes the rows and counts that result
// (table_out and references_out may be table and references) and U to *used.
bool kv_compact(Kernel &, int device, void * k, void * v, int * table_out, int * references_out, int * used,
                const int * table, const int * lengths, const int * references, const KVCacheLayout &,
                const KVPagesLayout &);
// Copies page sources[i] to destinations[i] in all layers (pairs with a negative
// entry are left out). No destination may be named twice or be a source.
bool kv_copy_pages(Kernel &, int device, void * k, void * v, const int * sources, const int * destinations,
                   int count, const KVCacheLayout &, const KVPagesLayout &);

// The same cache in 8 bits. A pool holds e4m3 codes (4 exponent and 3 mantissa bits, largest 448), a byte each, at the
// places that `cache` names for values. Beside it stands an F32 scale for every block_tokens tokens of a head:
// token t of head h of page p has scale [(p * heads + h) * (page_tokens / block_tokens) + t / block_tokens], and a value is its
// code times its scale. block_tokens is a power of two up to 64 that divides page_tokens. Pools are 16-byte, scales
// 4-byte aligned. Tables, lengths and counts are those of the F16 cache, with kv_reserve(cache) and kv_free(cache).
struct KVCacheF8Layout {
    KVCacheLayout cache;
    int block_tokens;
};
// "" or the first rule broken: those of kv_cache_reason, "block".
const char * kv_cache_f8_reason(const KVCacheF8Layout &);

// paged_attention over such a cache, with its rules and numerics: products run on the codes, which F16 holds exactly; a
// token's key scale multiplies its score, its value scale its weight, in F32, and the product of weight and value
// scale is held to 2^-22 of itself, 2^-38 of the largest one or 2^-149, whichever is most. Any finite F32 scales will do, within
// F32's range: weights below 2^-126 of the largest are 0, and a row whose values, weighted and summed before they are divided by
// the weights' sum, leave that range is infinite. A scale or a code that is not
// a number makes the rows that read it not a number. What stands past a row's length or before its window may be anything.
const char * paged_attention_f8_reason(const KVCacheF8Layout &, const PagedAttentionLayout &);
bool paged_attention_f8(Kernel &, int device, void * y, const void * q, const void * k, const void * v,
                        const float * k_scales, const float * v_scales, const int * table, const int * lengths,
                        const KVCacheF8Layout &, const PagedAttentionLayout &);

// kv_append into such a cache: the same arguments, rules and rows of q. A block's scale becomes the least power of
// two, 2^-64 or more, that takes the largest of its new tokens' values to at most 448, or what it was where the block
// holds earlier tokens and their scale (of either sign) is no smaller in size; where it grows, the earlier tokens' codes are
// rounded to the new one.
// A new value is rounded once, to the nearest code of its F64 rotation (ties to the even code; beside an earlier scale that
// is no power of two, which only another producer leaves, of the rotation rounded to odd in F32). A value that is not finite
// makes its block's scale, so all of the block, not a number, until the block is begun again. Tokens of one block must
// stand in consecutive entries of consecutive positions (some of which may be left out); what the block held from the first
// of them on is forgotten. A list that breaks this rule is reported, and the blocks concerned hold nothing of use.
// (query_heads * width / 8 + 512 * heads) * tokens stays below 2^31 - 1024; longer lists go in several calls, parted where a
// block begins.
const char * kv_append_f8_reason(const KVCacheF8Layout &, const KVAppendLayout &);
bool kv_append_f8(Kernel &, int device, void * k_pool, void * v_pool, float * k_scales, float * v_scales, void * q_out,
                  const void * q, const void * k, const void * v, const int * sequence, const int * position,
                  const int * lengths, const int * table, const float * cosine, const float * sine,
                  const KVCacheF8Layout &, const KVAppendLayout &);

// Reads tokens back: row i of k and v (rows of [heads][width] values of `type`, *_stride elements apart, of their own or
// side by side in common rows) becomes token position[i] of sequence[i], code times scale, rounded once where `type` is F16.
// Tokens are named as for kv_append (position null: the newest of each sequence), in any order; those left out, out of
// range or without a page leave their rows as they were, the latter two reported.
struct KVReadLayout {
    int tokens, sequences, row_pages;
    int64_t k_stride, v_stride;
    InputType type;
};
const char * kv_read_f8_reason(const KVCacheF8Layout &, const KVReadLayout &);
bool kv_read_f8(Kernel &, int device, void * k, void * v, const void * k_pool, const void * v_pool,
                const float * k_scales, const float * v_scales, const int * sequence, const int * position,
                const int * lengths, const int * table, const KVCacheF8Layout &, const KVReadLayout &);

// kv_fork, kv_compact and kv_copy_pages for such a cache: pages move with their scales. layer_stride counts codes; the
// layers' scales follow one another, pages * heads * (page_tokens / block_tokens) each. The first rule broken is one of
// kv_cache_f8_reason or kv_pages_reason.
const char * kv_pages_f8_reason(const KVCacheF8Layout &, const KVPagesLayout &);
bool kv_fork_f8(Kernel &, int device, void * k, void * v, float * k_scales, float * v_scales, int * table, int * lengths,
                int * references, const int * parents, const int * children, int count, const KVCacheF8Layout &,
                const KVPagesLayout &);
bool kv_compact_f8(Kernel &, int device, void * k, void * v, float * k_scales, float * v_scales, int * table_out,
                   int * references_out, int * used, const int * table, const int * lengths, const int * references,
                   const KVCacheF8Layout &, const KVPagesLayout &);
bool kv_copy_pages_f8(Kernel &, int device, void * k, void * v, float * k_scales, float * v_scales, const int * sources,
                      const int * destinations, int count, const KVCacheF8Layout &, const KVPagesLayout &);

// Logits before a token is chosen, F32, row by row: with n the times that token t
// stands among the row's first history_lengths[row] history entries and
// (r, f, p) = penalties[row], z = logits[t]; n > 0: z = z > 0 ? z / r : z * r; z
// -= n f + (n > 0) p; z += the value of the row's last bias entry for t; then
// -inf where bit t % 32 of mask word t / 32 is 0. penalties, history, bias_ids
// and mask may be null (nothing of the kind; the bias arrays go together, history
// needs penalties). history_stride and bias_stride are the lists' room as well: above 0 for a list that is given; a length
// out of it is cut and reported by kv_cache_status.
// mask_stride 0: one mask for all rows. Entries outside the vocabulary are left out. y may be logits
// (equal strides). Strides are elements between rows.
struct LogitsLayout {
    int rows, vocabulary;
    int64_t logits_stride, y_stride, history_stride, bias_stride, mask_stride;
};
const char * logits_reason(const LogitsLayout &);
bool process_logits(Kernel &, int device, void * y, const void * logits, const float * penalties,
                    const int * history, const int * history_lengths, const int * bias_ids,
                    const float * bias_values, const int * bias_lengths, const uint32_t * mask,
                    const LogitsLayout &);

// Same layout as the reference (reference k200.h:345-350): matmul submissions
// on devices 0 and 1, peer copy count and bytes.
struct Statistics {
    size_t matmuls[2];
    size_t peer_copies, peer_bytes;
};
Statistics statistics();
const char * version();

} // namespace kunlun
