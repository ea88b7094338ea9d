// C entry points of the int8 products and of the routing of tokens to experts (include/inferencequant_b200.h): argument checks,
// workspace layout, order of launches.
#include <climits>

#include "int8.cuh"

namespace b200q {

static constexpr long long pad_to(long long v, long long to) { return (v + to - 1) / to * to; }
static bool elem_ok(int elem) { return elem == ELEM_F32 || elem == ELEM_F16 || elem == ELEM_BF16; }
static bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
static int cuda_result(cudaError_t e) { return e == cudaSuccess ? B200Q_OK : set_error((int)e, cudaGetErrorString(e)); }

static int check_int8_rows(const void* q, long long ldq, int k, const char* what) {
    if (!aligned(q, 16) || ldq % 16 != 0 || ldq < pad_to(k, 16)) return set_error(B200Q_ERR_INVALID, what);
    return B200Q_OK;
}
static int check_k(int k) {
    if (k < 1) return set_error(B200Q_ERR_INVALID, "k must be positive");
    if (k > INT8_MAX_K) return set_error(B200Q_ERR_UNSUPPORTED, "sums of more than 131071 int8 products do not fit 32 bits");
    return B200Q_OK;
}
// a step over a row's columns is less than 2^20 of them
static bool columns_ok(int h) { return h >= 0 && h <= INT_MAX - (1 << 20); }
static int check_routing(long long tokens, int topk, int experts) {
    if (tokens < 0 || topk < 1) return set_error(B200Q_ERR_INVALID, "a negative number of tokens, or no slots");
    if (experts < 1 || experts > INT8_MAX_EXPERTS) return set_error(B200Q_ERR_UNSUPPORTED, "1 to 1024 experts");
    if (tokens * topk > INT_MAX - 65536) return set_error(B200Q_ERR_TOO_LARGE, "more than 2^31 slots");
    return B200Q_OK;
}

static int int8_product(int elem, const Int8Product& p, cudaStream_t s, bool dependent) {
    if (int8_rows_pays(p) || !int8_pair_ready()) return cuda_result(int8_product_rows(elem, p, s, dependent));
    return int8_product_pair(elem, p, s, dependent);
}

// What the experts' layer keeps between its launches, one region after the other, each on a 256-byte boundary.
struct ExpertsWorkspace {
    int *order, *offsets, *position;
    int8_t *xq, *hq;
    float *xs, *hs, *y;
    void* hidden;
    long long ldx, ldh, ldy, bytes;
};
static ExpertsWorkspace experts_workspace(void* base, int elem, long long slots, int experts, int hidden, int ffn) {
    ExpertsWorkspace w{};
    uint8_t* p = static_cast<uint8_t*>(base);
    long long used = 0;
    const auto take = [&](long long bytes) {
        void* at = p + used;
        used += pad_to(bytes, 256);
        return at;
    };
    w.ldx = pad_to(hidden, 16);
    w.ldh = pad_to(ffn, 16);
    w.ldy = pad_to(hidden, 4);
    w.order = static_cast<int*>(take(slots * 4));
    w.offsets = static_cast<int*>(take((experts + 1) * 4));
    w.position = static_cast<int*>(take(slots * 4));
    w.xs = static_cast<float*>(take(slots * 4));
    w.hs = static_cast<float*>(take(slots * 4));
    // the tokens' integers are done with when the hidden values' are written, and these when the outputs are
    const long long hidden_bytes = w.ldh * (elem == ELEM_F32 ? 4 : 2), y_bytes = w.ldy * 4;
    w.xq = w.hq = static_cast<int8_t*>(take(slots * (w.ldx > w.ldh ? w.ldx : w.ldh)));
    w.hidden = take(slots * (hidden_bytes > y_bytes ? hidden_bytes : y_bytes));
    w.y = static_cast<float*>(w.hidden);
    w.bytes = used;
    return w;
}

}  // namespace b200q

using namespace b200q;

extern "C" {

int b200q_int8_quantize(int elem, const void* x, long long ldx, void* q, long long ldq, float* scales, long long rows, int k, void* stream) {
    if (!elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "values are f32, f16 or bf16");
    if (const int rc = check_k(k)) return rc;
    if (rows < 0 || rows > INT_MAX || ldx < k) return set_error(B200Q_ERR_INVALID, "bad number of rows, or rows that overlap");
    if (rows == 0) return B200Q_OK;
    if (!x || !q || !scales) return set_error(B200Q_ERR_INVALID, "null pointer");
    if (const int rc = check_int8_rows(q, ldq, k, "int8 rows start on 16-byte boundaries and are a multiple of 16 bytes apart")) return rc;
    return cuda_result(int8_quantize_rows(elem, x, ldx, static_cast<int8_t*>(q), ldq, scales, rows, k, nullptr, 1, nullptr, (cudaStream_t)stream, false));
}

int b200q_int8_dequantize(int elem, const void* q, long long ldq, const float* scales, void* out, long long rows, int k, void* stream) {
    if (!elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "values are f32, f16 or bf16");
    if (const int rc = check_k(k)) return rc;
    if (rows < 0 || rows > INT_MAX) return set_error(B200Q_ERR_INVALID, "bad number of rows");
    if (rows == 0) return B200Q_OK;
    if (!q || !scales || !out) return set_error(B200Q_ERR_INVALID, "null pointer");
    if (const int rc = check_int8_rows(q, ldq, k, "int8 rows start on 16-byte boundaries and are a multiple of 16 bytes apart")) return rc;
    return cuda_result(int8_dequantize_rows(elem, static_cast<const int8_t*>(q), ldq, scales, out, rows, k, (cudaStream_t)stream));
}

int b200q_int8_gemm(int elem, const void* xq, const float* xs, const void* wq, const float* ws, void* y, int rows, int n, int k, long long ldx,
                    long long ldw, long long ldy, const int* offsets, int experts, void* stream) {
    if (!elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "outputs are f32, f16 or bf16");
    if (const int rc = check_k(k)) return rc;
    if (rows < 0 || n < 0 || ldy < n) return set_error(B200Q_ERR_INVALID, "bad shape");
    if (experts < 1 || experts > INT8_MAX_EXPERTS || (long long)experts * n > INT_MAX - 512) return set_error(B200Q_ERR_UNSUPPORTED, "1 to 1024 matrices of 2^31 rows in all");
    if (experts > 1 && !offsets) return set_error(B200Q_ERR_INVALID, "several matrices need offsets");
    if (rows == 0 || n == 0) return B200Q_OK;
    if (!xq || !xs || !wq || !ws || !y) return set_error(B200Q_ERR_INVALID, "null pointer");
    const char* align = "int8 rows start on 16-byte boundaries and are a multiple of 16 bytes apart";
    if (const int rc = check_int8_rows(xq, ldx, k, align)) return rc;
    if (const int rc = check_int8_rows(wq, ldw, k, align)) return rc;
    if (ldx > INT_MAX || ldw > INT_MAX) return set_error(B200Q_ERR_INVALID, "rows too far apart");
    const Int8Product p{static_cast<const int8_t*>(xq), xs, static_cast<const int8_t*>(wq), ws, y, offsets, rows, n, k, (int)ldx, (int)ldw, experts, INT8_ACT_NONE, n, ldy, status_ptr(), false, nullptr, false};
    return int8_product(elem, p, (cudaStream_t)stream, false);
}

long long b200q_int8_matmul_workspace_bytes(int m, int k) {
    if (m < 1 || k < 1) return 0;
    return pad_to((long long)m * 4, 256) + m * pad_to(k, 16);
}

int b200q_int8_matmul(int elem, const void* x, const void* wq, const float* ws, void* y, int m, int n, int k, long long ldx, long long ldw,
                      long long ldy, void* workspace, long long workspace_bytes, void* stream) {
    if (!elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "activations are f32, f16 or bf16");
    if (const int rc = check_k(k)) return rc;
    if (m < 0 || n < 0 || ldx < k || ldy < n) return set_error(B200Q_ERR_INVALID, "bad shape");
    if (m == 0 || n == 0) return B200Q_OK;
    if (!x || !wq || !ws || !y || !workspace) return set_error(B200Q_ERR_INVALID, "null pointer");
    if (!aligned(workspace, 128)) return set_error(B200Q_ERR_INVALID, "the workspace must be 128-byte aligned");
    if (workspace_bytes < b200q_int8_matmul_workspace_bytes(m, k)) return set_error(B200Q_ERR_TOO_LARGE, "workspace too small");
    if (const int rc = check_int8_rows(wq, ldw, k, "int8 rows start on 16-byte boundaries and are a multiple of 16 bytes apart")) return rc;
    if (ldw > INT_MAX) return set_error(B200Q_ERR_INVALID, "rows too far apart");
    cudaStream_t s = (cudaStream_t)stream;
    float* xs = static_cast<float*>(workspace);
    int8_t* xq = static_cast<int8_t*>(workspace) + pad_to((long long)m * 4, 256);
    const long long kp = pad_to(k, 16);
    const cudaError_t e = int8_quantize_rows(elem, x, ldx, xq, kp, xs, m, k, nullptr, 1, nullptr, s, false);
    if (e != cudaSuccess) return cuda_result(e);
    const Int8Product p{xq, xs, static_cast<const int8_t*>(wq), ws, y, nullptr, m, n, k, (int)kp, (int)ldw, 1, INT8_ACT_NONE, n, ldy, status_ptr(), false, nullptr, false};
    return int8_product(elem, p, s, true);
}

int b200q_route_sort(const void* ids, int id_bytes, int slots, int experts, int* order, int* offsets, int* position, void* stream) {
    if (id_bytes != 4 && id_bytes != 8) return set_error(B200Q_ERR_UNSUPPORTED, "expert ids have 4 or 8 bytes");
    if (const int rc = check_routing(slots, 1, experts)) return rc;
    if (!offsets || (slots > 0 && (!ids || !order || !position))) return set_error(B200Q_ERR_INVALID, "null pointer");
    return cuda_result(route_sort(ids, id_bytes == 8, slots, experts, order, offsets, position, (cudaStream_t)stream));
}

int b200q_route_dispatch(int elem, const void* x, long long ldx, const int* position, const int* offsets, int experts, void* rows, int tokens,
                         int topk, int h, void* stream) {
    if (!elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "rows are f32, f16 or bf16");
    if (const int rc = check_routing(tokens, topk, experts)) return rc;
    if (!columns_ok(h) || ldx < h) return set_error(B200Q_ERR_INVALID, "bad shape");
    if (tokens == 0 || h == 0) return B200Q_OK;
    if (!x || !position || !offsets || !rows) return set_error(B200Q_ERR_INVALID, "null pointer");
    return cuda_result(route_dispatch(elem, x, ldx, position, offsets + experts, rows, tokens, topk, h, (cudaStream_t)stream));
}

int b200q_route_combine(int elem_in, int elem_out, const void* rows, long long ldr, const int* position, const float* weights, void* out, int tokens,
                        int topk, int h, void* stream) {
    if (!elem_ok(elem_in) || !elem_ok(elem_out)) return set_error(B200Q_ERR_UNSUPPORTED, "rows are f32, f16 or bf16");
    if (const int rc = check_routing(tokens, topk, 1)) return rc;
    if (!columns_ok(h) || ldr < h) return set_error(B200Q_ERR_INVALID, "bad shape");
    if (tokens == 0 || h == 0) return B200Q_OK;
    if (!rows || !position || !out) return set_error(B200Q_ERR_INVALID, "null pointer");
    return cuda_result(route_combine(elem_in, elem_out, rows, ldr, position, weights, out, tokens, topk, h, (cudaStream_t)stream, false));
}

int b200q_route_combine_grad(int elem_grad, int elem, const void* grad_out, long long ldg, const void* rows, long long ldr, const int* position,
                             const int* offsets, int experts, const float* weights, void* grad_rows, float* grad_weights, int tokens, int topk,
                             int h, void* stream) {
    if (!elem_ok(elem_grad) || !elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "rows are f32, f16 or bf16");
    if (const int rc = check_routing(tokens, topk, experts)) return rc;
    if (!columns_ok(h) || ldg < h || (grad_weights && ldr < h)) return set_error(B200Q_ERR_INVALID, "bad shape");
    if (tokens == 0 || (!grad_rows && !grad_weights)) return B200Q_OK;
    if (!position || !offsets || !weights || (h > 0 && (!grad_out || (grad_weights && !rows)))) return set_error(B200Q_ERR_INVALID, "null pointer");
    return cuda_result(route_combine_grad(elem_grad, elem, grad_out, ldg, rows, ldr, position, offsets + experts, weights, grad_rows, grad_weights, tokens, topk, h, (cudaStream_t)stream));
}

long long b200q_int8_experts_workspace_bytes(int elem, int tokens, int topk, int experts, int hidden, int ffn) {
    if (!elem_ok(elem) || tokens < 1 || topk < 1 || experts < 1 || hidden < 1 || ffn < 1) return 0;
    return experts_workspace(nullptr, elem, (long long)tokens * topk, experts, hidden, ffn).bytes;
}

int b200q_int8_experts(int elem, int activation, const void* x, long long ldx, const void* ids, int id_bytes, const float* weights,
                       const void* gate_up, const float* gate_up_scales, const void* down, const float* down_scales, void* out, int tokens,
                       int experts, int topk, int hidden, int ffn, void* workspace, long long workspace_bytes, void* stream) {
    if (!elem_ok(elem)) return set_error(B200Q_ERR_UNSUPPORTED, "activations are f32, f16 or bf16");
    if (activation < INT8_ACT_SILU || activation > INT8_ACT_SIGMOID) return set_error(B200Q_ERR_INVALID, "unknown activation");
    if (id_bytes != 4 && id_bytes != 8) return set_error(B200Q_ERR_UNSUPPORTED, "expert ids have 4 or 8 bytes");
    if (const int rc = check_routing(tokens, topk, experts)) return rc;
    if (const int rc = check_k(hidden)) return rc;
    if (const int rc = check_k(ffn)) return rc;
    if (ldx < hidden) return set_error(B200Q_ERR_INVALID, "bad shape");
    const int pairs = (int)pad_to(ffn, 8);
    if ((long long)experts * 2 * pairs > INT_MAX - 512 || (long long)experts * hidden > INT_MAX - 512) return set_error(B200Q_ERR_UNSUPPORTED, "matrices of 2^31 rows in all");
    if (tokens == 0) return B200Q_OK;
    if (!x || !ids || !weights || !gate_up || !gate_up_scales || !down || !down_scales || !out || !workspace) return set_error(B200Q_ERR_INVALID, "null pointer");
    if (!aligned(workspace, 128)) return set_error(B200Q_ERR_INVALID, "the workspace must be 128-byte aligned");
    if (!aligned(gate_up, 16) || !aligned(down, 16)) return set_error(B200Q_ERR_INVALID, "int8 rows start on 16-byte boundaries");
    const int slots = tokens * topk;
    const ExpertsWorkspace w = experts_workspace(workspace, elem, slots, experts, hidden, ffn);
    if (workspace_bytes < w.bytes) return set_error(B200Q_ERR_TOO_LARGE, "workspace too small");
    cudaStream_t s = (cudaStream_t)stream;
    // Where the experts' rows begin is known to the products: the launch before has waited for the one that wrote it, or, where the
    // quantizer does, the product of gate and up counts the ids for itself while there are few, in all and of an expert. us, waiting ->
    // counting: 1 token through 2 of 8 experts of 4096 x 14336 66.3 -> 65.0, 1 through 8 of 128 of 2048 x 768 20.1 -> 18.5, 64 through 8 of
    // 128 100.5 -> 98.2, 128 of them 115.2 -> 114.3, but 256 122.1 -> 125.4, and 190 through 2 of 8 of 1024 x 512 21.4 -> 22.0.
    const bool routes = int8_routes_quantizing(tokens, topk, hidden), counts = routes && experts > 1 && slots <= 1024 && slots <= 12 * experts;
    const Int8Product up{w.xq, w.xs, static_cast<const int8_t*>(gate_up), gate_up_scales, w.hidden, w.offsets, slots, 2 * pairs, hidden, (int)w.ldx, (int)w.ldx, experts, activation, ffn, w.ldh, status_ptr(), !routes || counts, counts ? ids : nullptr, id_bytes == 8};
    const Int8Product dn{w.hq, w.hs, static_cast<const int8_t*>(down), down_scales, w.y, w.offsets, slots, hidden, ffn, (int)w.ldh, (int)w.ldh, experts, INT8_ACT_NONE, hidden, w.ldy, status_ptr(), true, nullptr, false};
    if (routes) {
        if (const int rc = cuda_result(int8_route_quantize(elem, x, ldx, w.xq, w.ldx, w.xs, tokens, hidden, ids, id_bytes == 8, topk, experts, w.position, w.offsets, s))) return rc;
    } else {
        if (const int rc = cuda_result(route_sort(ids, id_bytes == 8, slots, experts, w.order, w.offsets, w.position, s))) return rc;
        if (const int rc = cuda_result(int8_quantize_rows(elem, x, ldx, w.xq, w.ldx, w.xs, tokens, hidden, w.position, topk, nullptr, s, true))) return rc;
    }
    if (const int rc = int8_product(elem, up, s, true)) return rc;
    if (const int rc = cuda_result(int8_quantize_rows(elem, w.hidden, w.ldh, w.hq, w.ldh, w.hs, slots, ffn, nullptr, 1, w.offsets + experts, s, true))) return rc;
    if (const int rc = int8_product(ELEM_F32, dn, s, true)) return rc;
    return cuda_result(route_combine(ELEM_F32, elem, w.y, w.ldy, w.position, weights, out, tokens, topk, hidden, s, true));
}

}  // extern "C"
