// The head's losses on the device (PSK_OP_HEAD_XENT, PSK_OP_HEAD_DISTILL and their _VJP, include/presk_cuda.h):
// argument checks, workspaces, the division of the vocabulary into pieces, the launches. Kernels: psk_head.cuh.
#include "psk_head.h"
#include "psk_head_shape.h"
#include <algorithm>
#include <cstring>
#include <vector>
#include "psk_head.cuh"

namespace psk {
namespace {

using namespace head;

constexpr int64_t kPieceBytes = 512ll << 20; // what a piece's g (and copy of the head, where one is needed) may take

int64_t up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }

// One buffer of the executor's pool a call, handed out in pieces of 256-byte alignment. It goes back to the pool when
// the call returns: the pool hands it on to later work of the same stream only.
struct Slab {
    HeadContext &x;
    std::vector<std::pair<void **, size_t>> want;
    size_t total = 0;
    void *base = nullptr;
    explicit Slab(HeadContext &c) : x(c) {}
    ~Slab() { psk_exec_free(x.e, base); }
    template <class T>
    void need(T *&p, int64_t n)
    {
        p = nullptr;
        if (n <= 0) return;
        want.push_back({reinterpret_cast<void **>(&p), total});
        total += ((size_t)n * sizeof(T) + 255) & ~(size_t)255;
    }
    bool take()
    {
        if (want.empty()) return true;
        base = psk_exec_alloc(x.e, total);
        if (!base) return false;
        for (auto &w : want) *w.first = (uint8_t *)base + w.second;
        return true;
    }
};

// A matrix operand of a product: element (row, k) at row·ld + k (k_contiguous) or k·ld + row; planes `plane` apart.
struct Operand {
    const void *p;
    int64_t rows, k, ld;
    bool k_contiguous;
    int planes;
    int64_t plane;
};

bool map_of(HeadContext &x, CUtensorMap *map, const Operand &o, int f16, int box_rows)
{
    const uint64_t inner = (uint64_t)(o.k_contiguous ? o.k : o.rows), outer = (uint64_t)(o.k_contiguous ? o.rows : o.k);
    const uint64_t ld = (uint64_t)(outer == 1 ? up((int64_t)inner, 8) : o.ld); // one row: its stride is never walked
    cuuint64_t dims[4] = {inner, outer, (cuuint64_t)o.planes, 1};
    cuuint64_t strides[3] = {ld * 2, (cuuint64_t)(o.planes > 1 ? o.plane * 2 : ld * 2 * outer), 0};
    strides[2] = strides[1] * (cuuint64_t)o.planes;
    for (int i = 0; i < 3; ++i)
        if (strides[i] % 16 != 0 || strides[i] == 0) return false;
    cuuint32_t box[4] = {(cuuint32_t)BK, (cuuint32_t)(o.k_contiguous ? box_rows : BK), 1, 1};
    cuuint32_t estr[4] = {1, 1, 1, 1};
    return x.encode(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void *>(o.p), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int fail(HeadContext &x, int code, const std::string &msg)
{
    x.error = msg;
    return code;
}

#define HEAD_TRY(call)                                                                                        \
    do {                                                                                                      \
        cudaError_t err__ = (call);                                                                           \
        if (err__ != cudaSuccess) return fail(x, PSK_E10001, std::string(#call) + ": " + cudaGetErrorString(err__)); \
    } while (0)

template <int MODE>
int product(HeadContext &x, Params P, const Operand &a, const Operand &b, int f16)
{
    CUtensorMap ma, mb;
    if (!map_of(x, &ma, a, f16, BM) || !map_of(x, &mb, b, f16, BN)) return fail(x, PSK_E10001, "head: an operand's layout does not make a tensor map");
    P.m = a.rows; P.n = b.rows;
    P.tiles_m = (P.m + BM - 1) / BM; P.tiles_n = (P.n + BN - 1) / BN;
    P.kb_k = (int32_t)((a.k + BK - 1) / BK);
    P.nprod = a.planes == 3 ? 6 : 1;
    if (MODE != MODE_OUT) { P.splits = 1; P.kb_split = P.kb_k; }
    P.chunk = P.nprod == 6 ? 6 : 4; // about 256 products of the summed axis an accumulator (see psk_head.cuh)
    // a panel's columns of b stay in a quarter of the L2 while a's rows stream past them
    P.panel = std::min<int64_t>(P.tiles_n, std::max<int64_t>(8, (32ll << 20) / std::max<int64_t>(1, BN * a.k * 2 * a.planes)));
    P.in_f16 = f16; P.a_m_major = !a.k_contiguous; P.b_n_major = !b.k_contiguous;
    P.status = x.status;
    HEAD_TRY(cudaFuncSetAttribute(k_head<MODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_TOTAL));
    const int64_t tiles = P.tiles_m * P.tiles_n * P.splits;
    k_head<MODE><<<(unsigned)std::min<int64_t>(tiles, x.sms), THREADS, SMEM_TOTAL, x.stream>>>(ma, mb, P);
    x.kernels += 1;
    x.flops += 2.0 * (double)P.m * (double)P.n * (double)a.k;
    return PSK_OK;
}

int grid_of(const HeadContext &x, int64_t work) { return (int)std::max<int64_t>(1, std::min<int64_t>((work + 255) / 256, (int64_t)x.sms * 8)); }

RowOperand row_operand(const psk_operand &o, void *base, int no)
{
    RowOperand r;
    memset(&r, 0, sizeof r);
    r.dtype = o.dtype;
    const int64_t eb = o.dtype == PSK_F64 || o.dtype == PSK_I64 ? 8 : o.dtype == PSK_F32 ? 4 : o.dtype == PSK_E8M15 ? 3 : 2;
    r.p = (const uint8_t *)base + o.offset * eb;
    for (int a = 0; a < no; ++a) r.stride[a] = o.stride[a];
    return r;
}

} // namespace

int head_run(HeadContext &x, const psk_launch *l, void *const *table)
{
    HeadShape h;
    if (const int rc = head_shape(l, h, x.error)) return rc;
    const std::string nm = l->name ? l->name : "head";
    if (!x.encode) return fail(x, PSK_E10001, "cuTensorMapEncodeTiled is not available from this driver");
    const bool vjp = h.vjp, distill = h.distill;
    const int no = l->n_outer, ax_v = no, ax_d = no + 1, ax_k = no + 2, first = h.first, dt = l->in[0].dtype;
    const int64_t V = h.classes, D = h.model, K = h.top, N = h.rows;
    const double tau = h.tau;
    const psk_operand &X = l->in[0], &W = l->in[1], &I = l->in[2], &O = l->out;
    const psk_operand *CT = h.ct >= 0 ? &l->in[h.ct] : nullptr, *LSE = h.lse >= 0 ? &l->in[h.lse] : nullptr, *DW = h.dw >= 0 ? &l->in[h.dw] : nullptr;
    RowSpace s;
    memset(&s, 0, sizeof s);
    s.no = no; s.rows = N;
    for (int a = 0; a < no; ++a) s.dims[a] = l->dims[a];
    cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
    HEAD_TRY(cudaStreamIsCapturing(x.stream, &capturing));
    if (capturing != cudaStreamCaptureStatusNone) return fail(x, PSK_E7005, nm + ": its workspace is the executor's, which a graph replayed later would share with other work; not while the stream is being captured");

    const int eb = dt == PSK_F32 ? 4 : 2, f16 = dt == PSK_F16, planes = dt == PSK_F32 ? 3 : 1;
    const float inv_tau = (float)(1.0 / tau);
    const RowOperand rx = row_operand(X, table[0], no), rids = row_operand(I, table[2], no);
    const uint8_t *wp = (const uint8_t *)table[1] + W.offset * eb;
    const int64_t w_v = W.stride[ax_v], w_d = W.stride[ax_d];
    const bool v_inner = w_v == 1 || V == 1; // the head as [model, classes]; otherwise rows of a class, [classes, model]
    auto aligned = [](const void *p) { return ((uintptr_t)p & 15u) == 0; };
    // read where it lies: 16-bit, one axis contiguous, rows on 16-byte boundaries
    const bool w_direct = planes == 1 && aligned(wp) && (v_inner ? w_v == 1 && w_d % 8 == 0 && w_d >= V : w_d == 1 && w_v % 8 == 0 && w_v >= D);
    // the rows of x one stride apart: one level over the outer axes
    bool x_rows = true;
    int64_t x_ld = 0;
    {
        int64_t want = 0;
        for (int a = no - 1; a >= 0; --a) {
            if (s.dims[a] == 1) continue;
            if (X.stride[a] == 0) { x_rows = false; break; }
            if (!want) { x_ld = X.stride[a]; want = x_ld * s.dims[a]; }
            else { x_rows = x_rows && X.stride[a] == want; want *= s.dims[a]; }
        }
        if (!x_ld) x_ld = up(D, 8);
    }
    const bool x_direct = !vjp && planes == 1 && x_rows && X.stride[ax_d] == 1 && x_ld % 8 == 0 && x_ld >= D && aligned(rx.p);

    // backward, few rows: g and what its rounding leaves as rows of their own in the same tile, which costs nothing there
    const int64_t Ng = vjp && planes == 1 && N <= BM / 2 ? 2 * N : N;
    const int64_t Dp = up(D, 8), Vp = up(V, 8);

    if (N == 0 && !vjp) return PSK_OK;

    // the vocabulary's pieces
    int64_t per_col = (vjp ? Ng * planes * 2 : 0) + (w_direct ? 0 : D * planes * 2);
    int64_t Vc = V;
    if (per_col > 0) {
        const int64_t most = std::max<int64_t>(BN, kPieceBytes / per_col / BN * BN);
        if (V > most) Vc = up((V + (V + most - 1) / most - 1) / ((V + most - 1) / most), BN);
    }
    const int64_t pieces = (V + Vc - 1) / Vc, halves = (V + COLS - 1) / COLS;
    const int64_t g_ld = up(Vc, 64), g_plane = planes == 3 ? Ng * g_ld : 0;
    const int64_t wc_ld = v_inner ? up(Vc, 8) : Dp, wc_plane = wc_ld * (v_inner ? D : Vc);
    const bool dw_v_inner = DW && (DW->stride[ax_v] == 1 || V == 1);
    const int64_t dwm = dw_v_inner ? D : Vc, dwn = dw_v_inner ? Vc : D, dw_ld = up(dwn, 4), dx_ld = up(D, 4);
    // splits of a product with few tiles along its summed axis, so that every SM has some of it
    auto splits_of = [&](int64_t m, int64_t n, int64_t k, int32_t &kb_split) {
        const int64_t tiles = ((m + BM - 1) / BM) * ((n + BN - 1) / BN), kb = (k + BK - 1) / BK;
        int64_t want = std::max<int64_t>(1, std::min<int64_t>(x.sms / tiles, kb / 4));
        kb_split = (int32_t)((kb + want - 1) / want);
        return (kb + kb_split - 1) / kb_split;
    };
    int32_t dx_kb = 1, dw_kb = 1;
    const int64_t dx_splits = vjp && N ? splits_of(Ng, D, Vc, dx_kb) : 1, dw_splits = DW && N ? splits_of(dwm, dwn, Ng, dw_kb) : 1;

    int32_t *label, *ids;
    float *p, *plogp, *coef, *lse2, *hit, *dxp, *dwp;
    float2 *part;
    uint16_t *xc, *wc, *g;
    uint32_t *words;
    Slab slab(x);
    slab.need(label, distill ? 0 : N);
    slab.need(ids, distill ? N * K : 0);
    slab.need(p, distill ? N * K : 0);
    slab.need(plogp, distill ? N : 0);
    slab.need(coef, vjp ? N : 0);
    slab.need(lse2, vjp ? N : 0);
    slab.need(part, vjp ? 0 : halves * N);
    slab.need(hit, vjp ? 0 : distill ? halves * N : N);
    slab.need(xc, x_direct ? 0 : Ng * Dp * planes);
    slab.need(wc, w_direct || !N ? 0 : wc_plane * planes);
    slab.need(g, vjp ? Ng * g_ld * planes : 0);
    slab.need(dxp, vjp && N ? dx_splits * Ng * dx_ld : 0);
    slab.need(dwp, DW && N ? dw_splits * dwm * dw_ld : 0);
    slab.need(words, 3); // the greatest |ct/τ|, binary16's scale and its reciprocal
    if (!slab.take()) return fail(x, PSK_E10001, nm + ": no memory for a workspace of " + std::to_string(slab.total) + " bytes (" + psk_last_error(x.e) + ")");

    // 1. targets
    const bool scaled = vjp && f16;
    if (N > 0) {
        RowOperand rct{}, rlse{};
        if (vjp) { rct = row_operand(*CT, table[first], no); rlse = row_operand(*LSE, table[first + 1], no); }
        if (scaled) HEAD_TRY(cudaMemsetAsync(words, 0, 4, x.stream));
        if (distill) {
            TeacherParams T;
            memset(&T, 0, sizeof T);
            T.s = s; T.ids = rids; T.t = row_operand(l->in[3], table[3], no); T.ct = rct; T.lse = rlse;
            T.ids_k = I.stride[ax_k]; T.t_k = l->in[3].stride[ax_k]; T.classes = V; T.top = (int32_t)K; T.inv_tau = inv_tau;
            T.out_ids = ids; T.out_p = p; T.plogp = plogp; T.coef = coef; T.lse2 = lse2; T.status = x.status; T.ctmax = scaled ? words : nullptr;
            k_head_teacher<<<(unsigned)N, (unsigned)up(K, 32), (size_t)K * 4, x.stream>>>(T);
        } else {
            LabelParams T;
            memset(&T, 0, sizeof T);
            T.s = s; T.ids = rids; T.ct = rct; T.lse = rlse; T.classes = V; T.inv_tau = inv_tau;
            T.label = label; T.coef = coef; T.lse2 = lse2; T.status = x.status; T.ctmax = scaled ? words : nullptr;
            k_head_labels<<<(unsigned)((N + 255) / 256), 256, 0, x.stream>>>(T);
        }
        x.kernels += 1;
        if (scaled) { k_head_scale<<<1, 1, 0, x.stream>>>(words, words + 1); x.kernels += 1; }
    }

    // 2. x where its layout (or a row without a target, backward) asks for a copy
    Operand a{rx.p, N, D, x_ld, true, planes, 0};
    if (!x_direct && N > 0) {
        PackParams k;
        memset(&k, 0, sizeof k);
        k.s = s; k.src = rx; k.col_stride = X.stride[ax_d]; k.cols = D; k.ld = Dp; k.plane = Ng * Dp; k.dst = xc; k.f32 = planes == 3; k.copies = (int32_t)(Ng / N);
        if (vjp) { k.label = label; k.ids = ids; k.top = (int32_t)K; }
        k_head_pack<<<grid_of(x, N * Dp / 8), 256, 0, x.stream>>>(k);
        x.kernels += 1;
        a = Operand{xc, N, D, Dp, true, planes, Ng * Dp};
    }

    const RowOperand rout = row_operand(O, table[l->n_inputs], no);
    for (int64_t piece = 0; piece < pieces && N > 0; ++piece) {
        const int64_t v0 = piece * Vc, vn = std::min(Vc, V - v0);
        // 3. the piece of the head
        Operand b{wp + v0 * w_v * 2, vn, D, v_inner ? w_d : w_v, !v_inner, planes, 0};
        if (!w_direct) {
            PackParams k;
            memset(&k, 0, sizeof k);
            k.s.no = 1; k.s.rows = k.s.dims[0] = v_inner ? D : vn;
            k.src.p = wp + v0 * w_v * eb; k.src.dtype = dt; k.src.stride[0] = v_inner ? w_d : w_v;
            k.col_stride = v_inner ? w_v : w_d; k.cols = v_inner ? vn : D; k.ld = wc_ld; k.plane = wc_plane; k.dst = wc; k.f32 = planes == 3; k.copies = 1;
            k_head_pack<<<grid_of(x, k.s.rows * wc_ld / 8), 256, 0, x.stream>>>(k);
            x.kernels += 1;
            b = Operand{wc, vn, D, wc_ld, !v_inner, planes, wc_plane};
        }
        // 4. the logits' tiles
        Params P;
        memset(&P, 0, sizeof P);
        P.c = (float)(1.4426950408889634 / tau); P.rows = N; P.col0 = v0;
        P.label = label; P.ids = ids; P.p = p; P.top = (int32_t)K;
        if (!vjp) {
            P.part = part; P.hit = hit; P.part0 = 2 * (v0 / BN);
            const int r = product<MODE_STATS>(x, P, a, b, f16);
            if (r != PSK_OK) return r;
            continue;
        }
        P.lse2 = lse2; P.coef = coef; P.scale = scaled ? words + 1 : nullptr;
        P.g = g; P.g_ld = g_ld; P.g_plane = g_plane; P.g_lo = Ng > N ? N : 0;
        int r = product<MODE_GRAD>(x, P, a, b, f16);
        if (r != PSK_OK) return r;
        // 5. dx += g·wᵀ over the piece: both operands along the classes
        Operand gk{g, Ng, vn, g_ld, true, planes, g_plane};
        Operand wk{b.p, D, vn, b.ld, v_inner, planes, b.plane};
        Params Q;
        memset(&Q, 0, sizeof Q);
        Q.splits = dx_splits; Q.kb_split = dx_kb; Q.out = dxp; Q.out_ld = dx_ld; Q.accumulate = piece > 0;
        if ((vn + BK - 1) / BK < (Vc + BK - 1) / BK) { // the last piece is shorter: as many splits as still have a block
            Q.splits = ((vn + BK - 1) / BK + dx_kb - 1) / dx_kb;
        }
        r = product<MODE_OUT>(x, Q, gk, wk, f16);
        if (r != PSK_OK) return r;
        // 6. dw of the piece = xᵀ·g: both operands along the rows
        if (DW) {
            Operand xr{xc, D, Ng, Dp, false, planes, Ng * Dp}, gr{g, vn, Ng, g_ld, false, planes, g_plane};
            memset(&Q, 0, sizeof Q);
            Q.splits = dw_splits; Q.kb_split = dw_kb; Q.out = dwp; Q.out_ld = dw_ld;
            r = product<MODE_OUT>(x, Q, dw_v_inner ? xr : gr, dw_v_inner ? gr : xr, f16);
            if (r != PSK_OK) return r;
            SumParams S;
            memset(&S, 0, sizeof S);
            S.s.no = 1; S.s.rows = S.s.dims[0] = dw_v_inner ? D : vn;
            S.part = dwp; S.parts = dw_splits; S.part_rows = S.s.rows; S.ld = dw_ld; S.cols = dw_v_inner ? vn : D;
            S.col_stride = DW->stride[dw_v_inner ? ax_v : ax_d]; S.scale = scaled ? words + 1 : nullptr;
            S.dst.p = (const uint8_t *)table[first + 2] + (DW->offset + v0 * DW->stride[ax_v]) * eb; S.dst.dtype = dt; S.dst.stride[0] = DW->stride[dw_v_inner ? ax_d : ax_v];
            S.ovf = x.ovf; S.guarded = x.guarded;
            k_head_sum<<<grid_of(x, S.s.rows * S.cols), 256, 0, x.stream>>>(S);
            x.kernels += 1;
        }
    }
    if (!vjp) {
        JoinParams J;
        memset(&J, 0, sizeof J);
        J.s = s; J.halves = halves; J.part = part; J.hit = hit; J.label = label; J.ids = ids; J.plogp = plogp; J.top = (int32_t)K; J.inv_tau = inv_tau;
        J.loss = rout; J.ovf = x.ovf; J.guarded = x.guarded;
        if (LSE) J.lse = row_operand(*LSE, table[first], no);
        k_head_join<<<(unsigned)((N + 31) / 32), 256, 0, x.stream>>>(J);
        x.kernels += 1;
    } else if (N > 0) {
        SumParams S;
        memset(&S, 0, sizeof S);
        S.s = s; S.part = dxp; S.parts = dx_splits; S.part_rows = Ng; S.ld = dx_ld; S.fold = Ng > N ? N : 0; S.cols = D; S.col_stride = O.stride[ax_d];
        S.scale = scaled ? words + 1 : nullptr; S.dst = rout; S.ovf = x.ovf; S.guarded = x.guarded;
        k_head_sum<<<grid_of(x, N * D), 256, 0, x.stream>>>(S);
        x.kernels += 1;
    } else if (DW) { // no rows: a gradient of zeros
        SumParams S;
        memset(&S, 0, sizeof S);
        S.s.no = 1; S.s.rows = S.s.dims[0] = D; S.cols = V; S.col_stride = DW->stride[ax_v];
        S.dst.p = (const uint8_t *)table[first + 2] + DW->offset * eb; S.dst.dtype = dt; S.dst.stride[0] = DW->stride[ax_d];
        k_head_sum<<<grid_of(x, D * V), 256, 0, x.stream>>>(S);
        x.kernels += 1;
    }
    HEAD_TRY(cudaGetLastError());
    return PSK_OK;
}

} // namespace psk
