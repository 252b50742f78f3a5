// Node execution of the sequence model operators: operands and shapes are checked here, results
// created, parameters gathered where several ranks take part, and the kernel launched.
//
// All of them work row by row of dimension 0 (tokens, or sequences), which is the dimension that
// arrays are partitioned along: a rank computes the rows that it owns, and only the parameters
// (weights, A, D, ...), whose dimension 0 is the channels, are gathered onto every rank.
#include <algorithm>
#include <cstring>
#include <initializer_list>

#include "context.hpp"
#include "sequence.hpp"

namespace cn {

struct Context::SeqArg {
    Array* a = nullptr;       // null: a literal, or left out
    double value = 0;
    const void* whole = nullptr;  // all of the array on this rank (seq_whole)
    explicit operator bool() const { return a != nullptr; }
    const void* data() const { return a ? a->buf.data : nullptr; }
};

namespace {

int acc_type(int dtype) { return dtype == DT_F64 ? DT_F64 : DT_F32; }
bool activation_type(int dtype) { return dtype == DT_F16 || dtype == DT_F32 || dtype == DT_F64; }

bool has_shape(const Array* a, std::initializer_list<int64_t> shape) {
    if (a->ndims != (int)shape.size()) return false;
    int d = 0;
    for (int64_t s : shape)
        if (a->shape[d++] != s) return false;
    return true;
}

}  // namespace

// Operand i of the node's first root: a whole array, or a literal.
int Context::seq_arg(const DagNode& node, size_t i, SeqArg* out) {
    const Operand& op = node.roots[0]->operands[i];
    if (op.is_ref || !op.leaf) return fail(CN_ERR_BAD_BLOB, "operand must name an array or be a literal");
    if (op.leaf->is_scalar) {
        out->a = nullptr;
        out->value = op.leaf->scalar;
        return CN_OK;
    }
    Region r;
    int rc = operand_array(op, &out->a, &r);
    if (rc) return rc;
    for (int d = 0; d < out->a->ndims; ++d)
        if (r.start[d] != 0 || r.stop[d] != out->a->shape[d] || r.step[d] != 1)
            return fail(CN_ERR_UNSUPPORTED, "this operator takes whole arrays; assign the view to an array first");
    return CN_OK;
}

// The results (roots) must be none of the operands and none of each other; with a state that is updated in place the
// second one is the state itself, which then is no other operand.  Checked before any result is made.
int Context::seq_names(const DagNode& node, const Array* in_place) {
    const auto& operands = node.roots[0]->operands;
    for (size_t i = 0; i < node.roots.size(); ++i) {
        const int name = node.roots[i]->result_name;
        size_t own = 0;
        for (auto& op : operands) own += op.leaf && !op.leaf->is_scalar && op.leaf->result_name == name;
        if (in_place && i == 1) {
            if (own > 1) return fail(CN_ERR_HAZARD, "a state that is updated in place is also another operand");
        } else if (own) {
            return fail(CN_ERR_HAZARD, "a result of this operator is one of its operands");
        }
        for (size_t j = 0; j < i; ++j)
            if (node.roots[j]->result_name == name) return fail(CN_ERR_HAZARD, "two results of this operator are the same array");
    }
    return CN_OK;
}

// Result i of the node (root i).
int Context::seq_result(const DagNode& node, size_t i, int ndims, const int64_t* shape, int dtype, Array** out) {
    int rc = create_array(node.roots[i]->result_name, ndims, shape, dtype, false, out);
    if (rc) return rc;
    (*out)->mark_written();
    return CN_OK;
}

// The whole of each array on this rank, side by side in the scratch buffer where there are several.
int Context::seq_whole(std::initializer_list<SeqArg*> args) {
    size_t bytes = 0;
    for (SeqArg* p : args) {
        if (!p->a) continue;
        p->whole = p->a->buf.data;
        if (nranks_ > 1 && !p->a->replicated) bytes += ((size_t)p->a->global_elems() * dtype_size(p->a->dtype) + 255) / 256 * 256;
    }
    if (!bytes) return CN_OK;
    if (!comm_.ready) return fail(CN_ERR_COMM, "this operator needs cn_comm_init first on several ranks");
    int rc = ensure_scratch(bytes);
    if (rc) return rc;
    CommGroup group(&err_);
    if ((rc = group.started())) return rc;
    size_t off = 0;
    for (SeqArg* p : args) {
        if (!p->a || p->a->replicated) continue;
        const size_t esz = dtype_size(p->a->dtype);
        char* to = (char*)scratch_ + off;
        for (int q = 0; q < nranks_; ++q) {
            int64_t b, e;
            partition(p->a->shape[0], &b, &e, q);
            if (e <= b) continue;
            if ((rc = comm_broadcast(&comm_, p->a->buf.data, to + (size_t)b * p->a->unit * esz, (e - b) * p->a->unit,
                                     p->a->dtype, q, stream_, &err_)))
                return rc;
        }
        p->whole = to;
        off += ((size_t)p->a->global_elems() * esz + 255) / 256 * 256;
    }
    return group.end();
}

// Several ranks: a rank computes the rows of x that it owns.  That needs rows (a 1-D array is
// partitioned along its only row), every operand on each rank that computes, and the results there
// and nowhere else: arrays of one element, which live on every rank, must not meet others.
int Context::seq_rows(const Array& x, std::initializer_list<const Array*> operands, std::initializer_list<const Array*> results) {
    if (nranks_ == 1) return CN_OK;
    if (x.ndims == 1 && !x.replicated) return fail(CN_ERR_UNSUPPORTED, "this operator needs a leading dimension of rows on several ranks");
    for (const Array* p : operands)
        if (p && x.replicated && !p->replicated) return fail(CN_ERR_UNSUPPORTED, "this operator cannot mix arrays of one element with others on several ranks");
    for (const Array* p : results)
        if (p && x.replicated != p->replicated) return fail(CN_ERR_UNSUPPORTED, "this operator cannot mix arrays of one element with others on several ranks");
    return CN_OK;
}

// operands: x, weight, residual, eps, group (0: y in x's type).  results: y [, scale] [, h].
int Context::execute_rms_norm(const DagNode& node) {
    const AstNode& r = *node.roots[0];
    if (r.operands.size() != 5) return fail(CN_ERR_BAD_BLOB, "RMS_NORM needs (x, weight, residual, eps, group)");
    SeqArg x, w, res, eps, grp;
    SeqArg* const all[5] = {&x, &w, &res, &eps, &grp};
    int rc;
    for (size_t i = 0; i < 5; ++i)
        if ((rc = seq_arg(node, i, all[i]))) return rc;
    if (!x || eps || grp) return fail(CN_ERR_BAD_BLOB, "RMS_NORM needs an array x and literal eps and group");
    const int dtype = x.a->dtype, nd = x.a->ndims;
    if (!activation_type(dtype)) return fail(CN_ERR_BAD_DTYPE, "RMS_NORM takes float16, float32 and float64");
    const int64_t n = x.a->shape[nd - 1];
    if (n < 1) return fail(CN_ERR_INVALID_ARGUMENT, "RMS_NORM of rows without columns");
    if (w && (w.a->dtype != dtype || !has_shape(w.a, {n}))) return fail(CN_ERR_SHAPE_MISMATCH, "RMS_NORM weight must have x's type and one value per column");
    if (res) {
        if (res.a->dtype != dtype) return fail(CN_ERR_BAD_DTYPE, "RMS_NORM residual and x have different dtypes");
        if ((rc = check_leaf(res.a, nd, x.a->shape, "RMS_NORM residual"))) return rc;
    }
    if (!(eps.value >= 0)) return fail(CN_ERR_INVALID_ARGUMENT, "RMS_NORM eps must not be negative");
    if (!(grp.value >= 0) || grp.value > (double)n || grp.value != (double)(int64_t)grp.value)
        return fail(CN_ERR_INVALID_ARGUMENT, "RMS_NORM group must be a number of columns");
    const int64_t group = (int64_t)grp.value;
    const size_t results = 1 + (group > 0) + (res ? 1 : 0);
    if (node.roots.size() != results) return fail(CN_ERR_BAD_BLOB, "RMS_NORM: wrong number of results");
    if ((rc = seq_names(node, nullptr))) return rc;
    Array *y = nullptr, *scale = nullptr, *h = nullptr;
    if ((rc = seq_result(node, 0, nd, x.a->shape, group > 0 ? DT_I8 : dtype, &y))) return rc;
    if (group > 0) {
        // the last dimension becomes the groups; a 1-D row has a 1-D array of scales
        int64_t ss[kMaxDims];
        for (int d = 0; d < nd; ++d) ss[d] = x.a->shape[d];
        ss[nd - 1] = (n + group - 1) / group;
        if ((rc = seq_result(node, 1, nd, ss, acc_type(dtype), &scale))) return rc;
    }
    if (res && (rc = seq_result(node, results - 1, nd, x.a->shape, dtype, &h))) return rc;
    if ((rc = seq_rows(*x.a, {res.a}, {y, scale, h}))) return rc;
    if ((rc = seq_whole({&w}))) return rc;
    RmsNormArgs a;
    a.x = x.data();
    a.residual = res.data();
    a.weight = w.whole;
    a.y = y->buf.data;
    a.scale = scale ? scale->buf.data : nullptr;
    a.h = h ? h->buf.data : nullptr;
    a.n = n;
    a.rows = x.a->local_elems() / n;
    a.group = group;
    a.eps = eps.value;
    a.dtype = dtype;
    if (a.rows == 0) return CN_OK;
    const double size = (double)a.rows * n, e = dtype_size(dtype);
    prof_start(std::string("rms_norm #") + kSequenceSourceDigest, size * e * (res ? 3 : 1) + size * (group ? 1 : e));
    rc = cuda_fail(launch_rms_norm(a, sm_count_, stream_), "rms_norm");
    prof_stop();
    if (rc) return rc;
    stats_.kernel_launches++;
    return CN_OK;
}

// operands: x, weight, bias, state, lengths, activation (0 none, 1 silu).  results: y, state.
// The second result may be the state operand itself: the state is then brought up to date in place.
int Context::execute_causal_conv(const DagNode& node) {
    const AstNode& r = *node.roots[0];
    if (r.operands.size() != 6 || node.roots.size() != 2) return fail(CN_ERR_BAD_BLOB, "CAUSAL_CONV needs (x, weight, bias, state, lengths, activation) and two results");
    SeqArg x, w, bias, state, len, act;
    SeqArg* const all[6] = {&x, &w, &bias, &state, &len, &act};
    int rc;
    for (size_t i = 0; i < 6; ++i)
        if ((rc = seq_arg(node, i, all[i]))) return rc;
    if (!x || !w || act) return fail(CN_ERR_BAD_BLOB, "CAUSAL_CONV needs arrays x and weight and a literal activation");
    const int dtype = x.a->dtype;
    if (!activation_type(dtype)) return fail(CN_ERR_BAD_DTYPE, "CAUSAL_CONV takes float16, float32 and float64");
    if (x.a->ndims != 3) return fail(CN_ERR_SHAPE_MISMATCH, "CAUSAL_CONV x must be (sequences, time, channels)");
    const int64_t b = x.a->shape[0], t = x.a->shape[1], d = x.a->shape[2];
    if (w.a->ndims != 2 || w.a->shape[0] != d) return fail(CN_ERR_SHAPE_MISMATCH, "CAUSAL_CONV weight must be (channels, width)");
    const int64_t k = w.a->shape[1];
    if (k < 2 || k > kMaxConvWidth) return fail(CN_ERR_UNSUPPORTED, "CAUSAL_CONV width must be 2 to 8");
    if (w.a->dtype != dtype || (bias && bias.a->dtype != dtype) || (state && state.a->dtype != dtype) || (len && len.a->dtype != DT_I32))
        return fail(CN_ERR_BAD_DTYPE, "CAUSAL_CONV: weight, bias and state have x's type, lengths are int32");
    if (bias && !has_shape(bias.a, {d})) return fail(CN_ERR_SHAPE_MISMATCH, "CAUSAL_CONV bias must be (channels)");
    if (state && !has_shape(state.a, {b, k - 1, d})) return fail(CN_ERR_SHAPE_MISMATCH, "CAUSAL_CONV state must be (sequences, width - 1, channels)");
    if (len && !has_shape(len.a, {b})) return fail(CN_ERR_SHAPE_MISMATCH, "CAUSAL_CONV lengths must be (sequences)");
    if (act.value != 0 && act.value != 1) return fail(CN_ERR_INVALID_ARGUMENT, "CAUSAL_CONV activation must be 0 or 1");
    const bool in_place = state && node.roots[1]->result_name == state.a->name;
    if ((rc = seq_names(node, in_place ? state.a : nullptr))) return rc;
    Array *y = nullptr, *ns = nullptr;
    if ((rc = seq_result(node, 0, 3, x.a->shape, dtype, &y))) return rc;
    const int64_t sshape[3] = {b, k - 1, d};
    if (!in_place && (rc = seq_result(node, 1, 3, sshape, dtype, &ns))) return rc;
    // a prompt's blocks read the old state while others write the new one: it goes into the
    // array's shadow buffer, which then takes its place (as stencil sweeps do)
    const bool swap = in_place && t != 1;
    if (swap && (rc = ensure_shadow(state.a))) return rc;
    if ((rc = seq_rows(*x.a, {state.a, len.a}, {y, in_place ? state.a : ns}))) return rc;
    if ((rc = seq_whole({&w, &bias}))) return rc;
    CausalConvArgs a;
    a.x = x.data();
    a.weight = w.whole;
    a.bias = bias.whole;
    a.state = state.data();
    a.lengths = (const int*)len.data();
    a.y = y->buf.data;
    a.new_state = swap ? state.a->shadow.data : in_place ? state.a->buf.data : ns->buf.data;
    a.b = x.a->local_rows();
    a.t = t;
    a.d = d;
    a.k = (int)k;
    a.silu = act.value == 1;
    a.dtype = dtype;
    if (a.b > 0 && d > 0) {
        prof_start(std::string("causal_conv #") + kSequenceSourceDigest, 2.0 * a.b * (t + k - 1) * d * dtype_size(dtype));
        rc = cuda_fail(launch_causal_conv(a, sm_count_, stream_), "causal_conv");
        prof_stop();
        if (rc) return rc;
        stats_.kernel_launches++;
    }
    if (swap) std::swap(state.a->buf, state.a->shadow);
    if (in_place) state.a->mark_written();
    return CN_OK;
}

// operands: x, delta, A, B, C, D, z, delta_bias, state, lengths, softplus.  results: y, state.
// The second result may be the state operand itself.
int Context::execute_selective_scan(const DagNode& node) {
    const AstNode& r = *node.roots[0];
    if (r.operands.size() != 11 || node.roots.size() != 2)
        return fail(CN_ERR_BAD_BLOB, "SELECTIVE_SCAN needs (x, delta, A, B, C, D, z, delta_bias, state, lengths, softplus) and two results");
    SeqArg x, delta, A, B, C, D, z, db, state, len, sp;
    SeqArg* const all[11] = {&x, &delta, &A, &B, &C, &D, &z, &db, &state, &len, &sp};
    int rc;
    for (size_t i = 0; i < 11; ++i)
        if ((rc = seq_arg(node, i, all[i]))) return rc;
    if (!x || !delta || !A || !B || !C || sp) return fail(CN_ERR_BAD_BLOB, "SELECTIVE_SCAN needs arrays x, delta, A, B, C and a literal softplus");
    const int dtype = x.a->dtype, acc = acc_type(dtype);
    if (!activation_type(dtype)) return fail(CN_ERR_BAD_DTYPE, "SELECTIVE_SCAN takes float16, float32 and float64");
    if (x.a->ndims != 3) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN x must be (sequences, time, channels)");
    const int64_t b = x.a->shape[0], t = x.a->shape[1], d = x.a->shape[2];
    if (A.a->ndims != 2 || A.a->shape[0] != d) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN A must be (channels, states)");
    const int64_t n = A.a->shape[1];
    if (n < 1 || n > kMaxScanStates) return fail(CN_ERR_UNSUPPORTED, "SELECTIVE_SCAN takes 1 to 256 states per channel");
    if (delta.a->dtype != dtype || B.a->dtype != dtype || C.a->dtype != dtype || (z && z.a->dtype != dtype))
        return fail(CN_ERR_BAD_DTYPE, "SELECTIVE_SCAN: delta, B, C and z have x's type");
    if (A.a->dtype != acc || (D && D.a->dtype != acc) || (db && db.a->dtype != acc) || (state && state.a->dtype != acc))
        return fail(CN_ERR_BAD_DTYPE, "SELECTIVE_SCAN: A, D, delta_bias and state are float32 (float64 where x is)");
    if (len && len.a->dtype != DT_I32) return fail(CN_ERR_BAD_DTYPE, "SELECTIVE_SCAN lengths are int32");
    if ((rc = check_leaf(delta.a, 3, x.a->shape, "SELECTIVE_SCAN delta"))) return rc;
    if (z && (rc = check_leaf(z.a, 3, x.a->shape, "SELECTIVE_SCAN z"))) return rc;
    if (B.a->ndims != 3 || B.a->shape[0] != b || B.a->shape[1] != t || B.a->shape[2] % n || B.a->shape[2] < n)
        return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN B must be (sequences, time, groups x states)");
    if ((rc = check_leaf(C.a, 3, B.a->shape, "SELECTIVE_SCAN C"))) return rc;
    const int64_t groups = B.a->shape[2] / n;
    if (d % groups) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN channels do not divide into the groups of B and C");
    if (D && !has_shape(D.a, {d})) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN D must be (channels)");
    if (db && !has_shape(db.a, {d})) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN delta_bias must be (channels)");
    if (state && !has_shape(state.a, {b, d, n})) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN state must be (sequences, channels, states)");
    if (len && !has_shape(len.a, {b})) return fail(CN_ERR_SHAPE_MISMATCH, "SELECTIVE_SCAN lengths must be (sequences)");
    if (sp.value != 0 && sp.value != 1) return fail(CN_ERR_INVALID_ARGUMENT, "SELECTIVE_SCAN softplus must be 0 or 1");
    const bool in_place = state && node.roots[1]->result_name == state.a->name;
    if ((rc = seq_names(node, in_place ? state.a : nullptr))) return rc;
    Array *y = nullptr, *ns = nullptr;
    if ((rc = seq_result(node, 0, 3, x.a->shape, dtype, &y))) return rc;
    const int64_t sshape[3] = {b, d, n};
    if (!in_place && (rc = seq_result(node, 1, 3, sshape, acc, &ns))) return rc;
    const bool swap = in_place && t != 1;
    if (swap && (rc = ensure_shadow(state.a))) return rc;
    if ((rc = seq_rows(*x.a, {delta.a, B.a, C.a, z.a, state.a, len.a}, {y, in_place ? state.a : ns}))) return rc;
    if ((rc = seq_whole({&A, &D, &db}))) return rc;
    SelectiveScanArgs a;
    a.x = x.data();
    a.delta = delta.data();
    a.A = A.whole;
    a.B = B.data();
    a.C = C.data();
    a.D = D.whole;
    a.z = z.data();
    a.delta_bias = db.whole;
    a.state = state.data();
    a.lengths = (const int*)len.data();
    a.y = y->buf.data;
    a.new_state = swap ? state.a->shadow.data : in_place ? state.a->buf.data : ns->buf.data;
    a.b = x.a->local_rows();
    a.t = t;
    a.d = d;
    a.n = (int)n;
    a.groups = (int)groups;
    a.softplus = sp.value == 1;
    a.dtype = dtype;
    if (a.b > 0 && d > 0) {
        void* ws = nullptr;
        const size_t need = selective_scan_workspace(a, sm_count_);
        if (need && (rc = cuda_fail(cudaMallocAsync(&ws, need, stream_), "selective_scan workspace"))) return rc;
        a.workspace = ws;
        prof_start(std::string("selective_scan #") + kSequenceSourceDigest,
                   (double)a.b * t * d * dtype_size(dtype) * (z ? 4 : 3) + 2.0 * a.b * d * n * dtype_size(acc));
        rc = cuda_fail(launch_selective_scan(a, sm_count_, stream_), "selective_scan");
        prof_stop();
        if (ws) cudaFreeAsync(ws, stream_);
        if (rc) return rc;
        stats_.kernel_launches += ws ? 2 : 1;    // pieces of the time axis are walked twice
    }
    if (swap) std::swap(state.a->buf, state.a->shadow);
    if (in_place) state.a->mark_written();
    return CN_OK;
}

// operands: logits, u, temperature, top_k, top_p, min_p.  results: token, log probability.
int Context::execute_sample(const DagNode& node) {
    const AstNode& r = *node.roots[0];
    if (r.operands.size() != 6 || node.roots.size() != 2) return fail(CN_ERR_BAD_BLOB, "SAMPLE needs (logits, u, temperature, top_k, top_p, min_p) and two results");
    SeqArg x, u, par[4];
    int rc;
    if ((rc = seq_arg(node, 0, &x)) || (rc = seq_arg(node, 1, &u))) return rc;
    for (size_t i = 0; i < 4; ++i)
        if ((rc = seq_arg(node, 2 + i, &par[i]))) return rc;
    if (!x || !u) return fail(CN_ERR_BAD_BLOB, "SAMPLE needs arrays of logits and of random numbers");
    const int dtype = x.a->dtype, nd = x.a->ndims;
    if (!activation_type(dtype)) return fail(CN_ERR_BAD_DTYPE, "SAMPLE takes float16, float32 and float64 logits");
    if (nd > 2) return fail(CN_ERR_SHAPE_MISMATCH, "SAMPLE logits must be (rows, vocabulary) or (vocabulary)");
    const int64_t v = x.a->shape[nd - 1], rows = nd == 2 ? x.a->shape[0] : 1;
    if (v < 1 || v > kMaxVocabulary) return fail(CN_ERR_LIMIT, "SAMPLE takes vocabularies of 1 to 2^24");
    if (u.a->dtype != DT_F32 && u.a->dtype != DT_F64) return fail(CN_ERR_BAD_DTYPE, "SAMPLE random numbers are float32 or float64");
    if (!has_shape(u.a, {rows})) return fail(CN_ERR_SHAPE_MISMATCH, "SAMPLE needs one random number per row");
    SampleArgs a;
    RowParam* const to[4] = {&a.temperature, &a.top_k, &a.top_p, &a.min_p};
    for (int i = 0; i < 4; ++i) {
        to[i]->value = par[i].value;
        if (!par[i]) continue;
        const int want = par[i].a->dtype;
        if (i == 1 ? want != DT_I32 : (want != DT_F32 && want != DT_F64))
            return fail(CN_ERR_BAD_DTYPE, "SAMPLE: top_k per row is int32, temperature, top_p and min_p are float32 or float64");
        if (!has_shape(par[i].a, {rows})) return fail(CN_ERR_SHAPE_MISMATCH, "SAMPLE needs one parameter per row");
        to[i]->data = par[i].data();
        to[i]->dtype = want;
    }
    if ((rc = seq_names(node, nullptr))) return rc;
    Array *tok = nullptr, *logp = nullptr;
    const int64_t shape[1] = {rows};
    if ((rc = seq_result(node, 0, 1, shape, DT_I32, &tok))) return rc;
    if ((rc = seq_result(node, 1, 1, shape, acc_type(dtype), &logp))) return rc;
    // the results of a single row live on every rank: each of them gathers the row and draws from it
    if (rows == 1 && (rc = seq_whole({&x}))) return rc;
    a.logits = rows == 1 ? x.whole : x.data();
    a.u = u.data();
    a.u_dtype = u.a->dtype;
    a.token = (int*)tok->buf.data;
    a.logp = logp->buf.data;
    a.rows = rows == 1 ? 1 : x.a->local_rows();
    a.v = v;
    a.dtype = dtype;
    if (a.rows == 0) return CN_OK;
    prof_start(std::string("sample #") + kSequenceSourceDigest, (double)a.rows * v * dtype_size(dtype));
    rc = cuda_fail(launch_sample(a, sm_count_, stream_), "sample");
    prof_stop();
    if (rc) return rc;
    stats_.kernel_launches++;
    return CN_OK;
}

// operands: array, scale, group.  Without a scale: the array in the result root's type.  With one:
// int8 codes times the scale of their row and group of columns, in the result root's type.
int Context::execute_convert(const DagNode& node) {
    const AstNode& r = *node.roots[0];
    if (r.operands.size() != 3 || node.roots.size() != 1) return fail(CN_ERR_BAD_BLOB, "CONVERT needs (array, scale, group) and one result");
    SeqArg x, scale, grp;
    int rc;
    if ((rc = seq_arg(node, 0, &x)) || (rc = seq_arg(node, 1, &scale)) || (rc = seq_arg(node, 2, &grp))) return rc;
    if (!x || grp) return fail(CN_ERR_BAD_BLOB, "CONVERT needs an array and a literal group");
    const int nd = x.a->ndims;
    const int64_t n = x.a->shape[nd - 1];
    if (!dtype_storable(r.dtype)) return fail(CN_ERR_BAD_DTYPE, "CONVERT to a bad dtype code");
    ConvertArgs a;
    a.from = x.a->dtype;
    a.to = r.dtype;
    a.n = n;
    if (scale) {
        if (a.from != DT_I8 || !activation_type(a.to)) return fail(CN_ERR_BAD_DTYPE, "CONVERT with scales makes floating point values of int8 codes");
        if (scale.a->dtype != DT_F32 && scale.a->dtype != DT_F64) return fail(CN_ERR_BAD_DTYPE, "CONVERT scales are float32 or float64");
        if (!(grp.value >= 1) || grp.value > (double)std::max<int64_t>(n, 1) || grp.value != (double)(int64_t)grp.value)
            return fail(CN_ERR_INVALID_ARGUMENT, "CONVERT group must be a number of columns");
        a.group = (int64_t)grp.value;
        bool ok = scale.a->ndims == nd && scale.a->shape[nd - 1] == (n + a.group - 1) / a.group;
        for (int d = 0; ok && d < nd - 1; ++d) ok = scale.a->shape[d] == x.a->shape[d];
        if (!ok) return fail(CN_ERR_SHAPE_MISMATCH, "CONVERT needs one scale per row and group of columns");
        a.scale_dtype = scale.a->dtype;
    }
    if ((rc = seq_names(node, nullptr))) return rc;
    Array* out = nullptr;
    if ((rc = seq_result(node, 0, nd, x.a->shape, a.to, &out))) return rc;
    if (scale && (rc = seq_rows(*x.a, {scale.a}, {out}))) return rc;
    a.in = x.data();
    a.out = out->buf.data;
    a.scale = scale.data();
    // rows matter to scales alone; without them a rank converts whatever it has (of a vector, a part of the only row)
    const int64_t size = x.a->local_elems();
    if (size == 0) return CN_OK;
    if (!scale) a.n = size;
    a.rows = size / a.n;
    prof_start(std::string("convert #") + kSequenceSourceDigest, (double)size * (dtype_size(a.from) + dtype_size(a.to)));
    rc = cuda_fail(launch_convert(a, sm_count_, stream_), "convert");
    prof_stop();
    if (rc) return rc;
    stats_.kernel_launches++;
    return CN_OK;
}

}  // namespace cn
