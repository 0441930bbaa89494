// The host side of a chunk's decode and encode calls, on torch's tensors: what stands between a Python call and the launches.
//
// A 37-token chunk keeps the GPU busy for 14 us; reading its tensors' shapes and addresses, making the result and filling in
// the job descriptors took 33 us of Python.  Here it takes 10 with the launches.  The decode looks at its chunks and does the
// usual case (plain contiguous tensors on the current GPU, everything of the right shape and type); whatever is different
// in any way, malformed chunks included, it leaves to the caller, whose general path decodes it or says what is wrong.
// An encode's buffers are made, its job is filled in and its kernels are launched in one call, and in another its sizes are waited
// for, its payload is made and gathered, with nothing in between that the GPU would have to wait for.
//
// The library's entries come as addresses from the binding (bind), so that one copy of the library is in use.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/cachegen_b200.h"

namespace {

decltype(&cg_decode_kv) decode_kv;
decltype(&cg_encode_kv) encode_kv;
decltype(&cg_encode_kv_workspace) encode_kv_workspace;
decltype(&cg_encode_kv_wait) encode_kv_wait;
decltype(&cg_encode_kv_gather) encode_kv_gather;
decltype(&cg_rotary) rotary_rows;
decltype(&cg_append_paged) append_rows;
decltype(&cg_gather_paged) gather_rows;
decltype(&cg_paged_attention_workspace) attention_workspace;
decltype(&cg_paged_attention) attention;
decltype(&cg_pages_workspace) pages_workspace;
decltype(&cg_copy_pages) copy_rows;
decltype(&cg_fork_pages) fork_rows;
decltype(&cg_free_pages) free_rows;
decltype(&cg_extend_pages) extend_rows;
decltype(&cg_compact_pages) compact_rows;
decltype(&cg_beam_workspace) beam_workspace;
decltype(&cg_beam_select) best_beams;

// attribute names
PyObject *s_cdf, *s_max_tensors_key, *s_max_tensors_value, *s_data_chunks, *s_num_heads, *s_head_size, *s_bytestream,
    *s_bytestream_lengths, *s_ntokens, *s_blob, *s_header, *s_sub_off, *s_group_off, *s_captured;
const char *const kHeaderNames[] = {"L", "H", "D", "T", "lp", "nsub", "scale_code", "table_kind", "length_kind", "bins_checksum",
                                    "off_scales", "off_tables", "off_lengths", "off_payload"};
enum HeaderField {
    kL, kH, kD, kT, kLp, kNsub, kScaleCode, kTableKind, kLengthKind, kChecksum, kOffScales, kOffTables, kOffLengths, kOffPayload, kHeaderFields
};
PyObject *s_header_fields[kHeaderFields];

// A new reference that is given back.
struct Ref {
    PyObject *p;
    explicit Ref(PyObject *o) : p(o) {}
    ~Ref() { Py_XDECREF(p); }
    Ref(const Ref &) = delete;
    Ref &operator=(const Ref &) = delete;
};

// Released while the library works, as ctypes does, and while torch's allocator may wait, as torch does.
struct WithoutGil {
    PyThreadState *s = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(s); }
};

at::Tensor make(at::IntArrayRef shape, at::TensorOptions options) {
    const WithoutGil released;
    return at::empty(shape, options);
}

bool plain(PyObject *o) { return o && THPVariable_CheckExact(o); }

// A plain contiguous tensor of this type on this GPU: the only kind that is taken as it is.
bool usable(const at::Tensor &t, at::ScalarType type, at::Device dev) {
    return t.defined() && t.unsafeGetTensorImpl()->has_storage() && t.layout() == at::kStrided && t.scalar_type() == type &&
           t.device() == dev && t.is_contiguous() && !t.is_conj() && !t.is_neg();
}

bool small_int(PyObject *o, int64_t *v) {
    if (!o || !PyLong_CheckExact(o)) return false;
    *v = PyLong_AsLongLong(o);
    if (*v == -1 && PyErr_Occurred()) {
        PyErr_Clear();
        return false;
    }
    return true;
}

bool attribute_int(PyObject *o, PyObject *name, int64_t *v) {
    const Ref a(PyObject_GetAttr(o, name));
    if (!a.p) PyErr_Clear();
    return small_int(a.p, v);
}

// The tensor under a name, alive as long as the object that has it: nobody else can run between here and the launch but
// while the library works, and then `held` keeps it.
bool attribute_tensor(PyObject *o, PyObject *name, std::vector<at::Tensor> *held) {
    const Ref a(PyObject_GetAttr(o, name));
    if (!a.p) PyErr_Clear();
    if (!plain(a.p)) return false;
    held->push_back(THPVariable_Unpack(a.p));
    return true;
}

struct Shape {
    int64_t L = 0, H = 0, D = 0, lp = 0, T = 0;
    at::ScalarType scale = at::kHalf;
};

bool is_16bit(at::ScalarType t) { return t == at::kHalf || t == at::kBFloat16; }
int code(at::ScalarType t) { return t == at::kBFloat16 ? CG_BF16 : CG_F16; }

// Whether this chunk is of the shape of those before it; adds its tokens to theirs.
bool merge(const Shape &s, Shape *all, bool first) {
    if (!first && (s.L != all->L || s.H != all->H || s.D != all->D || s.lp != all->lp || s.scale != all->scale)) return false;
    const int64_t before = first ? 0 : all->T;
    *all = s;
    all->T = before + s.T;
    return true;
}

// One chunk's jobs, without what depends on the output.  false: not the usual case.
bool add_chunk(PyObject *eo, PyTypeObject *piece_type, at::Device dev, Shape *all, bool first, std::vector<cg_decode_job> *jobs,
               std::vector<at::Tensor> *held) {
    Shape s;
    if (!attribute_int(eo, s_num_heads, &s.H) || !attribute_int(eo, s_head_size, &s.D)) return false;
    if (s.H <= 0 || s.D <= 0 || s.H > 0xFFFFFF || s.D > 0xFFFFFF) return false;
    const size_t at = held->size();
    if (!attribute_tensor(eo, s_cdf, held) || !attribute_tensor(eo, s_max_tensors_key, held) || !attribute_tensor(eo, s_max_tensors_value, held))
        return false;
    // (by value: the vector grows)
    const at::Tensor cdf = (*held)[at], mk = (*held)[at + 1], mv = (*held)[at + 2];
    if (!usable(cdf, at::kShort, dev) || cdf.dim() != 3 || cdf.size(0) % 2 || cdf.size(1) != s.H * s.D) return false;
    s.L = cdf.size(0) / 2;
    s.lp = cdf.size(2);
    s.scale = mk.scalar_type();
    if (!is_16bit(s.scale) || !usable(mk, s.scale, dev) || !usable(mv, s.scale, dev) || mk.dim() < 2 || mv.dim() < 2) return false;
    s.T = mk.size(1);
    if (s.L <= 0 || s.T <= 0 || s.T > 0x7FFFFFFF || mk.size(0) != s.L || mv.size(0) != s.L || mv.size(1) != s.T || mk.numel() != s.L * s.T ||
        mv.numel() != s.L * s.T)
        return false;
    if (!merge(s, all, first)) return false;
    const Ref pieces(PyObject_GetAttr(eo, s_data_chunks));
    if (!pieces.p) PyErr_Clear();
    if (!pieces.p || !PyList_CheckExact(pieces.p)) return false;
    const int64_t streams = 2 * s.L * s.H * s.D;
    int64_t tokens = 0;
    for (Py_ssize_t k = 0; k < PyList_GET_SIZE(pieces.p); ++k) {
        PyObject *piece = PyList_GET_ITEM(pieces.p, k);
        int64_t n;
        if (Py_TYPE(piece) != piece_type || !attribute_int(piece, s_ntokens, &n) || n <= 0 || n > CG_MAX_TOKENS_PER_STREAM) return false;
        if (!attribute_tensor(piece, s_bytestream, held) || !attribute_tensor(piece, s_bytestream_lengths, held)) return false;
        const at::Tensor &bytes = (*held)[held->size() - 2], &lengths = held->back();
        if (!usable(bytes, at::kByte, dev) || bytes.dim() != 1 || !usable(lengths, at::kInt, dev) || lengths.numel() != streams) return false;
        cg_decode_job j{};
        j.tables = cdf.data_ptr();
        j.bytes = static_cast<const uint8_t *>(bytes.data_ptr());
        j.lengths = lengths.data_ptr();
        j.scales_k = static_cast<const uint16_t *>(mk.data_ptr()) + tokens;
        j.scales_v = static_cast<const uint16_t *>(mv.data_ptr()) + tokens;
        j.nbytes = bytes.numel();
        j.tables_nbytes = 2 * cdf.numel();
        j.ntokens = static_cast<int32_t>(n);
        j.scale_stride = static_cast<int32_t>(s.T);
        j.table_kind = CG_TABLES_CDF;
        j.length_kind = CG_LENGTHS_I32;
        jobs->push_back(j);
        tokens += n;
    }
    return tokens == s.T;
}

// Containers' kind of tables, what the bins of the decode say about them (see _HostBins), and the row offsets of their byte counts
// or masks.
struct FlatBins {
    int64_t kind = 0, checksum = 0, counts_bytes = 0, sparse_bytes = 0;
    at::Tensor row_off;
};

// The same for a container (flat_format.FlatChunk).
bool add_container(PyObject *chunk, at::Device dev, const FlatBins &bins, Shape *all, bool first, std::vector<cg_decode_job> *jobs,
                   std::vector<at::Tensor> *held) {
    if (!attribute_tensor(chunk, s_blob, held)) return false;
    const at::Tensor blob = held->back();
    if (!usable(blob, at::kByte, dev) || blob.dim() != 1) return false;
    const Ref header(PyObject_GetAttr(chunk, s_header));
    if (!header.p) PyErr_Clear();
    if (!header.p) return false;
    int64_t f[kHeaderFields];
    for (int k = 0; k < kHeaderFields; ++k)
        if (!attribute_int(header.p, s_header_fields[k], f + k) || f[k] < 0 || f[k] >= int64_t{1} << 48) return false;
    if (f[kL] < 1 || f[kL] > 0x7FFF || f[kH] < 1 || f[kD] < 1 || f[kH] > 0xFFFFFF || f[kD] > 0xFFFFFF || f[kH] * f[kD] > 0xFFFFFF || f[kT] < 1 ||
        f[kT] > 0x7FFFFFFF || f[kNsub] != (f[kT] + CG_MAX_TOKENS_PER_STREAM - 1) / CG_MAX_TOKENS_PER_STREAM || f[kScaleCode] > 1 || f[kLengthKind] > 1)
        return false;
    Shape s;
    s.L = f[kL];
    s.H = f[kH];
    s.D = f[kD];
    s.lp = f[kLp];
    s.T = f[kT];
    s.scale = f[kScaleCode] ? at::kBFloat16 : at::kHalf;
    if (!merge(s, all, first)) return false;
    if (f[kChecksum] && f[kChecksum] != bins.checksum) return false;
    const int64_t table_bytes = f[kOffLengths] - f[kOffTables];
    if (f[kTableKind] != bins.kind) return false;
    const int64_t least = bins.kind == CG_TABLES_COUNTS   ? bins.counts_bytes
                          : bins.kind == CG_TABLES_SPARSE ? bins.sparse_bytes
                                                          : 4 * s.L * s.H * s.D * s.lp;
    if (bins.kind > CG_TABLES_SPARSE || table_bytes < least) return false;
    if (bins.kind != CG_TABLES_CDF) {
        if (!usable(bins.row_off, at::kLong, dev) || bins.row_off.numel() != 2 * s.L + 1) return false;
        held->push_back(bins.row_off);
    }
    const Ref sub_off(PyObject_GetAttr(header.p, s_sub_off));
    if (!sub_off.p) PyErr_Clear();
    if (!sub_off.p || !PyList_CheckExact(sub_off.p) || PyList_GET_SIZE(sub_off.p) != f[kNsub] + 1) return false;
    uint8_t *const at = static_cast<uint8_t *>(blob.data_ptr());
    const int64_t size = blob.numel(), wide = f[kLengthKind] == CG_LENGTHS_U16 ? 2 : 4, row = 2 * s.L * s.H * s.D * wide;
    const uintptr_t a = reinterpret_cast<uintptr_t>(at);
    if (size < f[kOffLengths] + f[kNsub] * row || size < f[kOffScales] + 4 * s.L * s.T || (a + f[kOffScales]) % 2 || (a + f[kOffLengths]) % wide ||
        (bins.kind == CG_TABLES_CDF && (a + f[kOffTables]) % 2))
        return false;
    for (int64_t k = 0; k < f[kNsub]; ++k) {
        int64_t from, to;
        if (!small_int(PyList_GET_ITEM(sub_off.p, k), &from) || !small_int(PyList_GET_ITEM(sub_off.p, k + 1), &to) || from < 0 || from > to ||
            to > int64_t{1} << 48)
            return false;
        from = std::min(f[kOffPayload] + from, size);
        to = std::min(f[kOffPayload] + to, size);
        const int64_t t0 = k * CG_MAX_TOKENS_PER_STREAM;
        cg_decode_job j{};
        j.tables = at + f[kOffTables];
        j.bytes = at + from;
        j.lengths = at + f[kOffLengths] + k * row;
        j.scales_k = at + f[kOffScales] + 2 * t0;
        j.scales_v = at + f[kOffScales] + 2 * s.L * s.T + 2 * t0;
        j.table_row_off = bins.row_off.defined() ? static_cast<const int64_t *>(bins.row_off.data_ptr()) : nullptr;
        j.nbytes = to - from;
        j.tables_nbytes = table_bytes;
        j.ntokens = static_cast<int32_t>(std::min<int64_t>(CG_MAX_TOKENS_PER_STREAM, s.T - t0));
        j.scale_stride = static_cast<int32_t>(s.T);
        j.table_kind = static_cast<int32_t>(bins.kind);
        j.length_kind = static_cast<int32_t>(f[kLengthKind]);
        jobs->push_back(j);
    }
    return true;
}

// Adds a tensor to the set that a workspace holds for graphs (see _keep_for_graph in cachegen_decoder.py).
bool keep_for_graph(PyObject *workspace, PyObject *tensor) {
    if (tensor == Py_None) return true;
    PyObject *held = PyDict_GetItem(workspace, s_captured);
    if (!held) {
        const Ref made(PySet_New(nullptr));
        if (!made.p || PyDict_SetItem(workspace, s_captured, made.p)) return false;
        held = made.p;
    }
    return PySet_Add(held, tensor) == 0;
}

// decode(chunks, chunk type, piece type or None, bins, vllm, bf16 out, out or None, workspace, status word, of containers
//        (kind of tables, checksum, counts_bytes, sparse_bytes, row offsets or None))
// -> the KV blob, or the library's error code, or None: not the usual case, nothing has been done.
PyObject *decode(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !PyList_CheckExact(a[0]) || !PyType_Check(a[1]) || !PyList_GET_SIZE(a[0])) Py_RETURN_NONE;
    const bool containers = a[2] == Py_None;
    FlatBins flat;
    if (containers) {
        if (!PyTuple_CheckExact(a[9]) || PyTuple_GET_SIZE(a[9]) != 5) Py_RETURN_NONE;
        int64_t *const to[4] = {&flat.kind, &flat.checksum, &flat.counts_bytes, &flat.sparse_bytes};
        for (int k = 0; k < 4; ++k)
            if (!small_int(PyTuple_GET_ITEM(a[9], k), to[k])) Py_RETURN_NONE;
        if (plain(PyTuple_GET_ITEM(a[9], 4))) flat.row_off = THPVariable_Unpack(PyTuple_GET_ITEM(a[9], 4));
    } else if (!PyType_Check(a[2])) {
        Py_RETURN_NONE;
    }
    if (!plain(a[3]) || !PyDict_CheckExact(a[7]) || !plain(a[8]) || !(a[6] == Py_None || plain(a[6]))) Py_RETURN_NONE;
    const at::Tensor bins = THPVariable_Unpack(a[3]), status = THPVariable_Unpack(a[8]);
    const at::Device dev = bins.device();
    if (dev.type() != at::kCUDA || dev.index() != c10::cuda::current_device()) Py_RETURN_NONE;
    const bool vllm = a[4] == Py_True;
    const at::ScalarType type = a[5] == Py_True ? at::kBFloat16 : at::kHalf;
    Shape s;
    std::vector<cg_decode_job> jobs;
    std::vector<at::Tensor> held;
    const Py_ssize_t chunks = PyList_GET_SIZE(a[0]);
    jobs.reserve(static_cast<size_t>(chunks));
    held.reserve(static_cast<size_t>(5 * chunks));
    for (Py_ssize_t k = 0; k < chunks; ++k) {
        PyObject *eo = PyList_GET_ITEM(a[0], k);
        if (Py_TYPE(eo) != reinterpret_cast<PyTypeObject *>(a[1])) Py_RETURN_NONE;
        if (!(containers ? add_container(eo, dev, flat, &s, k == 0, &jobs, &held)
                         : add_chunk(eo, reinterpret_cast<PyTypeObject *>(a[2]), dev, &s, k == 0, &jobs, &held)))
            Py_RETURN_NONE;
    }
    const int64_t C = s.H * s.D, groups = 2 * s.L * ((C + CG_GROUP_CHANNELS - 1) / CG_GROUP_CHANNELS);
    const int64_t njobs = static_cast<int64_t>(jobs.size());
    if (!usable(bins, at::kFloat, dev) || bins.numel() != 2 * s.L || !usable(status, at::kInt, dev) || status.numel() != 1 || !njobs)
        Py_RETURN_NONE;
    const int64_t shape[5] = {s.L, 2, vllm ? s.T : s.H, vllm ? s.H : s.T, s.D};
    at::Tensor out;
    if (a[6] == Py_None) {
        out = make(shape, at::TensorOptions().dtype(type).device(dev));
    } else {
        out = THPVariable_Unpack(a[6]);
        if (!out.unsafeGetTensorImpl()->has_storage() || out.layout() != at::kStrided || out.scalar_type() != type || out.device() != dev ||
            out.sizes() != at::IntArrayRef(shape) || out.stride(4) != 1 || out.is_conj() || out.is_neg())
            Py_RETURN_NONE;
    }
    // The group offsets' buffer is kept in the workspace between calls.  A graph writes to its buffer at every replay: it gets one of
    // its own memory, and what else it uses of the workspace's stays there when other calls replace it.
    at::Tensor goff;
    if (c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) {
        goff = make({njobs * groups}, at::TensorOptions().dtype(at::kLong).device(dev));
        for (PyObject *used : {a[3], a[8], containers ? PyTuple_GET_ITEM(a[9], 4) : Py_None})
            if (!keep_for_graph(a[7], used)) throw python_error();
    } else {
        PyObject *const kept = PyDict_GetItem(a[7], s_group_off);
        if (plain(kept)) goff = THPVariable_Unpack(kept);
        if (!usable(goff, at::kLong, dev) || goff.numel() < njobs * groups) {
            goff = make({njobs * groups}, at::TensorOptions().dtype(at::kLong).device(dev));
            const Ref made(THPVariable_Wrap(goff));
            if (PyDict_SetItem(a[7], s_group_off, made.p)) throw python_error();
        }
    }
    const int64_t o_token = out.stride(vllm ? 2 : 3), o_head = out.stride(vllm ? 3 : 2);
    uint8_t *at_out = static_cast<uint8_t *>(out.data_ptr());
    int64_t *at_goff = static_cast<int64_t *>(goff.data_ptr());
    for (cg_decode_job &j : jobs) {
        j.out = at_out;
        j.group_off = at_goff;
        at_out += 2 * o_token * j.ntokens;
        at_goff += groups;
    }
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(dev.index());
    int rc;
    {
        const WithoutGil released;
        rc = decode_kv(jobs.data(), static_cast<int>(njobs), static_cast<int>(s.L), static_cast<int>(s.H), static_cast<int>(s.D),
                       static_cast<int>(s.lp), static_cast<const float *>(bins.data_ptr()), 0,
                       nullptr, code(s.scale), code(type), out.stride(0), out.stride(1), o_token,
                       o_head, static_cast<int32_t *>(status.data_ptr()), stream.stream());
    }
    if (rc) return PyLong_FromLong(rc);
    {
        const WithoutGil released;
        for (const at::Tensor &t : held) c10::cuda::CUDACachingAllocator::recordStream(t.storage().data_ptr(), stream);
    }
    return THPVariable_Wrap(out);
    END_HANDLE_TH_ERRORS
}

int64_t integer(PyObject *o) {
    const int64_t v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw python_error();
    return v;
}

// encode_start(address of a cg_encode_kv_job with delta_group and res_bins set, kv, bins, max_bins, address of the tail,
//              workspace or None, row offsets of byte counts or None, their size, stream or None: the current one, launch)
// -> (error code, stream, scales [2, L, T, 1], scales_k, scales_v, cdf, workspace, counts or None).  kv: [L, 2, T, H, D] on a GPU, 16-bit,
// unit innermost stride.  With counts the two scales are parts of one tensor, else tensors of their own and the first is None.
PyObject *encode_start(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 10 || !THPVariable_Check(a[1]) || !THPVariable_Check(a[2])) {
        PyErr_SetString(PyExc_TypeError, "encode_start: wrong arguments");
        return nullptr;
    }
    cg_encode_kv_job &job = *reinterpret_cast<cg_encode_kv_job *>(integer(a[0]));
    const at::Tensor kv = THPVariable_Unpack(a[1]), bins = THPVariable_Unpack(a[2]);
    const int64_t max_bins = integer(a[3]), L = kv.size(0), T = kv.size(2), H = kv.size(3), D = kv.size(4);
    const bool with_counts = a[6] != Py_None;
    const c10::cuda::CUDAGuard device(kv.device());
    const at::TensorOptions on = at::TensorOptions().device(kv.device()), bytes = on.dtype(at::kByte);
    at::Tensor scales, scales_k, scales_v, counts, workspace;
    if (with_counts) {
        scales = make({2, L, T, 1}, on.dtype(kv.scalar_type()));
        scales_k = scales.select(0, 0);
        scales_v = scales.select(0, 1);
    } else {
        scales_k = make({L, T, 1}, on.dtype(kv.scalar_type()));
        scales_v = make({L, T, 1}, on.dtype(kv.scalar_type()));
    }
    const at::Tensor cdf = make({2 * L, H * D, max_bins + 1}, on.dtype(at::kShort));
    const int64_t need = encode_kv_workspace(static_cast<int>(L), static_cast<int>(T), static_cast<int>(H), static_cast<int>(D));
    if (need < 0) return Py_BuildValue("(LOOOOOOO)", static_cast<long long>(need), Py_None, Py_None, Py_None, Py_None, Py_None, Py_None, Py_None);
    if (a[5] != Py_None) workspace = THPVariable_Unpack(a[5]);
    if (!workspace.defined() || workspace.numel() < need) workspace = make({need}, bytes);
    job.kv = kv.data_ptr();
    job.bins = static_cast<const float *>(bins.data_ptr());
    job.scales_k = scales_k.data_ptr();
    job.scales_v = scales_v.data_ptr();
    job.cdf = static_cast<int16_t *>(cdf.data_ptr());
    if (with_counts) {
        counts = make({integer(a[7])}, bytes);
        job.counts = static_cast<uint8_t *>(counts.data_ptr());
        job.table_row_off = static_cast<const int64_t *>(THPVariable_Unpack(a[6]).data_ptr());
    }
    job.workspace = workspace.data_ptr();
    job.workspace_bytes = workspace.numel();
    job.tail = reinterpret_cast<int64_t *>(integer(a[4]));
    job.s_layer = kv.stride(0);
    job.s_kv = kv.stride(1);
    job.s_token = kv.stride(2);
    job.s_head = kv.stride(3);
    job.dtype = code(kv.scalar_type());
    job.nlayers = static_cast<int32_t>(L);
    job.ntokens = static_cast<int32_t>(T);
    job.nheads = static_cast<int32_t>(H);
    job.head_size = static_cast<int32_t>(D);
    job.max_bins = static_cast<int32_t>(max_bins);
    void *const stream = a[8] == Py_None ? c10::cuda::getCurrentCUDAStream(kv.device().index()).stream() : reinterpret_cast<void *>(integer(a[8]));
    int rc = CG_OK;
    if (a[9] == Py_True) {
        const WithoutGil released;
        rc = encode_kv(&job, stream);
    }
    const auto wrap = [](const at::Tensor &t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); };
    return Py_BuildValue("(iKNNNNNN)", rc, static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(stream)), wrap(scales),
                         wrap(scales_k), wrap(scales_v), wrap(cdf), wrap(workspace), wrap(counts));
    END_HANDLE_TH_ERRORS
}

// encode_finish(address of a job that has been launched, number of its GPU, stream, its tensors of lengths or None)
// -> (error code, tail, pieces or None): waits for the sizes; with lengths, and if no stream is bad, makes a tensor for
// every sub-chunk's streams (a view would pickle the whole buffer) and launches the gather.
// tail: the nsub + 1 payload offsets, the status bits and the number of non-zero byte counts.
PyObject *encode_finish(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    if (n != 4 || !(a[3] == Py_None || PyList_CheckExact(a[3]))) {
        PyErr_SetString(PyExc_TypeError, "encode_finish: wrong arguments");
        return nullptr;
    }
    cg_encode_kv_job &job = *reinterpret_cast<cg_encode_kv_job *>(integer(a[0]));
    const c10::cuda::CUDAGuard device(static_cast<c10::DeviceIndex>(integer(a[1])));
    void *stream = reinterpret_cast<void *>(integer(a[2]));
    const int nsub = (job.ntokens + CG_MAX_TOKENS_PER_STREAM - 1) / CG_MAX_TOKENS_PER_STREAM;
    int rc;
    {
        const WithoutGil released;
        rc = encode_kv_wait(&job, stream);
    }
    if (rc) return Py_BuildValue("(iOO)", rc, Py_None, Py_None);
    // the tail goes back to its pool before anything can fail
    const std::vector<int64_t> sizes(job.tail, job.tail + nsub + 3);
    PyObject *pieces = nullptr;
    if (a[3] != Py_None && !(sizes[nsub + 1] & ~CG_S_COUNT_OVERFLOW)) {
        if (PyList_GET_SIZE(a[3]) != nsub) {
            PyErr_SetString(PyExc_TypeError, "encode_finish: wrong arguments");
            return nullptr;
        }
        std::vector<uint8_t *> to(static_cast<size_t>(nsub));
        std::vector<int32_t *> lengths(static_cast<size_t>(nsub));
        std::vector<at::Tensor> made(static_cast<size_t>(nsub));
        for (int k = 0; k < nsub; ++k) {
            const at::Tensor t = THPVariable_Unpack(PyList_GET_ITEM(a[3], k));
            lengths[k] = static_cast<int32_t *>(t.data_ptr());
            made[k] = make({sizes[k + 1] - sizes[k]}, at::TensorOptions().dtype(at::kByte).device(t.device()));
            to[k] = static_cast<uint8_t *>(made[k].data_ptr());
        }
        {
            const WithoutGil released;
            rc = encode_kv_gather(&job, to.data(), lengths.data(), stream);
        }
        pieces = PyList_New(nsub);
        for (int k = 0; k < nsub; ++k) PyList_SET_ITEM(pieces, k, THPVariable_Wrap(made[k]));
    }
    PyObject *tail = PyList_New(nsub + 3);
    for (int k = 0; k < nsub + 3; ++k) PyList_SET_ITEM(tail, k, PyLong_FromLongLong(sizes[k]));
    return Py_BuildValue("(iNN)", rc, tail, pieces ? pieces : Py_NewRef(Py_None));
    END_HANDLE_TH_ERRORS
}

// ---- calls on a paged cache -------------------------------------------------------------------------
// Each looks whether its arguments are the usual case, everything of the right shape and type on the current GPU, and then does all of
// the call.  For any other arguments, wrong ones included, it does nothing: cachegen_b200.paged says what is wrong, or does it.
enum class Use { kRead, kWritten };

// Rows or pages: a plain strided tensor of this type whose innermost axis is contiguous.
bool rows_of(PyObject *o, at::ScalarType type, at::Device dev, int64_t dims, Use use, at::Tensor *t) {
    if (!plain(o)) return false;
    *t = THPVariable_Unpack(o);
    if (!t->defined() || !t->unsafeGetTensorImpl()->has_storage() || t->layout() != at::kStrided || t->scalar_type() != type || t->device() != dev ||
        t->dim() != dims || t->is_conj() || t->is_neg() || t->requires_grad() || (t->stride(dims - 1) != 1 && t->size(dims - 1) > 1))
        return false;
    for (int64_t k = 0; use == Use::kWritten && k < dims; ++k)
        if (t->stride(k) == 0 && t->size(k) > 1) return false;
    return true;
}
bool first_of(PyObject *o, at::Tensor *t, at::Device *dev) {
    if (!plain(o)) return false;
    *t = THPVariable_Unpack(o);
    if (!t->defined() || !is_16bit(t->scalar_type()) || !t->is_cuda()) return false;
    *dev = t->device();
    return dev->index() == c10::cuda::current_device();
}
bool indices_of(PyObject *o, at::Device dev, bool wide_too, at::Tensor *t) {
    if (!plain(o)) return false;
    *t = THPVariable_Unpack(o);
    return usable(*t, at::kInt, dev) || (wide_too && usable(*t, at::kLong, dev));
}
// Whether two tensors of 16-bit values share none, as cachegen_b200.paged's _are_apart: by ranges, or along the axes that they step along together.
struct Axis {
    int64_t step, size;
};
struct Axes {
    Axis axis[5];
    int n = 0;
    int64_t span(int from) const {
        int64_t values = 1;
        for (int k = from; k < n; ++k) values += (axis[k].size - 1) * axis[k].step;
        return values;
    }
};
bool no_value_shared(int64_t gap, const Axes &a, int ia, const Axes &b, int ib) {
    if (gap >= 2 * a.span(ia) || -gap >= 2 * b.span(ib)) return true;
    const int64_t step = std::max(ia < a.n ? a.axis[ia].step : 0, ib < b.n ? b.axis[ib].step : 0);
    if (step == 0) return false;
    const bool in_a = ia < a.n && a.axis[ia].step == step, in_b = ib < b.n && b.axis[ib].step == step;
    const int64_t na = in_a ? a.axis[ia].size : 1, nb = in_b ? b.axis[ib].size : 1;
    const int64_t reach_a = 2 * a.span(ia + in_a), reach_b = 2 * b.span(ib + in_b), bytes = 2 * step;
    const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
    const int64_t first = std::max(floor_div(gap - reach_a, bytes) + 1, 1 - nb), last = std::min(-floor_div(-gap - reach_b, bytes) - 1, na - 1);
    if (last - first >= 4) return false;
    for (int64_t k = first; k <= last; ++k)
        if (!no_value_shared(gap - k * bytes, a, ia + in_a, b, ib + in_b)) return false;
    return true;
}
Axes axes_of(const at::Tensor &t) {
    Axes x;
    for (int64_t k = 0; k < t.dim(); ++k)
        if (t.size(k) > 1) x.axis[x.n++] = Axis{t.stride(k), t.size(k)};
    std::sort(x.axis, x.axis + x.n, [](const Axis &p, const Axis &q) { return p.step > q.step; });
    return x;
}
bool apart(const at::Tensor &a, const at::Tensor &b) {
    if (!a.numel() || !b.numel()) return true;
    const auto reach = [](const at::Tensor &t) {
        const at::IntArrayRef sizes = t.sizes(), strides = t.strides();
        int64_t values = 1;
        for (size_t k = 0; k < sizes.size(); ++k) values += (sizes[k] - 1) * strides[k];
        return 2 * values;
    };
    const int64_t gap = static_cast<const char *>(b.const_data_ptr()) - static_cast<const char *>(a.const_data_ptr());
    return gap >= reach(a) || -gap >= reach(b) || no_value_shared(gap, axes_of(a), 0, axes_of(b), 0);
}
bool same_or_apart(const at::Tensor &a, const at::Tensor &b) { return (a.data_ptr() == b.data_ptr() && a.strides() == b.strides()) || apart(a, b); }
void strides_of(const at::Tensor &t, int64_t *to, int64_t outer) {  // of all axes but the innermost; a layer axis that is not there: 0
    const int64_t dims = t.dim() - 1;
    for (int64_t k = 0; k < outer; ++k) to[k] = k < outer - dims ? 0 : t.stride(k - (outer - dims));
}
at::Tensor like(const at::Tensor &t, at::IntArrayRef shape) { return make(shape, t.options()); }

// (turns or None, the stream that they were made on, rotary_dims, interleaved, head size, positions): with them or without them as the job needs it
bool turning(cg_rows_job *job, PyObject *const *a, at::Device dev, int64_t layers, int64_t tokens, int64_t head, at::Tensor *positions) {
    if (a[0] == Py_None) return a[5] == Py_None;
    int64_t made_on, rot, of;
    if (!plain(a[0]) || !small_int(a[1], &made_on) || !small_int(a[2], &rot) || !small_int(a[4], &of) || of != head ||
        !indices_of(a[5], dev, true, positions))
        return false;
    const at::Tensor &turns = THPVariable_Unpack(a[0]);
    if (!usable(turns, at::kLong, dev) || turns.numel() != rot / 2) return false;
    if (positions->dim() == 2 && layers >= 0) {
        if (positions->size(0) != layers || positions->size(1) != tokens) return false;
        job->pos_layer = layers > 1 ? tokens : 0;
    } else if (positions->dim() != 1 || positions->size(0) != tokens) {
        return false;
    }
    job->positions = positions->data_ptr();
    job->wide_positions = positions->scalar_type() == at::kLong;
    job->turns = static_cast<const uint64_t *>(turns.data_ptr());
    job->rotary_dims = static_cast<int32_t>(rot);
    job->interleaved = a[3] == Py_True;
    // a Rotary may be dropped while the kernel reads its turns on another stream than theirs (a graph's is kept by its user)
    const c10::cuda::CUDAStream stream = c10::cuda::getCurrentCUDAStream(dev.index());
    if (reinterpret_cast<int64_t>(stream.stream()) != made_on && c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None)
        c10::cuda::CUDACachingAllocator::recordStream(turns.storage().data_ptr(), stream);
    return true;
}
bool fits(std::initializer_list<int64_t> sizes) {
    for (const int64_t n : sizes)
        if (n > INT32_MAX) return false;
    return true;
}
// Tells torch that a tensor was written to: a backward pass that kept it for later must not use what is in it now.
void wrote(const at::Tensor &t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();  // (those have no versions)
}
template <class Job> int run(int (*entry)(const Job *, void *), const Job &job, at::Device dev) {
    void *stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const WithoutGil released;
    return entry(&job, stream);
}

// rotary(x, out or None, inverse, turns, their stream, rotary_dims, interleaved, head size, positions) -> out, an error code, or None
PyObject *rotary(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor x, out, positions;
    at::Device dev(at::kCPU);
    if (n != 9 || !first_of(a[0], &x, &dev) || x.dim() < 3 || x.dim() > 4 || a[3] == Py_None) Py_RETURN_NONE;
    if (!rows_of(a[0], x.scalar_type(), dev, x.dim(), Use::kRead, &x)) Py_RETURN_NONE;
    const int64_t d = x.dim(), layers = d == 4 ? x.size(0) : 1, T = x.size(d - 3), H = x.size(d - 2), D = x.size(d - 1);
    cg_rows_job job{};
    if (!fits({layers, T, H, D}) || !turning(&job, a + 3, dev, d == 4 ? layers : -1, T, D, &positions)) Py_RETURN_NONE;
    if (a[1] == Py_None) out = like(x, x.sizes());
    else if (!rows_of(a[1], x.scalar_type(), dev, d, Use::kWritten, &out) || out.sizes() != x.sizes() || !same_or_apart(x, out)) Py_RETURN_NONE;
    job.k = x.data_ptr();
    job.k_out = out.data_ptr();
    strides_of(x, job.k_strides, 3);
    strides_of(out, job.k_out_strides, 3);
    job.dtype = code(x.scalar_type());
    job.nlayers = static_cast<int32_t>(layers), job.ntokens = static_cast<int32_t>(T), job.heads = static_cast<int32_t>(H);
    job.head_size = static_cast<int32_t>(D), job.inverse = a[2] == Py_True;
    const int rc = run(rotary_rows, job, dev);
    if (!rc) wrote(out);
    return rc ? PyLong_FromLong(rc) : a[1] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[1]);
    END_HANDLE_TH_ERRORS
}

// What append and gather have in common: k, v, k_pages, v_pages, slots, status, turns, their stream, rotary_dims, interleaved, head size,
// positions
bool pages_job(PyObject *const *a, const at::Tensor &k, const at::Tensor &v, bool append, at::Device dev, cg_rows_job *job, at::Tensor *held) {
    const int64_t d = k.dim(), layers = d == 4 ? k.size(0) : 1, T = k.size(d - 3), H = k.size(d - 2), D = k.size(d - 1);
    at::Tensor &kp = held[0], &vp = held[1], &slots = held[2], &status = held[3];
    const Use pages = append ? Use::kWritten : Use::kRead;
    if (!rows_of(a[2], k.scalar_type(), dev, d + 1, pages, &kp) || !rows_of(a[3], k.scalar_type(), dev, d + 1, pages, &vp)) return false;
    const int64_t P = kp.size(d - 3), S = kp.size(d - 2);
    if (kp.sizes() != vp.sizes() || (d == 4 && kp.size(0) != layers) || kp.size(d - 1) != H || kp.size(d) != D || S == 0) return false;
    if (!indices_of(a[4], dev, true, &slots) || slots.dim() != 1 || slots.size(0) != T) return false;
    if (T && (append ? !apart(kp, vp) : !apart(k, v))) return false;
    if (a[5] != Py_None && (!indices_of(a[5], dev, false, &status) || status.numel() != 1)) return false;
    if (!fits({layers, T, H, D, S}) || !turning(job, a + 6, dev, -1, T, D, held + 4)) return false;
    if (!apart(k, kp) || !apart(k, vp) || !apart(v, kp) || !apart(v, vp)) return false;
    job->k = k.data_ptr(), job->v = v.data_ptr(), job->pages_k = kp.data_ptr(), job->pages_v = vp.data_ptr();
    strides_of(k, job->k_strides, 3);
    strides_of(v, job->v_strides, 3);
    strides_of(kp, job->pages_k_strides, 4);
    strides_of(vp, job->pages_v_strides, 4);
    job->slots = slots.data_ptr(), job->wide_slots = slots.scalar_type() == at::kLong;
    job->status = status.defined() ? static_cast<int32_t *>(status.data_ptr()) : nullptr;
    job->num_pages = P, job->page_size = static_cast<int32_t>(S);
    job->dtype = code(k.scalar_type());
    job->nlayers = static_cast<int32_t>(layers), job->ntokens = static_cast<int32_t>(T), job->heads = static_cast<int32_t>(H);
    job->head_size = static_cast<int32_t>(D);
    return true;
}

// append(k, v, k_pages, v_pages, slots, status, turns, their stream, rotary_dims, interleaved, head size, positions, q or None, q_out or None)
// -> q_out or True, an error code, or None
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor k, v, q, q_out, held[5];
    at::Device dev(at::kCPU);
    cg_rows_job job{};
    if (n != 14 || !first_of(a[0], &k, &dev) || k.dim() < 3 || k.dim() > 4 || !rows_of(a[0], k.scalar_type(), dev, k.dim(), Use::kRead, &k) ||
        !rows_of(a[1], k.scalar_type(), dev, k.dim(), Use::kRead, &v) || v.sizes() != k.sizes() || !pages_job(a, k, v, true, dev, &job, held))
        Py_RETURN_NONE;
    const bool queries = a[12] != Py_None;
    if (!queries && a[13] != Py_None) Py_RETURN_NONE;
    if (queries) {
        if (k.dim() != 3 || !rows_of(a[12], k.scalar_type(), dev, 3, Use::kRead, &q) || q.size(0) != k.size(0) || q.size(2) != k.size(2)) Py_RETURN_NONE;
        if (a[13] == Py_None) q_out = like(q, q.sizes());
        else if (!rows_of(a[13], k.scalar_type(), dev, 3, Use::kWritten, &q_out) || q_out.sizes() != q.sizes() || !same_or_apart(q, q_out) ||
                 !apart(q_out, k) || !apart(q_out, v) || !apart(q_out, held[0]) || !apart(q_out, held[1]))
            Py_RETURN_NONE;
        if (!apart(q, held[0]) || !apart(q, held[1])) Py_RETURN_NONE;
        job.q = q.data_ptr(), job.q_out = q_out.data_ptr();
        strides_of(q, job.q_strides, 3);
        strides_of(q_out, job.q_out_strides, 3);
        job.q_heads = static_cast<int32_t>(q.size(1));
    }
    const int rc = run(append_rows, job, dev);
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor *t : {&held[0], &held[1], &q_out}) wrote(*t);
    return !queries ? Py_NewRef(Py_True) : a[13] == Py_None ? THPVariable_Wrap(q_out) : Py_NewRef(a[13]);
    END_HANDLE_TH_ERRORS
}

// gather(k or None, v or None, k_pages, v_pages, slots, status, turns, their stream, rotary_dims, interleaved, head size, positions)
// -> (k, v), an error code, or None
PyObject *gather(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor k, v, pages, slots, held[5];
    at::Device dev(at::kCPU);
    if (n != 12 || !first_of(a[2], &pages, &dev) || pages.dim() < 4 || pages.dim() > 5 || !indices_of(a[4], dev, true, &slots) || slots.dim() != 1) Py_RETURN_NONE;
    std::vector<int64_t> shape(pages.sizes().begin(), pages.sizes().end());
    shape.erase(shape.end() - 4);
    shape[shape.size() - 3] = slots.size(0);
    for (at::Tensor *t : {&k, &v}) {
        PyObject *const given = t == &k ? a[0] : a[1];
        if (given == Py_None) *t = like(pages, shape);
        else if (!rows_of(given, pages.scalar_type(), dev, pages.dim() - 1, Use::kWritten, t) || t->sizes() != at::IntArrayRef(shape)) Py_RETURN_NONE;
    }
    cg_rows_job job{};
    if (!pages_job(a, k, v, false, dev, &job, held)) Py_RETURN_NONE;
    const int rc = run(gather_rows, job, dev);
    if (rc) return PyLong_FromLong(rc);
    wrote(k), wrote(v);
    return Py_BuildValue("(NN)", a[0] == Py_None ? THPVariable_Wrap(k) : Py_NewRef(a[0]), a[1] == Py_None ? THPVariable_Wrap(v) : Py_NewRef(a[1]));
    END_HANDLE_TH_ERRORS
}

// attend(q, k_pages, v_pages, table, kv_lens, q_starts or None, scale, causal, window, max_q, out or None, lse wanted, status)
// -> out or (out, lse), an error code, or None
PyObject *attend(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor q, kp, vp, table, lens, starts, out, lse, status, workspace;
    at::Device dev(at::kCPU);
    int64_t window, max_q;
    if (n != 13 || !first_of(a[0], &q, &dev) || !rows_of(a[0], q.scalar_type(), dev, 3, Use::kRead, &q) ||
        !rows_of(a[1], q.scalar_type(), dev, 4, Use::kRead, &kp) || !rows_of(a[2], q.scalar_type(), dev, 4, Use::kRead, &vp) ||
        !indices_of(a[3], dev, false, &table) || !indices_of(a[4], dev, false, &lens) || (a[12] != Py_None && !indices_of(a[12], dev, false, &status)) ||
        !PyFloat_CheckExact(a[6]) || !small_int(a[8], &window) || !small_int(a[9], &max_q))
        Py_RETURN_NONE;
    const int64_t R = q.size(0), Q = q.size(1), D = q.size(2), P = kp.size(0), S = kp.size(1), H = kp.size(2), B = lens.numel();
    if (kp.sizes() != vp.sizes() || kp.size(3) != D || D % 8 || D == 0 || D > 128 || S == 0 || H == 0 || Q == 0 || Q % H || lens.dim() != 1 ||
        B > CG_MAX_REQUESTS || table.dim() != 2 || table.size(0) != B || (status.defined() && status.numel() != 1) || window < 0 || max_q < 0 ||
        !fits({R, Q, H, S, table.size(1), window, max_q}))
        Py_RETURN_NONE;
    if (a[5] == Py_None ? R != B : !indices_of(a[5], dev, false, &starts) || starts.dim() != 1 || starts.numel() != B + 1) Py_RETURN_NONE;
    if (a[10] != Py_None && (!rows_of(a[10], q.scalar_type(), dev, 3, Use::kWritten, &out) || out.sizes() != q.sizes() || !apart(out, q) || !apart(out, kp) ||
                             !apart(out, vp)))
        Py_RETURN_NONE;
    if (a[10] == Py_None) out = like(q, q.sizes());
    for (const at::Tensor *t : {&q, &kp, &vp, &out}) {
        if (reinterpret_cast<uintptr_t>(t->data_ptr()) % 16) Py_RETURN_NONE;
        for (int64_t k = 0; k + 1 < t->dim(); ++k)
            if (t->stride(k) % 8 && t->size(k) > 1) Py_RETURN_NONE;
    }
    cg_attention_job job{};
    if (a[11] == Py_True) {
        lse = make({R, Q}, at::TensorOptions().dtype(at::kFloat).device(dev));
        job.lse = static_cast<float *>(lse.data_ptr());
    }
    job.q = q.data_ptr(), job.pages_k = kp.data_ptr(), job.pages_v = vp.data_ptr(), job.out = out.data_ptr();
    job.table = static_cast<const int32_t *>(table.data_ptr()), job.kv_lens = static_cast<const int32_t *>(lens.data_ptr());
    job.q_starts = starts.defined() ? static_cast<const int32_t *>(starts.data_ptr()) : nullptr;
    job.status = status.defined() ? static_cast<int32_t *>(status.data_ptr()) : nullptr;
    job.table_row = table.stride(0), job.num_pages = P;
    const auto steps = [](const at::Tensor &t, int64_t *to) {
        for (int64_t k = 0; k + 1 < t.dim(); ++k) to[k] = t.size(k) > 1 ? t.stride(k) : 0;
    };
    steps(q, job.q_strides);
    steps(out, job.out_strides);
    steps(kp, job.pages_k_strides);
    steps(vp, job.pages_v_strides);
    job.dtype = code(q.scalar_type());
    job.nrequests = static_cast<int32_t>(B), job.nrows = static_cast<int32_t>(R), job.q_heads = static_cast<int32_t>(Q);
    job.heads = static_cast<int32_t>(H), job.head_size = static_cast<int32_t>(D), job.page_size = static_cast<int32_t>(S);
    job.table_width = static_cast<int32_t>(table.size(1)), job.causal = a[7] == Py_True;
    job.window = static_cast<int32_t>(window), job.max_q = static_cast<int32_t>(max_q);
    job.scale = static_cast<float>(PyFloat_AS_DOUBLE(a[6]));
    const int64_t need = attention_workspace(&job);
    if (need < 0) return PyLong_FromLongLong(need);
    if (need) {
        workspace = make({need}, at::TensorOptions().dtype(at::kByte).device(dev));
        job.workspace = workspace.data_ptr(), job.workspace_bytes = need;
    }
    const int rc = run(attention, job, dev);
    if (rc) return PyLong_FromLong(rc);
    wrote(out);
    PyObject *const result = a[10] == Py_None ? THPVariable_Wrap(out) : Py_NewRef(a[10]);
    return a[11] == Py_True ? Py_BuildValue("(NN)", result, THPVariable_Wrap(lse)) : result;
    END_HANDLE_TH_ERRORS
}

// ---- pages that rows share, and beams ----------------------------------------------------------------
// Whether the memory from the first to the last value of two tensors is apart; where it is not, the general path looks closer.
bool ranges_apart(const at::Tensor &a, const at::Tensor &b) {
    if (!a.defined() || !b.defined() || !a.numel() || !b.numel()) return true;
    const auto reach = [](const at::Tensor &t) {
        int64_t values = 1;
        for (int64_t k = 0; k < t.dim(); ++k) values += (t.size(k) - 1) * t.stride(k);
        return values * static_cast<int64_t>(t.element_size());
    };
    const int64_t gap = static_cast<const char *>(b.const_data_ptr()) - static_cast<const char *>(a.const_data_ptr());
    return gap >= reach(a) || -gap >= reach(b);
}
bool all_apart(std::initializer_list<const at::Tensor *> written, std::initializer_list<const at::Tensor *> read) {
    for (auto a = written.begin(); a != written.end(); ++a) {
        for (auto b = a + 1; b != written.end(); ++b)
            if (!ranges_apart(**a, **b)) return false;
        for (const at::Tensor *b : read)
            if (!ranges_apart(**a, *b)) return false;
    }
    return true;
}
int32_t *ints(const at::Tensor &t) { return static_cast<int32_t *>(t.data_ptr()); }
at::Tensor make_ints(at::IntArrayRef shape, at::Device dev) { return make(shape, at::TensorOptions().dtype(at::kInt).device(dev)); }

// table, lens, refs, status: what calls on tables have in common.  *page_size is known.
struct Tables {
    at::Tensor table, lens, refs, status, workspace;
    at::Device dev{at::kCPU};
    int64_t rows = 0, width = 0, pages = 0;
    bool read(PyObject *a_table, PyObject *a_lens, PyObject *a_refs, PyObject *a_status) {
        if (!plain(a_refs)) return false;
        refs = THPVariable_Unpack(a_refs);
        if (!refs.defined() || !refs.is_cuda() || refs.device().index() != c10::cuda::current_device()) return false;
        dev = refs.device();
        if (!usable(refs, at::kInt, dev) || refs.dim() != 1 || !indices_of(a_lens, dev, false, &lens) || lens.dim() != 1 ||
            !rows_of(a_table, at::kInt, dev, 2, Use::kWritten, &table) || (a_status != Py_None && (!indices_of(a_status, dev, false, &status) || status.numel() != 1)))
            return false;
        rows = lens.numel(), width = table.size(1), pages = refs.numel();
        return table.size(0) == rows && rows <= CG_MAX_REQUESTS && pages <= INT32_MAX - 1024;
    }
    bool fill(cg_pages_job *job, int64_t page_size) const {
        if (page_size <= 0 || page_size > INT32_MAX || width > INT32_MAX / page_size || width > INT32_MAX - 1024) return false;
        job->table = ints(table), job->kv_lens = ints(lens), job->refs = ints(refs), job->status = status.defined() ? ints(status) : nullptr;
        job->table_row = table.stride(0), job->num_pages = pages;
        job->nrows = static_cast<int32_t>(rows), job->width = static_cast<int32_t>(width), job->page_size = static_cast<int32_t>(page_size);
        return true;
    }
    void with_workspace(cg_pages_job *job) {
        const int64_t need = pages_workspace(pages);
        workspace = make({need}, at::TensorOptions().dtype(at::kByte).device(dev));
        job->workspace = workspace.data_ptr(), job->workspace_bytes = need;
    }
};
// A cache that copies are made in.
struct CacheOf {
    at::Tensor k, v;
    cg_copy_job job{};
    bool read(PyObject *a_k, PyObject *a_v, at::Device dev, const at::Tensor &status) {
        at::Device on(at::kCPU);
        if (!first_of(a_k, &k, &on) || on != dev || k.dim() < 4 || k.dim() > 5 || !rows_of(a_k, k.scalar_type(), dev, k.dim(), Use::kWritten, &k) ||
            !rows_of(a_v, k.scalar_type(), dev, k.dim(), Use::kWritten, &v) || k.sizes() != v.sizes() || !apart(k, v))
            return false;
        const int64_t d = k.dim(), layers = d == 5 ? k.size(0) : 1;
        if (!k.numel() || !fits({layers, k.size(d - 3), k.size(d - 2), k.size(d - 1)})) return false;
        job.pages_k = k.data_ptr(), job.pages_v = v.data_ptr();
        for (int64_t i = 0; i < 4; ++i) {
            const int64_t axis = i + d - 5;
            job.pages_k_strides[i] = axis >= 0 && k.size(axis) > 1 ? k.stride(axis) : 0;
            job.pages_v_strides[i] = axis >= 0 && v.size(axis) > 1 ? v.stride(axis) : 0;
        }
        job.status = status.defined() ? ints(status) : nullptr;
        job.num_pages = k.size(d - 4), job.nlayers = static_cast<int32_t>(layers), job.page_size = static_cast<int32_t>(k.size(d - 3));
        job.heads = static_cast<int32_t>(k.size(d - 2)), job.head_size = static_cast<int32_t>(k.size(d - 1));
        return true;
    }
};
// The page size and the cache, from (k, v, page size), each of which may be None.
bool cache_and_page(PyObject *const *a, const Tables &t, CacheOf *cache, bool *given, int64_t *page_size) {
    *given = a[0] != Py_None;
    if (!*given) return a[1] == Py_None && small_int(a[2], page_size);
    if (!cache->read(a[0], a[1], t.dev, t.status) || cache->job.num_pages != t.pages) return false;
    *page_size = cache->job.page_size;
    int64_t said;
    return a[2] == Py_None || (small_int(a[2], &said) && said == *page_size);
}
int run_pages(int (*entry)(const cg_pages_job *, const cg_copy_job *, void *), const cg_pages_job &job, const cg_copy_job *copy, at::Device dev) {
    void *stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
    const WithoutGil released;
    return entry(&job, copy, stream);
}

// copy_pages(k, v, src, dst, tokens or None, status) -> True, an error code, or None
PyObject *copy_pages(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor first, src, dst, tokens, status;
    at::Device dev(at::kCPU);
    CacheOf cache;
    if (n != 6 || !first_of(a[0], &first, &dev) || (a[5] != Py_None && (!indices_of(a[5], dev, false, &status) || status.numel() != 1)) ||
        !cache.read(a[0], a[1], dev, status) || !indices_of(a[2], dev, true, &src) || src.dim() != 1 || !indices_of(a[3], dev, true, &dst) ||
        dst.scalar_type() != src.scalar_type() || dst.sizes() != src.sizes() ||
        (a[4] != Py_None && (!indices_of(a[4], dev, false, &tokens) || tokens.sizes() != src.sizes())) || !fits({src.numel()}) ||
        !all_apart({&cache.k}, {&src, &dst, &tokens}) || !all_apart({&cache.v}, {&src, &dst, &tokens}))
        Py_RETURN_NONE;
    cg_copy_job &job = cache.job;
    job.src = src.data_ptr(), job.dst = dst.data_ptr(), job.tokens = tokens.defined() ? ints(tokens) : nullptr;
    job.wide = src.scalar_type() == at::kLong, job.ncopies = static_cast<int32_t>(src.numel());
    const int rc = run(copy_rows, job, dev);
    if (rc) return PyLong_FromLong(rc);
    wrote(cache.k), wrote(cache.v);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// fork(table, lens, parents, refs, k or None, v or None, page size or None, release, out or None, status) -> (table, lens, moves), an error code, or None
PyObject *fork_pages(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tables t;
    CacheOf cache;
    at::Tensor parents, table, lens;
    bool given;
    int64_t page_size;
    cg_pages_job job{};
    if (n != 10 || !t.read(a[0], a[1], a[3], a[9]) || !indices_of(a[2], t.dev, true, &parents) || parents.dim() != 1 || parents.numel() > CG_MAX_REQUESTS ||
        !cache_and_page(a + 4, t, &cache, &given, &page_size) || !t.fill(&job, page_size))
        Py_RETURN_NONE;
    const int64_t N = parents.numel();
    if (a[8] != Py_None) {
        if (!PyTuple_CheckExact(a[8]) || PyTuple_GET_SIZE(a[8]) != 2 || !rows_of(PyTuple_GET_ITEM(a[8], 0), at::kInt, t.dev, 2, Use::kWritten, &table) ||
            table.size(0) != N || table.size(1) != t.width || !indices_of(PyTuple_GET_ITEM(a[8], 1), t.dev, false, &lens) || lens.dim() != 1 || lens.numel() != N)
            Py_RETURN_NONE;
    }
    if (!all_apart({&t.refs, &table, &lens, &cache.k}, {&t.table, &t.lens, &parents}) || !all_apart({&t.refs, &table, &lens, &cache.v}, {&t.table, &t.lens, &parents}))
        Py_RETURN_NONE;
    if (a[8] == Py_None) table = make_ints({N, t.width}, t.dev), lens = make_ints({N}, t.dev);
    const at::Tensor moves = make_ints({3, N}, t.dev);
    job.which = parents.data_ptr(), job.wide = parents.scalar_type() == at::kLong, job.release = a[7] == Py_True;
    job.new_table = ints(table), job.new_lens = ints(lens), job.moves = ints(moves), job.new_table_row = table.stride(0), job.nnew = static_cast<int32_t>(N);
    t.with_workspace(&job);
    const int rc = run_pages(fork_rows, job, given ? &cache.job : nullptr, t.dev);
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor *x : {&t.refs, &table, &lens, &cache.k, &cache.v}) wrote(*x);
    if (a[8] == Py_None) return Py_BuildValue("(NNN)", THPVariable_Wrap(table), THPVariable_Wrap(lens), THPVariable_Wrap(moves));
    return Py_BuildValue("(OON)", PyTuple_GET_ITEM(a[8], 0), PyTuple_GET_ITEM(a[8], 1), THPVariable_Wrap(moves));
    END_HANDLE_TH_ERRORS
}

// free_pages(table, lens, refs, page size, rows or None, status) -> True, an error code, or None
PyObject *free_pages(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tables t;
    at::Tensor rows;
    int64_t page_size;
    cg_pages_job job{};
    if (n != 6 || !t.read(a[0], a[1], a[2], a[5]) || !small_int(a[3], &page_size) || !t.fill(&job, page_size)) Py_RETURN_NONE;
    if (a[4] != Py_None) {
        if (!indices_of(a[4], t.dev, true, &rows) || rows.dim() != 1 || rows.numel() > CG_MAX_REQUESTS) Py_RETURN_NONE;
        if (!rows.numel()) Py_RETURN_TRUE;
        job.which = rows.data_ptr(), job.wide = rows.scalar_type() == at::kLong, job.nnew = static_cast<int32_t>(rows.numel());
    }
    if (!all_apart({&t.refs, &t.table, &t.lens}, {&rows})) Py_RETURN_NONE;
    const int rc = run(free_rows, job, t.dev);
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor *x : {&t.refs, &t.table, &t.lens}) wrote(*x);
    Py_RETURN_TRUE;
    END_HANDLE_TH_ERRORS
}

// extend(table, lens, refs, page size, q_starts or None, tokens or None, status) -> slots, an error code, or None
PyObject *extend_pages(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tables t;
    at::Tensor starts;
    int64_t page_size, tokens;
    cg_pages_job job{};
    if (n != 7 || !t.read(a[0], a[1], a[2], a[6]) || !small_int(a[3], &page_size) || !t.fill(&job, page_size)) Py_RETURN_NONE;
    if (a[4] == Py_None) {
        if (a[5] != Py_None && (!small_int(a[5], &tokens) || tokens != t.rows)) Py_RETURN_NONE;
        tokens = t.rows;
    } else {
        if (!small_int(a[5], &tokens) || tokens < 0 || tokens > INT32_MAX || !t.rows || !indices_of(a[4], t.dev, false, &starts) || starts.dim() != 1 ||
            starts.numel() != t.rows + 1)
            Py_RETURN_NONE;
        job.q_starts = ints(starts);
    }
    if (!all_apart({&t.refs, &t.table, &t.lens}, {&starts})) Py_RETURN_NONE;
    const at::Tensor slots = make({tokens}, at::TensorOptions().dtype(at::kLong).device(t.dev));
    job.slots = static_cast<int64_t *>(slots.data_ptr()), job.ntokens = static_cast<int32_t>(tokens);
    t.with_workspace(&job);
    const int rc = run(extend_rows, job, t.dev);
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor *x : {&t.refs, &t.table, &t.lens}) wrote(*x);
    return THPVariable_Wrap(slots);
    END_HANDLE_TH_ERRORS
}

// compact(table, lens, refs, k or None, v or None, page size or None, status) -> (places, moves), an error code, or None
PyObject *compact_pages(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    Tables t;
    CacheOf cache;
    bool given;
    int64_t page_size;
    cg_pages_job job{};
    if (n != 7 || !t.read(a[0], a[1], a[2], a[6]) || !cache_and_page(a + 3, t, &cache, &given, &page_size) || !t.fill(&job, page_size) ||
        !all_apart({&t.refs, &t.table, &cache.k}, {&t.lens}) || !all_apart({&t.refs, &t.table, &cache.v}, {&t.lens}))
        Py_RETURN_NONE;
    const at::Tensor places = make_ints({t.pages}, t.dev), moves = make_ints({2, t.pages / 2}, t.dev);
    job.places = ints(places), job.moves = ints(moves);
    t.with_workspace(&job);
    const int rc = run_pages(compact_rows, job, given ? &cache.job : nullptr, t.dev);
    if (rc) return PyLong_FromLong(rc);
    for (const at::Tensor *x : {&t.refs, &t.table, &cache.k, &cache.v}) wrote(*x);
    return Py_BuildValue("(NN)", THPVariable_Wrap(places), THPVariable_Wrap(moves));
    END_HANDLE_TH_ERRORS
}

// beam_select(logits, scores, k) -> (scores, tokens, parents), an error code, or None
PyObject *beam_select(PyObject *, PyObject *const *a, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    at::Tensor logits, scores;
    int64_t k;
    if (n != 3 || !plain(a[0]) || !plain(a[1]) || !small_int(a[2], &k)) Py_RETURN_NONE;
    logits = THPVariable_Unpack(a[0]), scores = THPVariable_Unpack(a[1]);
    if (!logits.defined() || !logits.is_cuda() || logits.device().index() != c10::cuda::current_device()) Py_RETURN_NONE;
    const at::Device dev = logits.device();
    const at::ScalarType type = logits.scalar_type();
    if ((!is_16bit(type) && type != at::kFloat) || !rows_of(a[0], type, dev, 2, Use::kRead, &logits) || !usable(scores, at::kFloat, dev) || scores.requires_grad() ||
        scores.dim() != 2)
        Py_RETURN_NONE;
    const int64_t B = scores.size(0), K = scores.size(1), V = logits.size(1);
    if (logits.size(0) != B * K || K <= 0 || K > CG_MAX_BEAMS || k <= 0 || k > CG_MAX_CHOICES || K * k > CG_MAX_BEAM_CHOICES || V <= 0 || V > CG_MAX_VOCAB ||
        B > INT32_MAX)
        Py_RETURN_NONE;
    const at::Tensor out = make({B, k}, scores.options()), tokens = make_ints({B, k}, dev), parents = make_ints({B, k}, dev);
    cg_beam_job job{};
    job.logits = logits.data_ptr(), job.scores = static_cast<const float *>(scores.data_ptr());
    job.out_scores = static_cast<float *>(out.data_ptr()), job.tokens = ints(tokens), job.parents = ints(parents);
    job.dtype = type == at::kFloat ? CG_LOGITS_F32 : code(type), job.row_stride = logits.stride(0);
    job.nrequests = static_cast<int32_t>(B), job.beams = static_cast<int32_t>(K), job.vocab = static_cast<int32_t>(V), job.k = static_cast<int32_t>(k);
    const int64_t need = beam_workspace(&job);
    if (need < 0) Py_RETURN_NONE;  // more than a call takes: the general path says what
    const at::Tensor workspace = make({need}, at::TensorOptions().dtype(at::kByte).device(dev));
    job.workspace = workspace.data_ptr(), job.workspace_bytes = need;
    const int rc = run(best_beams, job, dev);
    if (rc) return PyLong_FromLong(rc);
    return Py_BuildValue("(NNN)", THPVariable_Wrap(out), THPVariable_Wrap(tokens), THPVariable_Wrap(parents));
    END_HANDLE_TH_ERRORS
}

// bind({name: address})
PyObject *bind(PyObject *, PyObject *addresses) {
    HANDLE_TH_ERRORS
    const auto address = [&](const char *name) {
        PyObject *v = PyDict_GetItemString(addresses, name);
        if (!v) throw std::runtime_error(std::string("bind: no ") + name);
        return reinterpret_cast<void *>(integer(v));
    };
    decode_kv = reinterpret_cast<decltype(decode_kv)>(address("cg_decode_kv"));
    encode_kv = reinterpret_cast<decltype(encode_kv)>(address("cg_encode_kv"));
    encode_kv_workspace = reinterpret_cast<decltype(encode_kv_workspace)>(address("cg_encode_kv_workspace"));
    encode_kv_wait = reinterpret_cast<decltype(encode_kv_wait)>(address("cg_encode_kv_wait"));
    encode_kv_gather = reinterpret_cast<decltype(encode_kv_gather)>(address("cg_encode_kv_gather"));
    rotary_rows = reinterpret_cast<decltype(rotary_rows)>(address("cg_rotary"));
    append_rows = reinterpret_cast<decltype(append_rows)>(address("cg_append_paged"));
    gather_rows = reinterpret_cast<decltype(gather_rows)>(address("cg_gather_paged"));
    attention_workspace = reinterpret_cast<decltype(attention_workspace)>(address("cg_paged_attention_workspace"));
    attention = reinterpret_cast<decltype(attention)>(address("cg_paged_attention"));
    pages_workspace = reinterpret_cast<decltype(pages_workspace)>(address("cg_pages_workspace"));
    copy_rows = reinterpret_cast<decltype(copy_rows)>(address("cg_copy_pages"));
    fork_rows = reinterpret_cast<decltype(fork_rows)>(address("cg_fork_pages"));
    free_rows = reinterpret_cast<decltype(free_rows)>(address("cg_free_pages"));
    extend_rows = reinterpret_cast<decltype(extend_rows)>(address("cg_extend_pages"));
    compact_rows = reinterpret_cast<decltype(compact_rows)>(address("cg_compact_pages"));
    beam_workspace = reinterpret_cast<decltype(beam_workspace)>(address("cg_beam_workspace"));
    best_beams = reinterpret_cast<decltype(best_beams)>(address("cg_beam_select"));
    Py_RETURN_NONE;
    END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {{"bind", bind, METH_O, nullptr},
                         {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL, nullptr},
                         {"encode_start", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(encode_start)), METH_FASTCALL, nullptr},
                         {"encode_finish", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(encode_finish)), METH_FASTCALL, nullptr},
                         {"rotary", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rotary)), METH_FASTCALL, nullptr},
                         {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
                         {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gather)), METH_FASTCALL, nullptr},
                         {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
                         {"copy_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(copy_pages)), METH_FASTCALL, nullptr},
                         {"fork_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(fork_pages)), METH_FASTCALL, nullptr},
                         {"free_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(free_pages)), METH_FASTCALL, nullptr},
                         {"extend_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(extend_pages)), METH_FASTCALL, nullptr},
                         {"compact_pages", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(compact_pages)), METH_FASTCALL, nullptr},
                         {"beam_select", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(beam_select)), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls() {
    s_cdf = PyUnicode_InternFromString("cdf");
    s_max_tensors_key = PyUnicode_InternFromString("max_tensors_key");
    s_max_tensors_value = PyUnicode_InternFromString("max_tensors_value");
    s_data_chunks = PyUnicode_InternFromString("data_chunks");
    s_num_heads = PyUnicode_InternFromString("num_heads");
    s_head_size = PyUnicode_InternFromString("head_size");
    s_bytestream = PyUnicode_InternFromString("bytestream");
    s_bytestream_lengths = PyUnicode_InternFromString("bytestream_lengths");
    s_ntokens = PyUnicode_InternFromString("ntokens");
    s_group_off = PyUnicode_InternFromString("group_off");
    s_captured = PyUnicode_InternFromString("captured");
    s_blob = PyUnicode_InternFromString("blob");
    s_header = PyUnicode_InternFromString("header");
    s_sub_off = PyUnicode_InternFromString("sub_off");
    for (int k = 0; k < kHeaderFields; ++k) s_header_fields[k] = PyUnicode_InternFromString(kHeaderNames[k]);
    PyObject *const m = PyModule_Create(&module);
    if (m && PyModule_AddStringConstant(m, "built_for", CG_BUILT_FOR)) {  // see build.py
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
