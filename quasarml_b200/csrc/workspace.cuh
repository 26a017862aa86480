// Device workspace of one call, and the joining of column sums: what the
// operators with a backward pass share.
#pragma once

#include <new>

#include "qsml_internal.cuh"

// The end of an entry point (extern "C" ... f(...) try { ... } QSML_NO_THROW): the
// standard library's exceptions, thrown where host memory runs out, become a status.
#define QSML_NO_THROW                                  \
    catch (const std::bad_alloc&) { return QSML_E_OOM; } \
    catch (...) { return QSML_E_INVALID; }

namespace qsml {

// Workspace of one call.  Outside stream capture it comes from the context's
// caching allocator and goes back when the call returns (reuse is in stream
// order, as for every block of the allocator).  A call that is being captured
// into a graph takes it from the stream's own allocator instead
// (cudaMallocAsync / cudaFreeAsync, recorded as the graph's allocation nodes):
// the memory belongs to the graph, so no later call, tensor or second graph
// is given it while the graph may still be replayed.
class Workspace {
public:
    explicit Workspace(Context* ctx) : ctx_(ctx) {}
    ~Workspace();
    Workspace(const Workspace&) = delete;
    Workspace& operator=(const Workspace&) = delete;
    // `bytes` bytes at *ptr, 256-byte aligned; at most kMax blocks a call.
    qsml_status_t get(size_t bytes, void** ptr);
    // Whether the last block belongs to a graph.
    bool captured() const { return n_ > 0 && captured_[n_ - 1]; }

private:
    static constexpr int kMax = 12;
    Context* ctx_;
    int n_ = 0;
    void* ptr_[kMax];
    bool captured_[kMax];
};

// out[c] = sum over p of partial[p * cols + c] for c < cols, added in a fixed
// order and rounded once to out_dtype (F32 or F16).  Up to two sums of the
// same size in one launch (a sum whose `out` is null is left out).
struct ColumnSum {
    const float* partial = nullptr;
    void* out = nullptr;
    int32_t out_dtype = QSML_F32;
};
qsml_status_t finish_column_sums(Context* ctx, const ColumnSum& s0, const ColumnSum& s1, int64_t parts, int64_t cols);

// True if the bytes of the two views' spans meet.
inline bool views_meet(const qsml_tdesc* a, const qsml_tdesc* b) {
    const Span x = view_span(a), y = view_span(b);
    return x.lo < x.hi && y.lo < y.hi && x.lo < y.hi && y.lo < x.hi;
}

}  // namespace qsml
