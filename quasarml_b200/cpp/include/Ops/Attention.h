// The attention sublayer's operators (additions of this backend; the reference has
// none of them): norms of queries and keys for each head with the rotation by
// positions, attention with a sliding window and first tokens that stay visible,
// and their backward passes.  Each is one call of the C ABI.
#pragma once

#include <memory>
#include <vector>

#include "../Core/Device.h"
#include "../Core/Tensor.h"

namespace QuasarML {

// Same codes as QSML_ROTARY_*: columns (i, n + i) or (2 i, 2 i + 1) are a pair.
enum class RotaryPairing : u32 { Halves = 0, Pairs };

struct RotaryOptions {
    f32 eps = 1e-6f;
    std::vector<i32> sections;  // pairs that go by each axis of the positions; empty: one axis
    RotaryPairing pairing = RotaryPairing::Halves;
};
struct QueriesKeys {
    std::shared_ptr<Tensor> q, k;
};
struct NormRotaryGrads {
    std::shared_ptr<Tensor> dq, dk, dwq, dwk;  // dk, dwq, dwk null where k, wq, wk are
};

struct AttentionOptions {
    f32 scale = 0.0f;  // 0: 1 / sqrt(columns)
    u64 window = 0;    // 0: all earlier tokens
    u64 sinks = 0;     // first tokens that stay visible
    std::shared_ptr<Tensor> q_lengths = nullptr, k_lengths = nullptr;  // I32 [sequences]; null: all
};
struct AttentionGrads {
    std::shared_ptr<Tensor> dq, dk, dv;
};

namespace Ops {

// q [tokens, heads, columns] (or with sequences in front), k alike (or null), read in place as slices of
// a projection; wq, wk [columns] or null; positions I32 [tokens], with a last dim of axes where there are
// sections; frequencies F32 [pairs].
QS_API QueriesKeys norm_rotary(Device& device, std::shared_ptr<Tensor> q, std::shared_ptr<Tensor> k, std::shared_ptr<Tensor> wq,
                               std::shared_ptr<Tensor> wk, std::shared_ptr<Tensor> positions,
                               std::shared_ptr<Tensor> frequencies, const RotaryOptions& options = {});
// dwq and dwk have their weights' dtype.
QS_API NormRotaryGrads norm_rotary_backward(Device& device, std::shared_ptr<Tensor> q, std::shared_ptr<Tensor> k,
                                            std::shared_ptr<Tensor> wq, std::shared_ptr<Tensor> wk,
                                            std::shared_ptr<Tensor> positions, std::shared_ptr<Tensor> frequencies,
                                            std::shared_ptr<Tensor> dq_out, std::shared_ptr<Tensor> dk_out,
                                            const RotaryOptions& options = {});

// q [sequences, queries, heads, columns], k and v [sequences, keys, kv heads, columns].  keep_lse: takes
// what attention_backward reads.
QS_API std::shared_ptr<Tensor> attention(Device& device, std::shared_ptr<Tensor> q, std::shared_ptr<Tensor> k,
                                         std::shared_ptr<Tensor> v, const AttentionOptions& options = {},
                                         std::shared_ptr<Tensor>* keep_lse = nullptr);
QS_API AttentionGrads attention_backward(Device& device, std::shared_ptr<Tensor> q, std::shared_ptr<Tensor> k,
                                         std::shared_ptr<Tensor> v, std::shared_ptr<Tensor> o, std::shared_ptr<Tensor> lse,
                                         std::shared_ptr<Tensor> dout, const AttentionOptions& options = {});

}  // namespace Ops
}  // namespace QuasarML
