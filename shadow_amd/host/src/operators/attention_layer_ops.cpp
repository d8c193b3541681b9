// Connected4, RotaryNorm, WindowAttention: the attention half of a transformer's layer on
// fp32 blobs, and int32 blobs for packed weights and positions.  The reference has no such
// operators; they are registered beside its own (REGISTER_EXTENSION).
#include <cmath>

#include "shadow/kernels/attention_layer.hpp"
#include "shadow/operator.hpp"

namespace Shadow {

namespace {

using Blobs = std::vector<std::shared_ptr<Blob>>;

// The inputs one after another; an optional one is there if its argument says so.
class Inputs {
 public:
  Inputs(const Operator* op, const Blobs& inputs) : op_(op), inputs_(inputs) {}
  const std::shared_ptr<Blob>& next(DataType type, const char* what) {
    CHECK_LT(at_, inputs_.size()) << op_->name() << ": no input for " << what;
    const auto& blob = inputs_[at_++];
    CHECK(blob->data_type() == type) << op_->name() << ": " << what << " must be "
                                     << (type == DataType::kI32 ? "an int32" : "a float") << " blob";
    return blob;
  }
  const float* floats(bool there, int count, const char* what) {
    if (!there) return nullptr;
    const auto& blob = next(DataType::kF32, what);
    CHECK_EQ(blob->count(), count) << op_->name() << ": " << what;
    return blob->data<float>();
  }
  const int* ints(bool there, int count, const char* what) {
    if (!there) return nullptr;
    const auto& blob = next(DataType::kI32, what);
    CHECK_EQ(blob->count(), count) << op_->name() << ": " << what;
    return blob->data<int>();
  }
  // No input may be an output: its memory may go when that one gets its shape.
  void done(const Blobs& outputs) const {
    CHECK_EQ(at_, inputs_.size()) << op_->name() << ": inputs left over";
    for (const auto& output : outputs) {
      CHECK(output->data_type() == DataType::kF32) << op_->name() << ": outputs are float blobs";
      for (const auto& input : inputs_) CHECK_NE(input, output) << op_->name() << ": an output is an input";
    }
  }

 private:
  const Operator* op_;
  const Blobs& inputs_;
  size_t at_ = 0;
};

// Blob counts are int32.
VecInt countable(const VecInt& shape, const std::string& name) {
  long long count = 1;
  for (int d : shape) {
    CHECK_GT(d, 0) << name;
    count *= d;
    CHECK_LE(count, 2147483647LL) << name << ": blob too large";
  }
  return shape;
}

}  // namespace

// Inputs x, codes (int32 [out, in / 8]), steps [out, ceil(in / group)], then lows (has_lows)
// and bias (has_bias).  `axis` (default -1): the axes from there on are `in`, the output has
// `out` in their place.
class Connected4Op : public Operator {
 public:
  Connected4Op(const shadow::OpParam& op_param, Workspace* ws) : Operator(op_param, ws) {
    axis_ = get_single_argument<int>("axis", -1);
    group_ = get_single_argument<int>("group", 128);
    has_lows_ = get_single_argument<bool>("has_lows", false);
    has_bias_ = get_single_argument<bool>("has_bias", false);
    CHECK(group_ == 32 || group_ == 64 || group_ == 128) << name() << ": group must be 32, 64 or 128";
  }

  void Run(const Blobs& inputs, Blobs& outputs) override {
    Inputs in(this, inputs);
    const auto& x = in.next(DataType::kF32, "x");
    const auto& codes = in.next(DataType::kI32, "codes");
    const int axis = x->canonical_index(axis_);
    const int size = x->count(axis), rows = x->count(0, axis);
    CHECK_EQ(size % 8, 0);
    CHECK_EQ(codes->num_axes(), 2);
    CHECK_EQ(codes->shape(1), size / 8);
    const int out = codes->shape(0), groups = (size + group_ - 1) / group_;
    const float* steps = in.floats(true, out * groups, "steps");
    const float* lows = in.floats(has_lows_, out * groups, "lows");
    const float* bias = in.floats(has_bias_, out, "bias");
    in.done(outputs);
    auto& output = outputs[0];
    VecInt shape(x->shape().begin(), x->shape().begin() + axis);
    shape.push_back(out);
    output->reshape(countable(shape, name()));
    Vision::Connected4<DeviceType::kGPU, float>(x->data<float>(), rows, size, out, group_, codes->data<int>(), steps, lows, bias,
                                                output->mutable_data<float>(), ws_);
  }

 private:
  int axis_, group_;
  bool has_lows_, has_bias_;
};

REGISTER_EXTENSION(Connected4, Connected4Op);

// Inputs x [batch, length, ...] with (q_heads + 2 kv_heads) * head_dim values a token, frequency
// (rotary_dim > 0; default head_dim), q_scale and k_scale (has_scale), starts (has_starts) and
// lengths (has_lengths), int32 of `batch`.  Outputs q [batch, length, q_heads, head_dim], k and v
// [batch, kv_heads, capacity or, where capacity is 0, length, head_dim].  With a capacity k and v
// are caches: rows that a run does not write keep what earlier runs wrote, until their shape changes.
class RotaryNormOp : public Operator {
 public:
  RotaryNormOp(const shadow::OpParam& op_param, Workspace* ws) : Operator(op_param, ws) {
    shape_.q_heads = get_single_argument<int>("q_heads", 0);
    shape_.kv_heads = get_single_argument<int>("kv_heads", shape_.q_heads);
    shape_.head_dim = get_single_argument<int>("head_dim", 0);
    shape_.rotary_dim = get_single_argument<int>("rotary_dim", shape_.head_dim - shape_.head_dim % 2);
    shape_.capacity = get_single_argument<int>("capacity", 0);
    interleaved_ = get_single_argument<bool>("interleaved", false);
    normalize_ = get_single_argument<bool>("normalize", true);
    has_scale_ = get_single_argument<bool>("has_scale", false);
    has_starts_ = get_single_argument<bool>("has_starts", false);
    has_lengths_ = get_single_argument<bool>("has_lengths", false);
    eps_ = get_single_argument<float>("eps", 1e-6f);
    CHECK_GT(shape_.q_heads, 0);
    CHECK_GT(shape_.kv_heads, 0);
    CHECK_GT(shape_.head_dim, 0);
    CHECK_GE(shape_.capacity, 0);
    CHECK_EQ(op_param.top_size(), 3) << name() << ": outputs are q, k and v";
  }

  void Run(const Blobs& inputs, Blobs& outputs) override {
    Inputs in(this, inputs);
    const auto& x = in.next(DataType::kF32, "x");
    CHECK_GE(x->num_axes(), 3);
    auto shape = shape_;
    shape.batch = x->shape(0), shape.length = x->shape(1);
    CHECK_EQ(static_cast<long long>(x->count(2)),
             (static_cast<long long>(shape.q_heads) + 2LL * shape.kv_heads) * shape.head_dim) << name() << ": values of a token";
    const float* frequency = in.floats(shape.rotary_dim > 0, shape.rotary_dim / 2, "frequency");
    const float* q_scale = in.floats(has_scale_, shape.head_dim, "q_scale");
    const float* k_scale = in.floats(has_scale_, shape.head_dim, "k_scale");
    const int* starts = in.ints(has_starts_, shape.batch, "starts");
    const int* lengths = in.ints(has_lengths_, shape.batch, "lengths");
    in.done(outputs);
    outputs[0]->reshape(countable({shape.batch, shape.length, shape.q_heads, shape.head_dim}, name()));
    const VecInt cache = countable(
        {shape.batch, shape.kv_heads, shape.capacity > 0 ? shape.capacity : shape.length, shape.head_dim}, name());
    outputs[1]->reshape(cache);
    outputs[2]->reshape(cache);
    Vision::RotaryNorm<DeviceType::kGPU, float>(x->data<float>(), shape, interleaved_, normalize_, eps_, q_scale, k_scale,
                                                frequency, starts, lengths, outputs[0]->mutable_data<float>(),
                                                outputs[1]->mutable_data<float>(), outputs[2]->mutable_data<float>(),
                                                ws_->Ctx().get());
  }

 private:
  Vision::RotaryNormShape shape_;
  bool interleaved_, normalize_, has_scale_, has_starts_, has_lengths_;
  float eps_;
};

REGISTER_EXTENSION(RotaryNorm, RotaryNormOp);

// Inputs q [batch, length, q_heads, head_dim], k and v [batch, kv_heads, capacity, head_dim],
// then starts (has_starts) and lengths (has_lengths), int32 of `batch`.  `window` (default 0: no
// limit), `sinks` (default 0), `causal` (default true), `scale` (default 1 / sqrt(head_dim)).
// The output has q's shape.
class WindowAttentionOp : public Operator {
 public:
  WindowAttentionOp(const shadow::OpParam& op_param, Workspace* ws) : Operator(op_param, ws) {
    window_ = get_single_argument<int>("window", 0);
    sinks_ = get_single_argument<int>("sinks", 0);
    causal_ = get_single_argument<bool>("causal", true);
    scale_ = get_single_argument<float>("scale", 0.f);
    has_scale_ = has_argument("scale");
    has_starts_ = get_single_argument<bool>("has_starts", false);
    has_lengths_ = get_single_argument<bool>("has_lengths", false);
    CHECK_GE(window_, 0);
    CHECK_GE(sinks_, 0);
  }

  void Run(const Blobs& inputs, Blobs& outputs) override {
    Inputs in(this, inputs);
    const auto& q = in.next(DataType::kF32, "q");
    const auto& k = in.next(DataType::kF32, "k");
    const auto& v = in.next(DataType::kF32, "v");
    CHECK_EQ(q->num_axes(), 4);
    CHECK_EQ(k->num_axes(), 4);
    CHECK(k->shape() == v->shape());
    CHECK_EQ(q->shape(0), k->shape(0));
    CHECK_EQ(q->shape(3), k->shape(3));
    CHECK_EQ(q->shape(2) % k->shape(1), 0);
    const Vision::WindowAttentionShape shape = {q->shape(0), q->shape(1), q->shape(2), k->shape(1),
                                                q->shape(3), k->shape(2), window_,     sinks_};
    const int* starts = in.ints(has_starts_, shape.batch, "starts");
    const int* lengths = in.ints(has_lengths_, shape.batch, "lengths");
    in.done(outputs);
    auto& output = outputs[0];
    output->reshape(q->shape());
    const float scale = has_scale_ ? scale_ : 1.f / std::sqrt(static_cast<float>(shape.head_dim));
    Vision::WindowAttention<DeviceType::kGPU, float>(q->data<float>(), k->data<float>(), v->data<float>(), shape, causal_, scale,
                                                     starts, lengths, output->mutable_data<float>(), ws_);
  }

 private:
  int window_, sinks_;
  bool causal_, has_scale_, has_starts_, has_lengths_;
  float scale_;
};

REGISTER_EXTENSION(WindowAttention, WindowAttentionOp);

}  // namespace Shadow
