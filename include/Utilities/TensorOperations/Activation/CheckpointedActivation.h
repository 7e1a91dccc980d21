// Activations that keep their input as an 8-bit checkpoint, and their backward pass from it.
//
//   forward   output = f(input), or f(input) * multiplier (gated layers), and checkpoints of input and multiplier, in one pass
//   backward  input_gradient = error * f'(x), or error * z * f'(x), and multiplier_gradient = error * f(x), where x and z are what the
//             checkpoints stand for (an infinity counts as the largest finite number there)
// with f one of relu, gelu(x) = x * Phi(x) and swish(x) = x * sigmoid(x), as Expression's methods of these names; relu's slope at zero
// is zero, and a NaN stays a NaN in value and slope.  All arithmetic is fp32, rounded once to the output's type: fp32 values are within
// ten units of 2^-24 of f over the whole range, subnormal results included, and 16-bit ones within 2e-5 before their rounding.  The tensors
// of a call share one shape and one of the types FP32, FP16, BF16; strides, segment_offsets, overlaps and errors as in
// ActivationCheckpoint.h.
#pragma once

#include "Utilities/TensorOperations/DataTypeConversions/ActivationCheckpoint.h"

namespace ThorImplementation {

enum class ActivationKind : int { Relu = THORHIP_RELU, Gelu = THORHIP_GELU, Swish = THORHIP_SWISH };

class StampedCheckpointedActivation : public StampedRowOperation {
   public:
    Tensor getOutputTensor() const { return output; }
    const ActivationCheckpoint& getCheckpoint() const { return checkpoint; }
    const std::optional<ActivationCheckpoint>& getMultiplierCheckpoint() const { return multiplierCheckpoint; }

   private:
    friend class CheckpointedActivation;
    explicit StampedCheckpointedActivation(const Stream& stream) : StampedRowOperation(stream) {}
    void enqueue(void* raw_stream) const override;

    Tensor input, output;
    std::optional<Tensor> multiplier, segmentOffsets;
    ActivationCheckpoint checkpoint;
    std::optional<ActivationCheckpoint> multiplierCheckpoint;
    thorhip_checkpointed call{};
};

class CheckpointedActivation {
   public:
    struct Outputs {
        std::optional<Tensor> output;
        std::optional<ActivationCheckpoint> checkpoint;
        std::optional<ActivationCheckpoint> multiplier_checkpoint;
    };
    CheckpointedActivation(ActivationKind kind, DataType checkpoint_dtype);
    std::shared_ptr<StampedCheckpointedActivation> stamp(const Tensor& input, const Stream& stream, const std::optional<Tensor>& multiplier = std::nullopt,
                                                         const std::optional<Tensor>& segment_offsets = std::nullopt, const Outputs& preallocated = {}) const;

   private:
    ActivationKind kind;
    DataType dtype;
};

class StampedCheckpointedActivationBackward : public StampedRowOperation {
   public:
    Tensor getInputGradientTensor() const { return inputGradient; }
    const std::optional<Tensor>& getMultiplierGradientTensor() const { return multiplierGradient; }

   private:
    friend class CheckpointedActivationBackward;
    explicit StampedCheckpointedActivationBackward(const Stream& stream) : StampedRowOperation(stream) {}
    void enqueue(void* raw_stream) const override;

    Tensor error, inputGradient;
    std::optional<Tensor> multiplierGradient, segmentOffsets;
    ActivationCheckpoint checkpoint;
    std::optional<ActivationCheckpoint> multiplierCheckpoint;
    thorhip_checkpointed call{};
};

class CheckpointedActivationBackward {
   public:
    struct Outputs {
        std::optional<Tensor> input_gradient;
        std::optional<Tensor> multiplier_gradient;
    };
    explicit CheckpointedActivationBackward(ActivationKind kind);
    // The multiplier's checkpoint must be of the input's checkpoint's type.
    std::shared_ptr<StampedCheckpointedActivationBackward> stamp(const Tensor& error_input, const ActivationCheckpoint& checkpoint, const Stream& stream,
                                                                 const std::optional<ActivationCheckpoint>& multiplier_checkpoint = std::nullopt,
                                                                 const std::optional<Tensor>& segment_offsets = std::nullopt,
                                                                 const Outputs& preallocated = {}) const;

   private:
    ActivationKind kind;
};

}  // namespace ThorImplementation
