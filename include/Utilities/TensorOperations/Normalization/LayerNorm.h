// Layer norm over the last axis, its gradients, and both with the normalised rows kept as an 8-bit checkpoint.
//
//   forward   mean = sum x / C,  rstd = 1 / sqrt(sum (x - mean)^2 / C + epsilon),  h = (x - mean) * rstd,  output = h * weight + bias
//   backward  g = error * weight,  input_gradient = rstd * (g - sum g / C - h * (sum g h / C)),
//             weight_gradient = sum over rows of error * h,  bias_gradient = sum over rows of error
// with h from the input, mean and rstd of the forward pass, or from the checkpoint of h that the forward pass wrote (which is all that
// has to be kept of a row then, beside rstd).
//
// Input, error, output and input gradient are FP32, FP16 or BF16, one type per call, with adjacent elements on the last axis (any
// stride on the leading ones, as long as they collapse to two), rows of fewer than 2^24 elements.  epsilon is a
// positive normal fp32 number.  weight and bias are dense [C] in FP32 or the input's type (one type for
// both); without them h is multiplied with ones and nothing is added.  mean and rstd are dense FP32 [..., 1].  The gradients of weight
// and bias are dense [C] in the weight's type, FP32 without a weight.  All arithmetic is fp32, rounded once where a tensor is stored;
// the output and the checkpoint have the precision of x - mean however large the mean is, the backward pass from the input that of the
// stored mean.  Differences of 2^64 and more have squares over fp32's range: rstd is zero then, and the output the bias.  Results are the
// same bits from run to run.  segment_offsets (UINT32 or UINT64 [B+1], read when the kernels run) marks a packed ragged
// batch: rows at and behind the last offset are neither read nor written and add nothing to a gradient.  No output may overlap another
// tensor of the call.  Errors are std::invalid_argument.  The reference has no counterpart (its normalisations are a vendor library's).
#pragma once

#include "Utilities/TensorOperations/DataTypeConversions/ActivationCheckpoint.h"

namespace ThorImplementation {

class StampedLayerNorm : public StampedRowOperation {
   public:
    Tensor getOutputTensor() const { return output; }
    Tensor getMeanTensor() const { return mean; }
    Tensor getReciprocalDeviationTensor() const { return rstd; }
    const std::optional<ActivationCheckpoint>& getCheckpoint() const { return checkpoint; }

   private:
    friend class LayerNorm;
    explicit StampedLayerNorm(const Stream& stream) : StampedRowOperation(stream) {}
    void enqueue(void* raw_stream) const override;

    Tensor input, output, mean, rstd;
    std::optional<Tensor> weight, bias, segmentOffsets;
    std::optional<ActivationCheckpoint> checkpoint;
    thorhip_layer_norm call{};
};

class LayerNorm {
   public:
    struct Outputs {
        std::optional<Tensor> output, mean, reciprocal_deviation;
        std::optional<ActivationCheckpoint> checkpoint;
    };
    explicit LayerNorm(double epsilon = 1e-5, std::optional<DataType> checkpoint_dtype = std::nullopt);
    std::shared_ptr<StampedLayerNorm> stamp(const Tensor& input, const Stream& stream, const std::optional<Tensor>& weight = std::nullopt,
                                            const std::optional<Tensor>& bias = std::nullopt, const std::optional<Tensor>& segment_offsets = std::nullopt,
                                            const Outputs& preallocated = {}) const;

   private:
    float epsilon;
    std::optional<DataType> checkpointDType;
};

class StampedLayerNormBackward : public StampedRowOperation {
   public:
    Tensor getInputGradientTensor() const { return inputGradient; }
    const std::optional<Tensor>& getWeightGradientTensor() const { return weightGradient; }
    const std::optional<Tensor>& getBiasGradientTensor() const { return biasGradient; }

   private:
    friend class LayerNormBackward;
    explicit StampedLayerNormBackward(const Stream& stream) : StampedRowOperation(stream) {}
    void enqueue(void* raw_stream) const override;

    Tensor error, rstd, inputGradient;
    std::optional<Tensor> input, mean, weight, segmentOffsets, weightGradient, biasGradient, workspace;
    std::optional<ActivationCheckpoint> checkpoint;
    thorhip_layer_norm_gradient call{};
};

class LayerNormBackward {
   public:
    struct Outputs {
        std::optional<Tensor> input_gradient, weight_gradient, bias_gradient;
    };
    explicit LayerNormBackward(bool weight_gradient = true, bool bias_gradient = true) : weightGradient(weight_gradient), biasGradient(bias_gradient) {}
    // from the forward pass's input
    std::shared_ptr<StampedLayerNormBackward> stamp(const Tensor& error_input, const Tensor& input, const Tensor& mean, const Tensor& reciprocal_deviation,
                                                    const Stream& stream, const std::optional<Tensor>& weight = std::nullopt,
                                                    const std::optional<Tensor>& segment_offsets = std::nullopt, const Outputs& preallocated = {}) const;
    // from the forward pass's checkpoint
    std::shared_ptr<StampedLayerNormBackward> stamp(const Tensor& error_input, const ActivationCheckpoint& checkpoint, const Tensor& reciprocal_deviation,
                                                    const Stream& stream, const std::optional<Tensor>& weight = std::nullopt,
                                                    const std::optional<Tensor>& segment_offsets = std::nullopt, const Outputs& preallocated = {}) const;

   private:
    std::shared_ptr<StampedLayerNormBackward> stampFrom(const Tensor& error_input, const std::optional<Tensor>& input, const std::optional<Tensor>& mean,
                                                        const std::optional<ActivationCheckpoint>& checkpoint, const Tensor& reciprocal_deviation,
                                                        const Stream& stream, const std::optional<Tensor>& weight,
                                                        const std::optional<Tensor>& segment_offsets, const Outputs& preallocated) const;
    bool weightGradient, biasGradient;
};

}  // namespace ThorImplementation
