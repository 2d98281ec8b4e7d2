// Host side of the serving operators: argument checks and launch plans, without a device.
#pragma once
#include <cstddef>
#include <cstdint>
#include <string>

#include "kernels/serving_args.hpp"
#include "pipeline_table.hpp"

namespace smelt_host {

inline bool is_serving(FamilyId f) { return f >= kFamRope && f <= kFamVerifyDraftsGiven; }

// What one pointer argument has to provide.
struct ServingOperand {
    void* ptr = nullptr;        // in
    size_t need = 0;            // bytes the launch touches from ptr on
    size_t align = 2;
    bool written = false;
    size_t row = 0, stride = 0; // rows: bytes of one and from one to the next (0: the bytes lie in one run)
};

constexpr int kServingMaxOperands = 16;
constexpr int kServingMaxSteps = 6;
constexpr size_t kServingArgBytes = 512;

struct ServingStep {
    int kernel = 0;             // index into ResolvedPipeline::serving_symbols
    uint32_t grid[3] = {1, 1, 1};
    uint32_t threads = 256;
    size_t lds = 0;
    size_t arg_bytes = 0;
    alignas(16) unsigned char args[kServingArgBytes];
};

struct ServingDevice {
    uint32_t compute_units = 256;
    void* workspace = nullptr;
    size_t workspace_bytes = 0;
};

struct ServingPlan {
    int operands = 0;
    ServingOperand operand[kServingMaxOperands];
    int steps = 0;              // 0: nothing to do
    ServingStep step[kServingMaxSteps];
};

// Resolves the pipeline names of the serving operators.
ResolveStatus resolve_serving(const std::string& entry, const char* act, ResolvedPipeline* out, std::string* why);

// Fills `plan` from the pipeline's pointers (plan->operand[i].ptr) and values (value[i], indexed as the pipeline's arguments).
// Returns 0 or a SMELT_HIP_ERR_* status with `why` set.
int plan_serving(const ResolvedPipeline& r, const uint32_t* value, const ServingDevice& dev, ServingPlan* plan, std::string* why);

}  // namespace smelt_host
