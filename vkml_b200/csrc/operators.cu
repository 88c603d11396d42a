// Whether a call of an operator would be accepted, told without a context.
#include "operators.cuh"

using namespace b200;

extern "C" {

int b200_check_operator(int which, const void* args, char* why, size_t why_len) {
    if (args == nullptr) return B200_INVALID_ARGUMENT;
    std::string message;
    int status = B200_OK;
    try {
        switch (which) {
            case B200_CALL_EMBEDDING:
            case B200_CALL_EMBEDDING_BACKWARD:
                check_embedding_call(*static_cast<const b200_embedding_args*>(args), which == B200_CALL_EMBEDDING_BACKWARD);
                break;
            case B200_CALL_BLOCK_NORM: check_block_norm(*static_cast<const b200_block_norm_args*>(args)); break;
            case B200_CALL_BLOCK_NORM_BACKWARD: check_block_norm_backward(*static_cast<const b200_block_norm_grad_args*>(args)); break;
            case B200_CALL_DISTILL_LOSS:
            case B200_CALL_DISTILL_LOSS_BACKWARD:
                check_distill_loss(*static_cast<const b200_distill_args*>(args), which == B200_CALL_DISTILL_LOSS);
                break;
            default: status = B200_INVALID_ARGUMENT; message = "unknown operator";
        }
    } catch (const Error& e) {
        status = e.status;
        message = e.message;
    } catch (const std::exception& e) {
        status = B200_INTERNAL_ERROR;
        message = e.what();
    }
    if (why != nullptr && why_len != 0) std::snprintf(why, why_len, "%s", message.c_str());
    return status;
}

}  // extern "C"
