// forwards to the op:: umbrella (layer_norm, token_logprobs, global_norm, clip_by_global_norm and their gradients)
#include "dali/array/op.h"
