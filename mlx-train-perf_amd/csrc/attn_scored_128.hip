// The kernels of attn_scored.hpp for head_dim 128.
#define MTP_SCORED_DH 128
#include "attn_scored.hpp"
