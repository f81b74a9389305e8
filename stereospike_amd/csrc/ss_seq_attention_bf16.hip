// ss_seq_attention_bf16.hip — leaky attention on bf16 operands (ss_seq_attention.hpp).
#include "ss_seq_attention.hpp"

long long ss_seq_leaky_ws_bf16(const LeakyArgs& p) { return LeakyShape<SS_SEQ_BF16>::ws_floats(p); }
int ss_seq_leaky_bf16(const LeakyArgs& p, float* ws, hipStream_t s) { return LeakyShape<SS_SEQ_BF16>::run(p, ws, s); }
