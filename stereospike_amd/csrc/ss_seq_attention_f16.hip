// ss_seq_attention_f16.hip — leaky attention on fp16 operands (ss_seq_attention.hpp).
#include "ss_seq_attention.hpp"

long long ss_seq_leaky_ws_f16(const LeakyArgs& p) { return LeakyShape<SS_SEQ_F16>::ws_floats(p); }
int ss_seq_leaky_f16(const LeakyArgs& p, float* ws, hipStream_t s) { return LeakyShape<SS_SEQ_F16>::run(p, ws, s); }
