// ss_seq_attention_bf16.hip — leaky attention on bf16 operands (ss_seq_attention.hpp).
#include "ss_seq_attention.hpp"

long long ss_seq_leaky_ws_bf16(const LeakyArgs& p) { return LeakyShape<SS_SEQ_BF16>::state_floats(p.T, p.B, p.H, p.DA, p.DC); }
int ss_seq_leaky_bf16(const LeakyArgs& p, float* ws, hipStream_t s) { return LeakyShape<SS_SEQ_BF16>::run(p, ws, s); }
long long ss_seq_leaky_bwd_ws_bf16(const LeakyBwdArgs& d) { return LeakyShape<SS_SEQ_BF16>::bwd_floats(d); }
int ss_seq_leaky_bwd_bf16(const LeakyBwdArgs& d, hipStream_t s) { return LeakyShape<SS_SEQ_BF16>::bwd(d, s); }
