#include "sas_fp8_attn.cuh"
namespace sas_host {
bool fp8_tc_supported(const SasFp8Args &) { return false; }
size_t fp8_tc_pieces(const SasFp8Args &) { return 1; }
int launch_fp8_tc(const SasFp8Args &, const sas_fp8::Args &, const sas_fp8::Layout &, char *, cudaStream_t) { return SAS_ERR_UNSUPPORTED; }
} // namespace sas_host
