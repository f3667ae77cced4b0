// device_ops.h — internal interface between engine.cu (the calling thread's error message) and device_ops.cu (operators on device tensors).
#pragma once

// sets the message of b200_last_error() and returns `code`
int dev_fail(int code, const char* msg);
// the watchdog's code of the operators in device_ops_experts.cu on the current device, which it clears (a cudaError_t)
int dev_experts_watchdog(int* code);
