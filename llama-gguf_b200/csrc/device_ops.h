// device_ops.h — internal interface between engine.cu (the calling thread's error message) and device_ops.cu (operators on device tensors).
#pragma once

// sets the message of b200_last_error() and returns `code`
int dev_fail(int code, const char* msg);
