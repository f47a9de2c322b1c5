// Every combination of what a device's kernels may have noted: the code that is answered, and that nothing is hidden.
#include <string.h>

#include "device_status.h"

int main() {
  int wrong = 0;
  for (int m = 0; m < 256; ++m) {
    ob::DeviceStatus s;
    int* waits[] = {&s.tensor_memory_wait, &s.decode_wait, &s.few_token_wait, &s.attend_wait, &s.attend_many_wait};
    int* batches[] = {&s.append_batch, &s.attend_batch, &s.attend_many_batch};
    for (int i = 0; i < 5; ++i) *waits[i] = m >> i & 1 ? 7 + i : 0;
    for (int i = 0; i < 3; ++i) *batches[i] = m >> (5 + i) & 1;
    char text[384] = "";
    const int rc = ob::describe(s, text, sizeof(text)), want = m & 31 ? ONEBIT_ERR_DEVICE_WAIT : m ? ONEBIT_ERR_BATCH : ONEBIT_OK;
    wrong += rc != want;
    wrong += (strstr(text, "gave up") != nullptr) != ((m & 31) != 0);
    wrong += (strstr(text, "page number") != nullptr) != (m >> 5 != 0);
    wrong += strlen(text) + 1 == sizeof(text);                // cut off
  }
  printf("%d\n", wrong);
  return wrong != 0;
}
