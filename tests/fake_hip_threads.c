/* The stand-in of fake_hip.c for calls of several threads: every launch notes its
 * thread and then waits a little, so that another thread's launches come in between
 * wherever the library lets them. */
#define hipLaunchKernel fake_base_launch
#define __hipPushCallConfiguration fake_base_push
#define __hipPopCallConfiguration fake_base_pop
#define hipMalloc fake_base_malloc
#include "fake_hip.c"
#undef hipLaunchKernel
#undef __hipPushCallConfiguration
#undef __hipPopCallConfiguration
#undef hipMalloc

#include <pthread.h>
#include <sys/syscall.h>
#include <unistd.h>

static pthread_mutex_t mu = PTHREAD_MUTEX_INITIALIZER;
static long launch_thread[MAX];
static __thread dim3 t_grid, t_block;
static __thread size_t t_lds;
static __thread hipStream_t t_stream;

long fake_launch_thread(int i) { return launch_thread[i]; }

hipError_t hipMalloc(void **p, size_t n) {
    pthread_mutex_lock(&mu);
    hipError_t e = fake_base_malloc(p, n);
    pthread_mutex_unlock(&mu);
    return e;
}
hipError_t __hipPushCallConfiguration(dim3 g, dim3 b, size_t lds, hipStream_t s) {
    return t_grid = g, t_block = b, t_lds = lds, t_stream = s, hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3 *g, dim3 *b, size_t *lds, hipStream_t *s) {
    return *g = t_grid, *b = t_block, *lds = t_lds, *s = t_stream, hipSuccess;
}
hipError_t hipLaunchKernel(const void *f, dim3 g, dim3 b, void **args, size_t lds,
                           hipStream_t s) {
    pthread_mutex_lock(&mu);
    if (n_launches < MAX) launch_thread[n_launches] = syscall(SYS_gettid);
    hipError_t e = fake_base_launch(f, g, b, args, lds, s);
    pthread_mutex_unlock(&mu);
    usleep(500);
    return e;
}
